// Rows into and out of a paged K/V cache of 8-bit codes (cache8.h); no
// counterpart in the reference.
//
// Write. Sequence s's new rows become its last logical tokens. A (block of
// tokens, kv head) has one scale:
//   a = max |x| over the block's new rows' finite values, at least 2^-92
//   need = the smallest 2^k with a <= 448 2^k (e4m3), a times the fp32 value of
//          1 / 127 (int8), as torch divides by 127 on the GPU
//   scale' = max(scale, need) if the block held earlier tokens of the sequence,
//            else need
//   code = nearest(x / scale'), +-448 or +-127 at most (an infinity too); NaN
//          stays one in e4m3 and is 0 in int8
// Where scale' grew, the earlier tokens' codes c become nearest(c scale / scale').
// The powers of two cost a floating code nothing and make the recoding exact but
// for the smallest values; an int8 code would lose up to a bit by them.
//
// Read. value = code * scale in fp32, rounded to the output's type (an int8 code's
// product takes up to 31 bits: two roundings where the scale is no power of two).
//
// Both are bound by HBM: 3 bytes per value for 16-bit rows.
#include "cache8.h"
#include "common.h"
#include "kernels.h"
#include "../../include/mtlattn_capi.h"

namespace mtlattn {

namespace {

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

struct Cache8KParams {
    const void* in[2]; int64_t in_rs[2];       // rows of K and V (write)
    void* out[2];                              // rows of K and V (read; contiguous)
    uint8_t* codes[2]; int64_t c_rs[2];
    float* scale[2];
    const int* block_table; int64_t bt_stride;
    const int* cu; const int* cu_kv;
    int64_t total;
    int num_seqs, hkv, d, page_size, block, num_pages;
    uint32_t div_row, div_unit;                // read: ceil(2^32 / units (8 values) of a row, of a head)
    uint32_t div_head;                         // ceil(2^16 / (d / 8))
};

// Eight values of a row, as they are stored, and as fp32.
template <typename T>
struct Raw8 {
    u32x4_t x;
    __device__ inline void load(const typename T::raw* p) { x = ld16(p); }
    __device__ inline void values(float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = lo16<T>(x[i]);
            f[2 * i + 1] = hi16<T>(x[i]);
        }
    }
    // The larger magnitudes' bits, in either half: patterns order as magnitudes do.
    static constexpr uint32_t kInf = T::code == BF16::code ? 0x7f80u : 0x7c00u;
    __device__ inline uint32_t max_bits(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u16x2_t a = __builtin_bit_cast(u16x2_t, x[i] & 0x7fff7fffu), b = __builtin_bit_cast(u16x2_t, m);
            m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
        }
        return m;
    }
    __device__ static inline uint32_t fold(uint32_t m) { return max(m & 0xffffu, m >> 16); }
    __device__ static inline float magnitude(uint32_t m) { return T::to_float((uint16_t)m); }
};
template <>
struct Raw8<F32> {
    u32x4_t x, y;
    __device__ inline void load(const float* p) {
        x = ld16(p);
        y = ld16(p + 4);
    }
    __device__ inline void values(float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = __uint_as_float(x[i]);
            f[4 + i] = __uint_as_float(y[i]);
        }
    }
    static constexpr uint32_t kInf = 0x7f800000u;
    __device__ inline uint32_t max_bits(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max(x[i] & 0x7fffffffu, y[i] & 0x7fffffffu));
        return m;
    }
    __device__ static inline uint32_t fold(uint32_t m) { return m; }
    __device__ static inline float magnitude(uint32_t m) { return __uint_as_float(m); }
};
template <typename T>
__device__ inline void store8(typename T::raw* p, const float* f) {
    st16(p, u32x4_t{T::pack2(f[0], f[1]), T::pack2(f[2], f[3]), T::pack2(f[4], f[5]), T::pack2(f[6], f[7])});
}
template <>
__device__ inline void store8<F32>(float* p, const float* f) {
    *reinterpret_cast<f32x4_t*>(p) = f32x4_t{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{f[4], f[5], f[6], f[7]};
}

// The scale that a block of largest magnitude a needs.
template <typename C>
__device__ inline float scale_for(float a) {
    a = fmaxf(a, 0x1p-92f);
    if (C::code == I8::code) return a * (1.f / 127.f);
    // a = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    const uint32_t bits = __float_as_uint(a);
    const int e = (int)(bits >> 23) - 126;
    return ldexpf(1.f, e - 9 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0));
}

// y, rounded to fp32 from an exact value that r's sign says it is below (r > 0) or above,
// as the odd one of the two floats next to that value: what is then rounded to fewer bits
// is rounded as if from the exact value.
__device__ inline float to_odd(float y, float r) {
    const uint32_t b = __float_as_uint(y), more = (r > 0.f) == (b >> 31 == 0) ? 1u : ~0u;
    return (r > 0.f || r < 0.f) && (b & 1u) == 0 ? __uint_as_float(b + more) : y;
}

// Four values as codes of this scale (pow2: the scale is a power of two; odd: there
// may be values that are not finite or too large for the scale).
template <typename C>
__device__ inline uint32_t encode4(const float* x, float scale, float inv, bool pow2, bool odd);
template <>
__device__ inline uint32_t encode4<E4M3>(const float* x, float scale, float inv, bool pow2, bool odd) {
    float y[4];
    if (pow2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = x[i] * inv;
    } else {
        // A caller's own scale m 2^e: x 2^-e / m, whose remainder is exact in one FMA.
        const int e = (int)(__float_as_uint(scale) >> 23) - 127;
        const float m = __uint_as_float((__float_as_uint(scale) & 0x7fffffu) | 0x3f800000u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = ldexpf(x[i], -e), q = v / m;
            y[i] = to_odd(q, fmaf(-q, m, v));
        }
    }
    if (odd) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = y[i] > 448.f ? 448.f : y[i];                 // (a NaN stays)
            y[i] = y[i] < -448.f ? -448.f : y[i];
        }
    }
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
}
template <>
__device__ inline uint32_t encode4<I8>(const float* x, float scale, float inv, bool, bool odd) {
    const float half = 0.5f * scale, lim = 127.f * scale;
    float n[4], r[4];
    bool tie = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = odd ? fminf(fmaxf(x[i], -lim), lim) : x[i];
        // n is nearest(v / scale) or, next to a tie, the other neighbour: the
        // remainder v - n scale is exact, and tells
        n[i] = __builtin_rintf(v * inv);
        r[i] = fmaf(-n[i], scale, v);
        tie = tie || fabsf(r[i]) >= half;
    }
    if (tie) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (fabsf(r[i]) > half || (fabsf(r[i]) == half && ((int)n[i] & 1) != 0)) n[i] += r[i] > 0.f ? 1.f : -1.f;
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int c = (int)n[i];
        if (odd) c = x[i] == x[i] ? min(max(c, -127), 127) : 0;
        w |= ((uint32_t)c & 0xffu) << (8 * i);
    }
    return w;
}

// Four codes of `scale` as codes of the larger scale `now`. For int8 in 64 bits: the
// scales of 16-bit rows are ratios of small numbers, so that quotients lie next to
// ties, closer than an fp32 rounding. For e4m3 `now`, which a block has grown to, is a
// power of two: a code times the ratio of the scales, the product's error in one FMA.
template <typename C>
__device__ inline uint32_t recode4(uint32_t w, float scale, float now) {
    float f[4];
    C::to_float4(w, f);
    if (C::code == E4M3::code) {
        const float ratio = scale / now;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y = f[i] * ratio;
            f[i] = to_odd(y, fmaf(f[i], ratio, -y));
        }
        return encode4<E4M3>(f, 1.f, 1.f, true, true);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)__builtin_rint((double)f[i] * scale / now);
    return encode4<I8>(f, 1.f, 1.f, true, true);
}

// One wave per 16 tokens of a block and kv head; the block / 16 waves of a
// (block, head) meet in LDS for its largest magnitude. A workgroup holds W waves:
// W / (block / 16) heads of one block, K or V; the other heads, then the other side,
// of the block come next in the grid. ITER * 64 lanes hold 8 values each, 16 d
// values in all, in registers between the two uses of them. (They do not fit where a
// workgroup has 16 waves, blocks of 256 tokens, and D > 128 in int8: of 128 registers a
// lane, 33 values go to memory for fp32 rows and 1 for 16-bit ones.)
// The blocks that a sequence's new rows touch are numbered over the sequences, 64 of
// them at a time, one lane each (total / block + 2 num_seqs bounds them); a wave's
// rows do not need the page table, so that their loads and its lookup go out
// together: offsets, then rows, then stores (a binary search, the ranges, the page
// and the rows one after the other took 132 us for 64800 tokens of 8 heads, D = 128,
// bf16, against 91 now, 402 MB).
template <typename T, typename C, int ITER, int W>
__global__ __launch_bounds__(W * 64) void cache8_write_kernel(Cache8KParams p) {
    __shared__ uint32_t s_max[W];
    __shared__ float s_old[W];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int sub = p.block / 16, team = w / sub, part = w - team * sub, heads = W / sub;
    const int groups = (p.hkv + heads - 1) / heads;
    const int head = (int)(blockIdx.x % groups) * heads + team, side = blockIdx.x / groups % 2;
    const int slot = blockIdx.x / groups / 2;

    int s = -1, blk = 0, start = 0, p0 = 0, p1 = 0, base = 0;
    for (int g0 = 0; g0 < p.num_seqs && s < 0; g0 += 64) {
        const int i = min(g0 + lane, p.num_seqs - 1);
        const SeqRange r = seq_range(p.cu, i, p.total);
        const int kv = kv_length(p.cu_kv, i), n = r.end - r.start, from = max(kv - n, 0) / p.block;
        const int mine = g0 + lane < p.num_seqs && n > 0 && kv > 0 ? (kv - 1) / p.block - from + 1 : 0;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(sum, o);
            if (lane >= o) sum += y;
        }
        const uint64_t past = __ballot(base + sum > slot);
        if (past != 0) {
            const int l = __builtin_ctzll(past);
            s = g0 + l;
            blk = __builtin_amdgcn_readlane(from, l) + slot - base - __builtin_amdgcn_readlane(sum - mine, l);
            start = __builtin_amdgcn_readlane(r.start, l);
            p1 = __builtin_amdgcn_readlane(kv, l);
            p0 = p1 - __builtin_amdgcn_readlane(n, l);
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    if (s < 0) return;
    const int b0 = blk * p.block;                               // first token of the block
    const bool active = head < p.hkv, held = b0 < p0;           // earlier tokens in the block
    const int64_t col = b0 / p.page_size;
    const int pg = col < p.bt_stride ? p.block_table[(int64_t)s * p.bt_stride + col] : -1;

    Raw8<T> x[ITER];
    int kind[ITER];                                             // 1: new, 2: earlier
    const int du = p.d / 8;
    const typename T::raw* in = (const typename T::raw*)p.in[side] + (int64_t)head * p.d;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int e = lane + 64 * it, t = (int)(((uint32_t)e * p.div_head) >> 16), c = e - t * du;
        const int pos = b0 + 16 * part + t;
        kind[it] = !active || t >= 16 || pos >= p1 ? 0 : pos >= p0 ? 1 : 2;
        if (kind[it] == 1) x[it].load(in + (start + (pos - p0)) * p.in_rs[side] + 8 * c);
    }
    if (pg < 0 || pg >= p.num_pages) return;                    // (the whole workgroup)
    const int64_t row0 = (int64_t)pg * p.page_size + (b0 - (int)col * p.page_size);
    float* scale_at = p.scale[side] + (row0 / p.block) * p.hkv + head;
    uint8_t* codes = p.codes[side] + (row0 + 16 * part) * p.c_rs[side] + (int64_t)head * p.d;
    float old = 0.f;
    u32x2_t code[ITER];
    if (held && active) {
        if (part == 0) old = *scale_at;
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            const int e = lane + 64 * it, t = (int)(((uint32_t)e * p.div_head) >> 16), c = e - t * du;
            if (kind[it] == 2) code[it] = ld8(codes + t * p.c_rs[side] + 8 * c);
        }
    }
    uint32_t bits = 0;
#pragma unroll
    for (int it = 0; it < ITER; ++it)
        if (kind[it] == 1) bits = x[it].max_bits(bits);
    bits = Raw8<T>::fold(bits);
    bool odd = __any(bits >= Raw8<T>::kInf);                    // something is not finite
    if (odd) {
        float a = 0.f;
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            if (kind[it] != 1) continue;
            float f[8];
            x[it].values(f);
#pragma unroll
            for (int i = 0; i < 8; ++i) a = fabsf(f[i]) < kPosInf ? fmaxf(a, fabsf(f[i])) : a;
        }
        bits = __float_as_uint(a);
    } else {
        bits = __float_as_uint(Raw8<T>::magnitude(bits));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, o));
    if (sub > 1) {
        if (lane == 0) {
            s_max[w] = bits;
            if (part == 0) s_old[team] = old;
        }
        __syncthreads();
        for (int i = 0; i < sub; ++i) bits = max(bits, s_max[team * sub + i]);
        old = s_old[team];
    }
    if (!active) return;
    old = __shfl(old, 0);
    const float need = scale_for<C>(__uint_as_float(bits));
    const float now = held && old > need ? old : need;
    const float inv = 1.f / now;
    const bool pow2 = (__float_as_uint(now) & 0x7fffffu) == 0;
    const bool grew = held && now != old;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int e = lane + 64 * it, t = (int)(((uint32_t)e * p.div_head) >> 16), c = e - t * du;
        if (kind[it] == 1) {
            float f[8];
            x[it].values(f);
            st8(codes + t * p.c_rs[side] + 8 * c,
                u32x2_t{encode4<C>(f, now, inv, pow2, odd), encode4<C>(f + 4, now, inv, pow2, odd)});
        } else if (kind[it] == 2 && grew) {
            st8(codes + t * p.c_rs[side] + 8 * c, u32x2_t{recode4<C>(code[it][0], old, now), recode4<C>(code[it][1], old, now)});
        }
    }
    if (part == 0 && lane == 0 && (!held || grew)) *scale_at = now;
}

constexpr int kReadRows = 16;

// 16 output rows per workgroup: 16 lanes find the rows' places, then all of
// them stream 8 values at a time. Rows of no sequence are written as 0.
template <typename T, typename C>
__global__ __launch_bounds__(256) void cache8_read_kernel(Cache8KParams p) {
    __shared__ int s_row[kReadRows], s_srow[kReadRows];         // cache row (-1: none), row of scales
    const int side = blockIdx.y, tid = threadIdx.x;
    const int64_t r0 = (int64_t)blockIdx.x * kReadRows;
    if (tid < 64) {
        // lane t: row r0 + t. Among 64 sequences by one load of all lanes, among more by a search
        const int r = (int)min(r0 + min(tid, kReadRows - 1), (int64_t)0x7fffffff);
        int lo = 0;
        SeqRange nr;
        int kv;
        if (p.num_seqs <= 64) {
            const int i = min(tid, p.num_seqs - 1), first = p.cu[i];
            const SeqRange mine = seq_range(p.cu, i, p.total);
            const int len = kv_length(p.cu_kv, i);
            for (int t = 0; t < kReadRows; ++t) {
                const uint64_t le = __ballot(tid < p.num_seqs && first <= r0 + t);
                if (tid == t) lo = 63 - __builtin_clzll(le | 1);
            }
            nr.start = __shfl(mine.start, lo);
            nr.end = __shfl(mine.end, lo);
            kv = __shfl(len, lo);
        } else {
            int hi = p.num_seqs - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (p.cu[mid] <= r) lo = mid; else hi = mid - 1;
            }
            nr = seq_range(p.cu, lo, p.total);
            kv = kv_length(p.cu_kv, lo);
        }
        if (tid < kReadRows) {
            const int pos = r < nr.end ? kv - (nr.end - r) : -1;
            int row = -1;
            if (r >= nr.start && pos >= 0) {
                const int page = pos / p.page_size;
                const int64_t col = min((int64_t)page, p.bt_stride - 1);
                const int pg = min(max(p.block_table[(int64_t)lo * p.bt_stride + col], 0), p.num_pages - 1);
                row = pg * p.page_size + (pos - page * p.page_size);
            }
            s_row[tid] = row;
            s_srow[tid] = row / p.block;
        }
    }
    __syncthreads();
    const int rows = (int)min((int64_t)kReadRows, p.total - r0), upr = p.hkv * (p.d / 8);
    typename T::raw* out = (typename T::raw*)p.out[side] + r0 * p.hkv * p.d;
    // four units' loads in flight (one at a time: 500 rows of 8 heads 6.6 us against 5.8)
    constexpr int U = 4;
    for (int u0 = tid; u0 < rows * upr; u0 += 256 * U) {
        u32x2_t w[U];
        float sc[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int u = u0 + 256 * k, t = (int)__umulhi((uint32_t)u, p.div_row), i = u - t * upr;
            const int row = u < rows * upr ? s_row[t] : -1;
            w[k] = u32x2_t{0u, 0u};
            sc[k] = 0.f;
            if (row >= 0) {
                const int head = (int)__umulhi((uint32_t)i, p.div_unit);
                w[k] = ld8(p.codes[side] + row * p.c_rs[side] + 8 * i);
                sc[k] = p.scale[side][(int64_t)s_srow[t] * p.hkv + head];
            }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int u = u0 + 256 * k;
            if (u >= rows * upr) break;
            float f[8];
            C::to_float4(w[k][0], f);
            C::to_float4(w[k][1], f + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= sc[k];
            store8<T>(out + (int64_t)u * 8, f);
        }
    }
}

Cache8KParams params(const Cache8Args& a) {
    Cache8KParams p;
    p.in[0] = a.k; p.in[1] = a.v;
    p.in_rs[0] = a.k_rs; p.in_rs[1] = a.v_rs;
    p.out[0] = a.k; p.out[1] = a.v;
    p.codes[0] = a.k_cache; p.codes[1] = a.v_cache;
    p.c_rs[0] = a.kc_rs; p.c_rs[1] = a.vc_rs;
    p.scale[0] = a.k_scale; p.scale[1] = a.v_scale;
    p.block_table = a.block_table; p.bt_stride = a.bt_stride;
    p.cu = a.cu; p.cu_kv = a.cu_kv;
    p.total = a.total;
    p.num_seqs = a.num_seqs; p.hkv = a.hkv; p.d = a.d;
    p.page_size = a.page_size; p.block = a.block; p.num_pages = a.num_pages;
    const uint64_t upr = (uint64_t)a.hkv * (a.d / 8);
    p.div_row = (uint32_t)(((1ull << 32) + upr - 1) / upr);
    p.div_unit = (uint32_t)(((1ull << 32) + a.d / 8 - 1) / (a.d / 8));
    p.div_head = (65536u + a.d / 8 - 1) / (a.d / 8);
    return p;
}

template <typename T, typename C, int ITER>
hipError_t write_iter(const Cache8KParams& p, hipStream_t st) {
    const int sub = p.block / 16, W = sub <= 8 ? 8 : 16;
    const int64_t slots = p.total / p.block + 2 * (int64_t)p.num_seqs;
    const int heads = W / sub;
    const int64_t wgs = slots * ((p.hkv + heads - 1) / heads) * 2;
    if (wgs > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)wgs);
    if (W == 8) hipLaunchKernelGGL((cache8_write_kernel<T, C, ITER, 8>), grid, dim3(512), 0, st, p);
    else hipLaunchKernelGGL((cache8_write_kernel<T, C, ITER, 16>), grid, dim3(1024), 0, st, p);
    return hipGetLastError();
}

template <typename T, typename C>
hipError_t write_typed(const Cache8KParams& p, hipStream_t st) {
    if (p.d <= 64) return write_iter<T, C, 2>(p, st);
    if (p.d <= 96) return write_iter<T, C, 3>(p, st);
    if (p.d <= 128) return write_iter<T, C, 4>(p, st);
    return write_iter<T, C, 8>(p, st);
}

template <typename T, typename C>
hipError_t read_typed(const Cache8KParams& p, hipStream_t st) {
    const int64_t tiles = (p.total + kReadRows - 1) / kReadRows;
    if (tiles > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL((cache8_read_kernel<T, C>), dim3((unsigned)tiles, 2), dim3(256), 0, st, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_cache8_write(int dtype, const Cache8Args& a, hipStream_t st) {
    if (a.total <= 0) return hipSuccess;
    const Cache8KParams p = params(a);
    const bool e4m3 = a.code == MTLATTN_CODE_E4M3;
    if (dtype == MTLATTN_DTYPE_BF16) return e4m3 ? write_typed<BF16, E4M3>(p, st) : write_typed<BF16, I8>(p, st);
    if (dtype == MTLATTN_DTYPE_F16) return e4m3 ? write_typed<F16, E4M3>(p, st) : write_typed<F16, I8>(p, st);
    if (dtype == MTLATTN_DTYPE_F32) return e4m3 ? write_typed<F32, E4M3>(p, st) : write_typed<F32, I8>(p, st);
    return hipErrorInvalidValue;
}

hipError_t launch_cache8_read(int dtype, const Cache8Args& a, hipStream_t st) {
    if (a.total <= 0) return hipSuccess;
    const Cache8KParams p = params(a);
    const bool e4m3 = a.code == MTLATTN_CODE_E4M3;
    if (dtype == MTLATTN_DTYPE_BF16) return e4m3 ? read_typed<BF16, E4M3>(p, st) : read_typed<BF16, I8>(p, st);
    if (dtype == MTLATTN_DTYPE_F16) return e4m3 ? read_typed<F16, E4M3>(p, st) : read_typed<F16, I8>(p, st);
    if (dtype == MTLATTN_DTYPE_F32) return e4m3 ? read_typed<F32, E4M3>(p, st) : read_typed<F32, I8>(p, st);
    return hipErrorInvalidValue;
}

}  // namespace mtlattn
