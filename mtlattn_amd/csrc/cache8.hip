// Rows into and out of a paged K/V cache of 8-bit codes (cache8.h); no
// counterpart in the reference.
//
// Write. Sequence s's new rows become its last logical tokens. A (block of
// tokens, kv head) has one scale:
//   a = max |x| over the block's new rows' finite values, at least 2^-92
//   need = the smallest 2^k with a <= 448 2^k (e4m3), a / 127 (int8)
//   scale' = max(scale, need) if the block held earlier tokens of the sequence,
//            else need
//   code = nearest(x / scale'), +-448 or +-127 at most (an infinity too); NaN
//          stays one in e4m3 and is 0 in int8
// Where scale' grew, the earlier tokens' codes c become nearest(c scale / scale').
// The powers of two cost a floating code nothing and make the recoding exact but
// for the smallest values; an int8 code would lose up to a bit by them.
//
// Read. value = code * scale, rounded once to the output's type.
//
// Both are bound by HBM: 3 bytes per value for 16-bit rows.
#include "cache8.h"
#include "common.h"
#include "kernels.h"
#include "../../include/mtlattn_capi.h"

namespace mtlattn {

namespace {

struct Cache8KParams {
    const void* in[2]; int64_t in_rs[2];       // rows of K and V (write)
    void* out[2];                              // rows of K and V (read; contiguous)
    uint8_t* codes[2]; int64_t c_rs[2];
    float* scale[2];
    const int* block_table; int64_t bt_stride;
    const int* cu; const int* cu_kv;
    int64_t total;
    int num_seqs, hkv, d, page_size, block, num_pages;
    uint32_t div_row;                          // read: ceil(2^32 / units of a row)
    uint32_t div_head;                         // ceil(2^16 / (d / 8))
};

// Logical length of sequence s (the offsets are not bounded by a tensor).
__device__ inline int kv_length(const int* __restrict__ cu_kv, int s) {
    const int64_t n = (int64_t)cu_kv[s + 1] - cu_kv[s];
    return (int)min(max(n, (int64_t)0), (int64_t)0x7ffffff0);
}

// Eight values of a row as fp32.
template <typename T>
__device__ inline void load8(const typename T::raw* p, float* f) {
    const u32x4_t x = ld16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = lo16<T>(x[i]);
        f[2 * i + 1] = hi16<T>(x[i]);
    }
}
template <>
__device__ inline void load8<F32>(const float* p, float* f) {
    const u32x4_t x = ld16(p), y = ld16(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = __uint_as_float(x[i]);
        f[4 + i] = __uint_as_float(y[i]);
    }
}
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
    if (C::code == I8::code) return a / 127.f;
    // a = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    const uint32_t bits = __float_as_uint(a);
    const int e = (int)(bits >> 23) - 126;
    return ldexpf(1.f, e - 9 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0));
}

// Four values as codes of this scale (pow2: the scale is a power of two).
template <typename C>
__device__ inline uint32_t encode4(const float* x, float scale, float inv, bool pow2);
template <>
__device__ inline uint32_t encode4<E4M3>(const float* x, float scale, float inv, bool pow2) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = pow2 ? x[i] * inv : x[i] / scale;
        const float u = v > 448.f ? 448.f : v;                  // (a NaN stays)
        y[i] = u < -448.f ? -448.f : u;
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
}
template <>
__device__ inline uint32_t encode4<I8>(const float* x, float scale, float inv, bool) {
    uint32_t w = 0;
    const float half = 0.5f * scale, lim = 127.f * scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = fminf(fmaxf(x[i], -lim), lim);
        // n is nearest(v / scale) or, next to a tie, the other neighbour: v - n scale
        // is exact, and tells
        float n = __builtin_rintf(v * inv);
        const float r = fmaf(-n, scale, v);
        const bool odd = ((int)n & 1) != 0;
        if (r > half || (r == half && odd)) n += 1.f;
        if (r < -half || (r == -half && odd)) n -= 1.f;
        n = fminf(fmaxf(n, -127.f), 127.f);
        const int c = x[i] == x[i] ? (int)n : 0;
        w |= ((uint32_t)c & 0xffu) << (8 * i);
    }
    return w;
}

// Four codes of `scale` as codes of the larger scale `now`. In 64 bits: the
// scales of 16-bit rows are ratios of small numbers, so that quotients lie next to
// ties, closer than an fp32 rounding.
template <typename C>
__device__ inline uint32_t recode4(uint32_t w, double scale, double now) {
    float f[4];
    C::to_float4(w, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double x = (double)f[i] * scale / now;
        f[i] = (float)(C::code == I8::code ? __builtin_rint(x) : x);
    }
    if (C::code == E4M3::code) return encode4<E4M3>(f, 1.f, 1.f, true);
    return encode4<I8>(f, 1.f, 1.f, true);
}

// One wave per 16 tokens of a block and kv head; the block / 16 waves of a
// (block, head) meet in LDS for its largest magnitude. A workgroup holds W waves:
// W / (block / 16) heads of one block. ITER * 64 lanes hold 8 values each,
// 16 d values in all, in registers between the two uses of them. Blocks that a
// sequence's new rows touch: slots cu[s] / block + 2 s + i, at least as many as
// there can be, found without the host.
template <typename T, typename C, int ITER, int W>
__global__ __launch_bounds__(W * 64) void cache8_write_kernel(Cache8KParams p) {
    __shared__ float s_max[W], s_old[W];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int sub = p.block / 16, team = w / sub, part = w - team * sub;
    const int side = blockIdx.z, slot = blockIdx.x;

    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        const int c = min(max(p.cu[mid], 0), (int)p.total);
        if (c / p.block + 2 * mid <= slot) lo = mid; else hi = mid - 1;
    }
    const int s = lo;
    const SeqRange nr = seq_range(p.cu, s, p.total);
    const int n_new = nr.end - nr.start, p1 = kv_length(p.cu_kv, s), p0 = p1 - n_new;
    const int64_t blk = max(p0, 0) / p.block + (slot - (nr.start / p.block + 2 * s));
    const int64_t b0 = blk * p.block;                           // first token of the block
    if (n_new == 0 || b0 >= p1) return;
    const int64_t col = b0 / p.page_size;
    if (col >= p.bt_stride) return;
    const int pg = p.block_table[(int64_t)s * p.bt_stride + col];
    if (pg < 0 || pg >= p.num_pages) return;
    const int64_t row0 = (int64_t)pg * p.page_size + (b0 - col * p.page_size);

    const int head = blockIdx.y * (W / sub) + team;
    const bool active = head < p.hkv;
    const int du = p.d / 8;
    float* scale_at = p.scale[side] + (row0 / p.block) * p.hkv + head;
    const bool held = b0 < p0;                                  // earlier tokens in the block
    float old = 0.f;
    if (active && held && part == 0) old = *scale_at;

    float x[ITER][8];
    u32x2_t code[ITER];
    int kind[ITER];                                             // 1: new, 2: earlier
    float amax = 0.f;
    const typename T::raw* in = (const typename T::raw*)p.in[side] + (int64_t)head * p.d;
    uint8_t* codes = p.codes[side] + (row0 + 16 * part) * p.c_rs[side] + (int64_t)head * p.d;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int e = lane + 64 * it, t = (int)(((uint32_t)e * p.div_head) >> 16), c = e - t * du;
        const int64_t pos = b0 + 16 * part + t;
        kind[it] = !active || t >= 16 || pos >= p1 ? 0 : pos >= p0 ? 1 : 2;
        if (kind[it] == 1) load8<T>(in + (nr.start + (pos - p0)) * p.in_rs[side] + 8 * c, x[it]);
        if (kind[it] == 2) code[it] = ld8(codes + t * p.c_rs[side] + 8 * c);
    }
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        if (kind[it] != 1) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float m = fabsf(x[it][i]);
            amax = m < kPosInf ? fmaxf(amax, m) : amax;         // (finite values)
        }
    }
    amax = wave_max(amax);
    if (sub > 1) {
        if (lane == 0) {
            s_max[w] = amax;
            if (part == 0) s_old[team] = old;
        }
        __syncthreads();
        for (int i = 0; i < sub; ++i) amax = fmaxf(amax, s_max[team * sub + i]);
        old = s_old[team];
    }
    if (!active) return;
    old = __shfl(old, 0);
    const float need = scale_for<C>(amax);
    const float now = held && old > need ? old : need;
    const float inv = 1.f / now;
    const bool pow2 = (__float_as_uint(now) & 0x7fffffu) == 0;
    const bool grew = held && now != old;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int e = lane + 64 * it, t = (int)(((uint32_t)e * p.div_head) >> 16), c = e - t * du;
        if (kind[it] == 1)
            st8(codes + t * p.c_rs[side] + 8 * c,
                u32x2_t{encode4<C>(x[it], now, inv, pow2), encode4<C>(x[it] + 4, now, inv, pow2)});
        else if (kind[it] == 2 && grew)
            st8(codes + t * p.c_rs[side] + 8 * c, u32x2_t{recode4<C>(code[it][0], old, now), recode4<C>(code[it][1], old, now)});
    }
    if (part == 0 && lane == 0 && (!held || grew)) *scale_at = now;
}

constexpr int kReadRows = 16;

// 16 output rows per workgroup: 16 lanes find the rows' places, then all of
// them stream 8 values at a time. Rows of no sequence are written as 0.
template <typename T, typename C>
__global__ __launch_bounds__(256) void cache8_read_kernel(Cache8KParams p) {
    __shared__ int64_t s_row[kReadRows];
    const int side = blockIdx.y;
    const int64_t r0 = (int64_t)blockIdx.x * kReadRows;
    if (threadIdx.x < kReadRows) {
        const int64_t r = r0 + threadIdx.x;
        int lo = 0, hi = p.num_seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (p.cu[mid] <= r) lo = mid; else hi = mid - 1;
        }
        const SeqRange nr = seq_range(p.cu, lo, p.total);
        int64_t row = -1;
        if (r >= nr.start && r < nr.end) {
            const int64_t pos = (int64_t)kv_length(p.cu_kv, lo) - (nr.end - r);
            if (pos >= 0) {
                const int64_t col = min(pos / p.page_size, p.bt_stride - 1);
                const int pg = min(max(p.block_table[(int64_t)lo * p.bt_stride + col], 0), p.num_pages - 1);
                row = (int64_t)pg * p.page_size + pos % p.page_size;
            }
        }
        s_row[threadIdx.x] = row;
    }
    __syncthreads();
    const int rows = (int)min((int64_t)kReadRows, p.total - r0), du = p.d / 8, upr = p.hkv * du;
    typename T::raw* out = (typename T::raw*)p.out[side] + r0 * p.hkv * p.d;
    for (int u = threadIdx.x; u < rows * upr; u += 256) {
        const int t = (int)__umulhi((uint32_t)u, p.div_row), i = u - t * upr;
        const int64_t row = s_row[t];
        float f[8] = {};
        if (row >= 0) {
            const int head = i / du;
            const u32x2_t w = ld8(p.codes[side] + row * p.c_rs[side] + 8 * i);
            const float sc = p.scale[side][(row / p.block) * p.hkv + head];
            C::to_float4(w[0], f);
            C::to_float4(w[1], f + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= sc;
        }
        store8<T>(out + (int64_t)u * 8, f);
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
    p.div_head = (65536u + a.d / 8 - 1) / (a.d / 8);
    return p;
}

template <typename T, typename C, int ITER>
hipError_t write_iter(const Cache8KParams& p, hipStream_t st) {
    const int sub = p.block / 16, W = sub <= 8 ? 8 : 16;
    const int64_t slots = p.total / p.block + 2 * (int64_t)p.num_seqs;
    const int heads = W / sub;
    const dim3 grid((unsigned)slots, (unsigned)((p.hkv + heads - 1) / heads), 2);
    if (slots > 0x7fffffff || grid.y > 65535) return hipErrorInvalidValue;
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
