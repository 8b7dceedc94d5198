// Decode over a paged K/V cache of 8-bit codes (e4m3 or int8) with an fp32
// scale per block of tokens and kv head; no counterpart in the reference.
//
//   S[n, j] = scale * s_k(j) * (q_n . c_k(j)) + bias,  P = softmax(S),
//   O[n] = sum_j P[n, j] s_v(j) c_v(j)
//
// As on the 16-bit caches (decode.hip) decode is bound by the stream of K and
// V, here 2 D bytes per key and kv head, and the rows of a GQA group share it
// as the 16 columns of v_mfma_f32_16x16x32. What differs:
//   * The scales never touch the codes: s_k multiplies the score, s_v the
//     softmax weight, both uniform over 16 keys (a block is a multiple of 16
//     tokens). The codes are converted exactly (cache8.h) to the query's type for
//     Q K^T, to bf16 for P V.
//   * P s_v, which spans fp32's range, goes into the P V product as the sum of two
//     bf16 values (16 significant bits): the weights are not what limits the
//     result, and the matrix cores have the time (MFMA is under a fifth of a
//     tile's issue slots).
//   * No LDS for the tiles. K goes from HBM into operand registers, 16 codes of a
//     row per load, the contraction over D permuted alike in q. V is loaded so
//     that a lane holds the 8 keys that its slots of the P V contraction need,
//     D / 16 neighbouring columns of each, and transposes 4 x 4 bytes in registers
//     (v_perm_b32); which column a lane's operand row stands for is a
//     permutation that only the output's addresses see.
//   * Page lookups and scales of up to 32 tiles are fetched at once, one lane per
//     16-key block, and read from there by v_readlane: no dependent loads per tile.
//   * The NW waves of a workgroup take the tiles of an item in turn and meet in
//     LDS at its end; items that are whole sequences write their rows, the others
//     normalised partials for the combine kernel.
#include "cache8.h"
#include "common.h"
#include "decode_common.h"
#include "kernels.h"
#include "../../include/mtlattn_capi.h"

namespace mtlattn {

namespace {

// Bytes of a lane's columns of one V row: D / 16 codes.
template <int D> struct VCodes;
template <> struct VCodes<128> {
    u32x2_t v;
    __device__ inline void load(const uint8_t* p) { v = ld8(p); }
    __device__ inline uint32_t word(int i) const { return v[i]; }
};
template <> struct VCodes<64> {
    uint32_t v;
    __device__ inline void load(const uint8_t* p) { v = *reinterpret_cast<const uint32_t*>(p); }
    __device__ inline uint32_t word(int) const { return v; }
};

template <int D, int KB>
struct Tile8 {
    u32x4_t k[KB][D / 64];      // per 16-key block: key n16, codes 64 c + 16 lg ..
    VCodes<D> v[KB][4];         // keys 4 lg + i, codes (D / 16) n16 ..
    float bias[KB][4];          // of the lane's row, keys 4 lg + i
    float ks[KB], vs[KB];       // scales: s_k * scale * log2 e, s_v
};

template <typename T, typename C, int D, bool BIAS, int NW, int KT>
__global__ __launch_bounds__(NW * 64) void decode8_kernel(DecKParams p, typename T::raw* __restrict__ out,
                                                          float* __restrict__ lse_out) {
    constexpr int KB = KT / 16, NC = D / 64, DB = D / 16, CW = D / 16;
    constexpr int TPV = 64 / KB;                     // tiles whose lookups one vector holds
    constexpr int OROW = D * 4 + 16;                 // bytes of an fp32 O row in LDS (padded)
    __shared__ __attribute__((aligned(16))) char smem[NW * 16 * OROW + NW * 32 * 4];
    float* ml = reinterpret_cast<float*>(smem + NW * 16 * OROW);   // [NW][16] row max (log2), [NW][16] row sum

    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n16 = lane & 15, lg = lane >> 4;

    int wid = blockIdx.x;
    const int hk = wid % p.hkv; wid /= p.hkv;
    const int hgi = wid % p.n_hg;
    const int slot = wid / p.n_hg;
    int s, ks, ke;
    const bool has_keys = item_range(p, slot, s, ks, ke);
    // fixed chunks past a sequence's end are not read by the combine
    if (!has_keys && p.chunk > 0) return;
    const SeqRange qr = seq_range(p.cu_q, s, p.total_q);
    const SeqRange kr = seq_range(p.cu_kv, s, p.total_kv);
    const int q_len = qr.end - qr.start, kv_len = kr.end - kr.start;
    if (q_len == 0) return;
    const int coff = kv_len - q_len;

    // Row n of the 16 columns: head hh = n / q_len of this group, query n % q_len.
    const int rows = min(p.hpb * q_len, 16);
    const bool row_ok = n16 < rows;
    const int hh = row_ok ? n16 / q_len : 0;
    const int qi = row_ok ? n16 - hh * q_len : 0;
    const int head = hk * p.g + hgi * p.hpb + hh;
    const int64_t grow = qr.start + qi;

    // operand kc = 2 c + h: codes 64 c + 16 lg + 8 h .. + 7 of a row
    u32x4_t qf[2 * NC];
    {
        const uint16_t* qp = p.q + grow * p.q_rs + (int64_t)head * D + 16 * lg;
#pragma unroll
        for (int kc = 0; kc < 2 * NC; ++kc) qf[kc] = ld16(qp + 64 * (kc >> 1) + 8 * (kc & 1));
    }
    const float* brow = nullptr;
    if (BIAS)
        brow = p.bias + bias_row_offset(grow, s, qr.start, p.bias_qs, p.bias_ss, p.bias_rows) +
               (int64_t)head * p.bias_hs;

    const int n_tiles = has_keys ? (ke - ks + KT - 1) / KT : 0;
    const int n_my = n_tiles > w ? (n_tiles - w + NW - 1) / NW : 0;   // tiles w, w + NW, ..
    const uint8_t* kbase = (const uint8_t*)p.k + (int64_t)hk * D;
    const uint8_t* vbase = (const uint8_t*)p.v + (int64_t)hk * D;
    const int* bt = p.block_table + (int64_t)s * p.bt_stride;
    const int bt_last = (int)min(p.bt_stride, (int64_t)0x7fffffff) - 1;
    const uint32_t k_rs = (uint32_t)p.k_rs, v_rs = (uint32_t)p.v_rs;
    const uint32_t koff = (uint32_t)n16 * k_rs + 16u * (uint32_t)lg;
    uint32_t voff[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) voff[i] = (uint32_t)(4 * lg + i) * v_rs + (uint32_t)(CW * n16);

    // lookups of tiles [i0, i0 + TPV) of this wave: lane l has block l % KB of tile
    // i0 + l / KB (blocks past the item's end: its last block)
    int vrow = 0;
    float vks = 0.f, vvs = 0.f;
    auto lookup = [&](int i0) {
        const int key = min(ks + (w + (i0 + lane / KB) * NW) * KT + 16 * (lane % KB), ke - 1) & ~15;
        const int col = min(key / p.page_size, bt_last), off = key % p.page_size;
        const int pg = min(max(bt[col], 0), p.num_pages - 1);
        vrow = pg * p.page_size + off;
        const int64_t sc = (int64_t)(vrow / p.block) * p.hkv + hk;
        vks = p.k_scale[sc] * p.scale_log2;
        vvs = p.v_scale[sc];
    };
    auto load = [&](int i, Tile8<D, KB>& t) {
        if (i % TPV == 0) lookup(i);
        const int kt = ks + (w + i * NW) * KT;
        const int l0 = (i % TPV) * KB;
        const bool full = kt + KT <= ke;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int row = __builtin_amdgcn_readlane(vrow, l0 + b);
            t.ks[b] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vks), l0 + b));
            t.vs[b] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vvs), l0 + b));
            const uint8_t* kp = kbase + (int64_t)row * p.k_rs;
            const uint8_t* vp = vbase + (int64_t)row * p.v_rs;
            if (full) {
#pragma unroll
                for (int c = 0; c < NC; ++c) t.k[b][c] = ld16(kp + koff + 64 * c);
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) t.v[b][i4].load(vp + voff[i4]);
            } else {
                // keys past the end read the last key: finite, masked to P = 0
                const int last = ke - 1 - (min(kt + 16 * b, ke - 1) & ~15);
                const uint32_t ko = (uint32_t)min(n16, last) * k_rs + 16u * (uint32_t)lg;
#pragma unroll
                for (int c = 0; c < NC; ++c) t.k[b][c] = ld16(kp + ko + 64 * c);
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4)
                    t.v[b][i4].load(vp + (uint32_t)min(4 * lg + i4, last) * v_rs + (uint32_t)(CW * n16));
            }
        }
        if (BIAS) {
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int key = kt + 16 * b + 4 * lg;
                if (p.bias_v4 && kt + KT <= p.bias_cols) {
                    const f32x4_t b4 = *reinterpret_cast<const f32x4_t*>(brow + key);
#pragma unroll
                    for (int r = 0; r < 4; ++r) t.bias[b][r] = b4[r];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = brow[min((int64_t)(key + r), p.bias_cols - 1)];
                        t.bias[b][r] = key + r < p.bias_cols ? x : 0.f;
                    }
                }
            }
        }
    };

    float m_run = kNegInf, l_run = 0.f;
    f32x4_t oacc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) oacc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    auto step = [&](int i, const Tile8<D, KB>& t) __attribute__((always_inline)) {
        const int kt = ks + (w + i * NW) * KT;
        // S^T = K Q^T, 16 keys at a time
        f32x4_t sc[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            sc[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x2_t a = C::template unpack4<T>(t.k[b][c][2 * h]), a2 = C::template unpack4<T>(t.k[b][c][2 * h + 1]);
                    sc[b] = mfma16<T>(u32x4_t{a[0], a[1], a2[0], a2[1]}, qf[2 * c + h], sc[b]);
                }
            }
        }
        // (rows' window bands start at qi + coff - W + 1 <= coff + q_len - W)
        const bool need_mask = (kt + KT > ke) || (p.causal && kt + KT - 1 > coff) ||
                               (p.window > 0 && kt < coff + q_len - p.window);
        float mx = kNegInf;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = kt + 16 * b + 4 * lg + r;
                bool ok = row_ok;
                if (need_mask) {
                    ok = ok && key < ke;
                    if (p.causal) ok = ok && key <= qi + coff;
                    if (p.window > 0) ok = ok && key > qi + coff - p.window;
                }
                float x = sc[b][r] * t.ks[b];
                if (BIAS) x = fmaf(t.bias[b][r], kLog2e, x);
                x = ok ? x : kNegInf;
                sc[b][r] = x;
                mx = fmaxf(mx, x);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > m_run)) {
            const float m_new = fmaxf(m_run, mx);
            const float corr = __builtin_amdgcn_exp2f(m_run - (m_new == kNegInf ? 0.f : m_new));
            m_run = m_new;
            l_run *= corr;
#pragma unroll
            for (int db = 0; db < DB; ++db) oacc[db] *= corr;
        }
        const float m_use = m_run == kNegInf ? 0.f : m_run;
#pragma unroll
        for (int pr = 0; pr < KB / 2; ++pr) {
            // P^T operand, slots j < 4: key 4 lg + j of block 2 pr, then of block 2 pr + 1
            u32x4_t hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int b = 2 * pr + (e >> 1), r = 2 * (e & 1);
                const float e0 = __builtin_amdgcn_exp2f(sc[b][r] - m_use), e1 = __builtin_amdgcn_exp2f(sc[b][r + 1] - m_use);
                l_run += e0 + e1;
                const float p0 = e0 * t.vs[b], p1 = e1 * t.vs[b];
                const uint32_t h = BF16::pack2(p0, p1);
                hi[e] = h;
                lo[e] = BF16::pack2(p0 - __uint_as_float(h << 16), p1 - __uint_as_float(h & 0xffff0000u));
            }
#pragma unroll
            for (int c4 = 0; c4 < CW / 4; ++c4) {
                uint32_t a[4], a2[4];
                transpose4x4b(t.v[2 * pr][0].word(c4), t.v[2 * pr][1].word(c4), t.v[2 * pr][2].word(c4),
                              t.v[2 * pr][3].word(c4), a);
                transpose4x4b(t.v[2 * pr + 1][0].word(c4), t.v[2 * pr + 1][1].word(c4), t.v[2 * pr + 1][2].word(c4),
                              t.v[2 * pr + 1][3].word(c4), a2);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const u32x2_t x = C::template unpack4<BF16>(a[c]), y = C::template unpack4<BF16>(a2[c]);
                    const u32x4_t va = u32x4_t{x[0], x[1], y[0], y[1]};
                    oacc[4 * c4 + c] = mfma16<BF16>(va, hi, oacc[4 * c4 + c]);
                    oacc[4 * c4 + c] = mfma16<BF16>(va, lo, oacc[4 * c4 + c]);
                }
            }
        }
    };

    // Two register sets alternate: tile i is computed while the loads of tile
    // i + 1 are in flight, then refilled with tile i + 2.
    Tile8<D, KB> ta, tb;
    if (n_my > 0) load(0, ta);
    if (n_my > 1) load(1, tb);
    for (int i = 0; i < n_my; i += 2) {
        step(i, ta);
        if (i + 2 < n_my) load(i + 2, ta);
        if (i + 1 < n_my) {
            step(i + 1, tb);
            if (i + 3 < n_my) load(i + 3, tb);
        }
    }

    // the wave's rows to LDS: operand row 4 lg + r of oacc[db] is column
    // CW (4 lg + r) + db
    float lt = l_run + __shfl_xor(l_run, 16);
    lt += __shfl_xor(lt, 32);
    char* ow = smem + w * 16 * OROW;
    if (row_ok) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c4 = 0; c4 < CW / 4; ++c4)
                *reinterpret_cast<f32x4_t*>(ow + n16 * OROW + (CW * (4 * lg + r) + 4 * c4) * 4) =
                    f32x4_t{oacc[4 * c4][r], oacc[4 * c4 + 1][r], oacc[4 * c4 + 2][r], oacc[4 * c4 + 3][r]};
        if (lg == 0) {
            ml[w * 16 + n16] = m_run;
            ml[(NW + w) * 16 + n16] = lt;
        }
    }
    __syncthreads();
    const bool whole = p.chunk == 0 && p.ns == 1;
    // one thread per row and 4 columns
    for (int u = threadIdx.x; u < rows * (D / 4); u += NW * 64) {
        const int n = u / (D / 4), d = 4 * (u - n * (D / 4));
        float m = kNegInf;
#pragma unroll
        for (int i = 0; i < NW; ++i) m = nan_max(ml[i * 16 + n], m);
        const float m_use = m == kNegInf ? 0.f : m;
        float l = 0.f;
        f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const float wgt = __builtin_amdgcn_exp2f(ml[i * 16 + n] - m_use);
            l += wgt * ml[(NW + i) * 16 + n];
            o += wgt * *reinterpret_cast<const f32x4_t*>(smem + i * 16 * OROW + n * OROW + d * 4);
        }
        o *= !(l <= 0.f) ? 1.f / l : 0.f;
        const float lse = !(l <= 0.f) ? m * kLn2 + logf(l) : kNegInf;
        if (whole) {
            const int h2 = n / q_len;
            const int64_t rh = (int64_t)(qr.start + n - h2 * q_len) * p.hq + hk * p.g + hgi * p.hpb + h2;
            st8(out + rh * D + d, u32x2_t{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])});
            if (lse_out != nullptr && d == 0) lse_out[rh] = lse;
        } else {
            const int64_t prow = ((int64_t)(hk * p.n_hg + hgi) * p.n_slots + slot) * 16 + n;
            *reinterpret_cast<f32x4_t*>(p.o_part + prow * D + d) = o;
            if (d == 0) p.lse_part[prow] = lse;
        }
    }
    // rows past the 16 that max_seqlen_q promised: NaN (the combine's, else)
    if (whole) {
        const int more = p.hpb * q_len - 16;
        for (int64_t u = threadIdx.x; u < (int64_t)more * D; u += NW * 64) {
            const int n = 16 + (int)(u / D), d = (int)(u % D), h2 = n / q_len;
            const int64_t rh = (int64_t)(qr.start + n - h2 * q_len) * p.hq + hk * p.g + hgi * p.hpb + h2;
            out[rh * D + d] = T::from_float(__builtin_nanf(""));
            if (lse_out != nullptr && d == 0) lse_out[rh] = __builtin_nanf("");
        }
    }
}

template <typename T, typename C, int D, int NW>
hipError_t launch_nw(const DecodeArgs& a, const DecKParams& p, unsigned items, hipStream_t st) {
    const dim3 grid(items), block(NW * 64);
    typename T::raw* out = (typename T::raw*)a.o;
    if (p.bias != nullptr) hipLaunchKernelGGL((decode8_kernel<T, C, D, true, NW, 32>), grid, block, 0, st, p, out, a.lse);
    else hipLaunchKernelGGL((decode8_kernel<T, C, D, false, NW, 32>), grid, block, 0, st, p, out, a.lse);
    return hipGetLastError();
}

template <typename T, typename C, int D>
hipError_t launch_typed(const DecodeArgs& a, hipStream_t st) {
    DecKParams p;
    if (!fill_decode_params(a, p)) return hipErrorInvalidValue;
    const int64_t items = (int64_t)p.hkv * p.n_hg * p.n_slots;
    if (items > 0x7fffffff) return hipErrorInvalidValue;
    hipError_t e = hipSuccess;
    if (items > 0) {
        e = a.wg == 8 ? launch_nw<T, C, D, 8>(a, p, (unsigned)items, st) : launch_nw<T, C, D, 4>(a, p, (unsigned)items, st);
        if (e != hipSuccess || (p.chunk == 0 && p.ns == 1)) return e;
    }
    const int64_t rh = p.total_q * p.hq;
    if (rh > 0)
        hipLaunchKernelGGL((decode_combine_kernel<T, true>), dim3((unsigned)((rh + 3) / 4)), dim3(256), 0, st, p,
                           (typename T::raw*)a.o, a.lse, D);
    return hipGetLastError();
}

template <typename T, typename C>
hipError_t launch_dim(const DecodeArgs& a, hipStream_t st) {
    if (a.geo.d == 128) return launch_typed<T, C, 128>(a, st);
    if (a.geo.d == 64) return launch_typed<T, C, 64>(a, st);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_decode8(int dtype, int code, const DecodeArgs& a, hipStream_t st) {
    if (a.block_table == nullptr || a.k_scale == nullptr || a.v_scale == nullptr || a.block < 16) return hipErrorInvalidValue;
    const bool e4m3 = code == MTLATTN_CODE_E4M3;
    if (dtype == MTLATTN_DTYPE_BF16) return e4m3 ? launch_dim<BF16, E4M3>(a, st) : launch_dim<BF16, I8>(a, st);
    if (dtype == MTLATTN_DTYPE_F16) return e4m3 ? launch_dim<F16, E4M3>(a, st) : launch_dim<F16, I8>(a, st);
    return hipErrorInvalidValue;
}

}  // namespace mtlattn
