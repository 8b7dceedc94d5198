// Work items of the decode kernels and the combine that merges their partials,
// shared by the 16-bit (decode.hip) and the 8-bit (decode8.hip) caches.
#pragma once

#include "common.h"
#include "kernels.h"

namespace mtlattn {

namespace {

constexpr int kDecKT = 32;      // keys per tile

// Work items: chunk > 0 -> fixed KV chunks, slot = cu_kv[s] / chunk + s + c
// (n_slots = total_kv / chunk + num_seqs + 1); chunk == 0 -> ns equal splits
// per sequence, slot = s * ns + split (n_slots = num_seqs * ns). Partials of
// item `slot` for kv head hk and head group hgi live at row
// ((hk * n_hg + hgi) * n_slots + slot) * 16 + n (n = 16-row group row).
struct DecKParams {
    const uint16_t* q; const uint16_t* k; const uint16_t* v;
    float* o_part; float* lse_part;
    const int* cu_q; const int* cu_kv;
    const float* bias;
    int64_t q_rs, k_rs, v_rs;
    int64_t bias_qs, bias_hs, bias_cols, bias_ss, bias_rows;
    int64_t total_q, total_kv;
    int num_seqs, hq, hkv, g, hpb, n_hg, ns, chunk, n_slots;
    float scale_log2;
    int causal, window;
    int bias_v4;      // bias rows 16-byte aligned (pointer and strides)
    // paged KV (PAGED kernels): block table rows of bt_stride page indices
    const int* block_table;
    int64_t bt_stride;
    int page_size, num_pages;
    // 8-bit caches: an fp32 scale per (block of tokens, kv head), in cache order
    const float* k_scale; const float* v_scale;
    int block;
};

// KV range [ks, ke) of work item `slot` of sequence s (false: no keys).
__device__ inline bool item_range(const DecKParams& p, int slot, int& s, int& ks, int& ke) {
    int kv_len;
    if (p.chunk > 0) {
        s = find_seq_for_tile(p.cu_kv, p.num_seqs, p.chunk, slot, p.total_kv);
        const SeqRange kr = seq_range(p.cu_kv, s, p.total_kv);
        kv_len = kr.end - kr.start;
        ks = (slot - tile_base(p.cu_kv, s, p.chunk, p.total_kv)) * p.chunk;
        ke = min(kv_len, ks + p.chunk);
    } else {
        s = slot / p.ns;
        const int split = slot - s * p.ns;
        const SeqRange kr = seq_range(p.cu_kv, s, p.total_kv);
        kv_len = kr.end - kr.start;
        // with a window, split only the keys the sequence's rows can see
        int lo = 0;
        if (p.window > 0) {
            const SeqRange qr = seq_range(p.cu_q, s, p.total_q);
            lo = max(0, kv_len - (qr.end - qr.start) - p.window + 1) / kDecKT * kDecKT;
        }
        int c = (kv_len - lo + p.ns - 1) / p.ns;
        c = (c + kDecKT - 1) / kDecKT * kDecKT;
        ks = lo + split * c;
        ke = min(kv_len, ks + c);
    }
    return ke > ks;
}

// Kernel parameters of a decode call; false: sizes that the kernels do not take.
inline bool fill_decode_params(const DecodeArgs& a, DecKParams& p) {
    const Geometry& g = a.geo;
    p.q = (const uint16_t*)a.q; p.k = (const uint16_t*)a.k; p.v = (const uint16_t*)a.v;
    p.o_part = a.o_part; p.lse_part = a.lse_part;
    p.cu_q = g.cu_q; p.cu_kv = g.cu_kv;
    p.bias = g.bias; p.bias_qs = g.bias_qs; p.bias_hs = g.bias_hs; p.bias_cols = g.bias_cols;
    p.bias_ss = g.bias_ss; p.bias_rows = g.bias_rows;
    p.q_rs = a.q_rs; p.k_rs = a.k_rs; p.v_rs = a.v_rs;
    p.total_q = g.total_q; p.total_kv = g.total_kv;
    p.num_seqs = g.num_seqs; p.hq = g.hq; p.hkv = g.hkv; p.g = g.g;
    const int mq = a.max_q > 0 ? a.max_q : 1;
    int hpb = 16 / mq;                  // heads per 16-row group: largest divisor of g that fits
    if (hpb < 1) return false;
    if (hpb > g.g) hpb = g.g;
    while (g.g % hpb != 0) --hpb;
    p.hpb = hpb;
    p.n_hg = g.g / hpb;
    p.ns = a.num_splits;
    p.chunk = a.chunk;
    const int64_t slots = a.chunk > 0 ? g.total_kv / a.chunk + g.num_seqs + 1 : (int64_t)g.num_seqs * a.num_splits;
    if (slots > 0x3fffffff) return false;
    p.n_slots = (int)slots;
    p.scale_log2 = g.scale * kLog2e;
    p.causal = g.causal;
    p.window = g.window;
    p.bias_v4 = g.bias != nullptr && ((uintptr_t)g.bias % 16 == 0) && g.bias_qs % 4 == 0 && g.bias_hs % 4 == 0 &&
                (g.bias_ss < 0 || g.bias_ss % 4 == 0);
    p.block_table = a.block_table;
    p.bt_stride = a.bt_stride;
    p.page_size = a.page_size;
    p.num_pages = a.num_pages;
    p.k_scale = a.k_scale;
    p.v_scale = a.v_scale;
    p.block = a.block;
    return true;
}

// One wave per (row, head): O = sum_i w_i O_i / sum_i w_i over the work items
// of the row's sequence, w_i = exp(lse_i - max lse). Rows outside every
// sequence are left untouched as the flash forward leaves them; rows beyond
// the 16-row group (max_seqlen_q too small) are extra_rows', and untouched
// after the one-wave kernel; with FILL they are NaN.
template <typename T, bool FILL = false>
__global__ __launch_bounds__(256) void decode_combine_kernel(DecKParams p, typename T::raw* __restrict__ out,
                                                             float* __restrict__ lse_out, int d) {
    const int64_t rh = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (rh >= p.total_q * p.hq) return;
    const int64_t row = rh / p.hq;
    const int head = (int)(rh - row * p.hq);
    // sequence of this row (largest s with cu_q[s] <= row)
    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu_q[mid] <= row) lo = mid; else hi = mid - 1;
    }
    const int s = lo;
    const SeqRange qr = seq_range(p.cu_q, s, p.total_q);
    if (row < qr.start || row >= qr.end) return;
    const int q_len = qr.end - qr.start, qi = (int)(row - qr.start);
    const int hk = head / p.g, hh_full = head - hk * p.g;
    const int hgi = hh_full / p.hpb, n = (hh_full - hgi * p.hpb) * q_len + qi;
    if (n >= 16) {
        if (FILL) {
            for (int dd = lane; dd < d; dd += 64) out[rh * d + dd] = T::from_float(__builtin_nanf(""));
            if (lse_out != nullptr && lane == 0) lse_out[rh] = __builtin_nanf("");
        }
        return;
    }
    const SeqRange kr = seq_range(p.cu_kv, s, p.total_kv);
    const int kv_len = kr.end - kr.start;
    int first, count;
    if (p.chunk > 0) {
        first = tile_base(p.cu_kv, s, p.chunk, p.total_kv);
        count = (kv_len + p.chunk - 1) / p.chunk;
    } else {
        first = s * p.ns;
        count = p.ns;
    }
    const int64_t base = (int64_t)(hk * p.n_hg + hgi) * p.n_slots;
    // max LSE: lanes over items, then across the wave
    float m = kNegInf;
    // (NaN-preserving: a NaN logit makes its item's LSE NaN, and a row whose
    // items are all NaN must not look empty)
    for (int i = lane; i < count; i += 64) m = nan_max(p.lse_part[(base + first + i) * 16 + n], m);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = nan_max(m, __shfl_xor(m, off));
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    float wsum = 0.f;
    if (m != kNegInf) {
        // items in groups of 4 whose loads all go out before the first use;
        // the sums still run in item order
        constexpr int U = 4;
        for (int i0 = 0; i0 < count; i0 += U) {
            float l[U], o[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = i0 + u < count;
                const int64_t prow = (base + first + min(i0 + u, count - 1)) * 16 + n;
                l[u] = in ? p.lse_part[prow] : kNegInf;
                const float* op = p.o_part + prow * d;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int dd = lane + 64 * j;
                    o[u][j] = dd < d ? op[dd] : 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (l[u] == kNegInf) continue;
                const float wgt = __expf(l[u] - m);
                wsum += wgt;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (lane + 64 * j < d) acc[j] += wgt * o[u][j];
            }
        }
    }
    const float inv = !(wsum <= 0.f) ? 1.f / wsum : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int dd = lane + 64 * j;
        if (dd < d) out[rh * d + dd] = T::from_float(acc[j] * inv);
    }
    if (lse_out != nullptr && lane == 0) lse_out[rh] = !(wsum <= 0.f) ? m + logf(wsum) : kNegInf;
}

}  // namespace

}  // namespace mtlattn
