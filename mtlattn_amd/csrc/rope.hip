// Position rotation of queries and keys, with their per-head norms in the same
// pass, forward and backward, and on the way into a paged K/V cache; no counterpart
// in the reference.
//
//   xh = x r w,  r = 1 / sqrt(mean(x^2) + eps)             (a norm; else xh = x)
//   y_a = s (a cos t - b sin t),  y_b = s (b cos t + a sin t),  t = position * f_i
// for the pairs (a, b) = (xh_i, xh_{i + R/2}), or (xh_2i, xh_{2i+1}) interleaved,
// i < R / 2; elements from R on pass. Backward: g, the rotation of dy by -t, and
//   dx = r (w g - xn mean(w g xn)),  dw = sum over rows of g xn,  xn = x r.
//
// All of it is bound by HBM: a value read, a value written (bf16, 32/8 heads, D = 128: 32768
// tokens 116 us, 5.8 TB/s; 16384 with norms 66-72 us, 4.7-5.1, their backward 92-101, 5.0-5.5;
// 16384 appended with norms 75 us, 5.3; a step of 16 tokens 3 us, its launch). Angles are formed in
// 64 bits (in turns, so that the reduction is exact; positions reach millions) and
// their cosines and sines in 32, once per token and frequency: a wave takes one
// token, a lane one frequency of it, and the heads of the token share them through
// LDS. A table in memory would cost what a head of the row does.
#include "common.h"
#include "kernels.h"
#include "../../include/mtlattn_capi.h"

namespace mtlattn {

namespace {

constexpr int kMaxD = 256;
constexpr int kWaves = 4;

struct RopeKParams {
    // q, k and (append) v: rows in, rows out. Backward: in = the gradients of the
    // rotated rows, x = the rows themselves
    const void* in[3]; int64_t in_rs[3];
    void* out[3]; int64_t out_rs[3];
    const void* x[2]; int64_t x_rs[2];
    const void* weight[2];
    int w_code;                         // element type of the weights
    const int* positions; const float* inv_freq;
    float scale, eps, inv_d, sign;      // sign: -1 rotates back
    int interleaved, norm;
    int hq, hkv, heads, d, rot;
    int64_t total, wg0;                 // rows; forward: workgroups of the launches before this one
    int units_log2, slices;             // lanes of a head (log2), waves that share a token's heads
    // append: the cache rows of k and v
    const int* cu; const int* cu_kv; const int* block_table;
    int64_t bt_stride;
    int num_seqs, page_size, num_pages;
    float* part;                        // backward: [workgroups][2][d] sums of the weights' gradients
};

// cos and sin of position * f, times scale. In turns the reduction to an eighth is
// exact in 64 bits but for the product's rounding (2^-27 turns at a position of
// 2^24); the series of the mathematics on [-pi/4, pi/4], to x^10 and x^9, are within
// 2e-9 there.
__device__ inline void turn(int pos, float f, float scale, float sign, float& c, float& s) {
    double t = (double)pos * ((double)f * 0.15915494309189533577);
    t -= __builtin_rint(t);
    const double q = __builtin_rint(4. * t);
    const float x = (float)((t - 0.25 * q) * 6.28318530717958647693), x2 = x * x;
    const float sn =
        fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), x);
    const float cs = fmaf(
        x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
    const int k = (int)q & 3;
    const float a = (k & 1) != 0 ? sn : cs, b = (k & 1) != 0 ? cs : sn;
    c = ((k + 1) & 2) != 0 ? -a : a;                  // quadrants 1 and 2
    s = (k & 2) != 0 ? -b : b;                        // quadrants 2 and 3
    c *= scale;
    s *= scale * sign;
}

// Eight neighbouring values of a row, as they are stored. FAR: past the caches, which
// keep what they hold (values that nothing reads again soon).
template <typename T>
struct Row8 {
    u32x4_t x;
    template <bool FAR = false>
    __device__ inline void load(const typename T::raw* p) {
        x = FAR ? __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p)) : ld16(p);
    }
    template <bool FAR = false>
    __device__ inline void store(typename T::raw* p) const {
        if (FAR) __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t*>(p));
        else st16(p, x);
    }
    __device__ inline void get(float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = lo16<T>(x[i]);
            f[2 * i + 1] = hi16<T>(x[i]);
        }
    }
    __device__ inline void set(const float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = T::pack2(f[2 * i], f[2 * i + 1]);
    }
    __device__ inline void clear() { x = u32x4_t{0u, 0u, 0u, 0u}; }
};
template <>
struct Row8<F32> {
    f32x4_t x, y;
    template <bool FAR = false>
    __device__ inline void load(const float* p) {
        const f32x4_t* f = reinterpret_cast<const f32x4_t*>(p);
        x = FAR ? __builtin_nontemporal_load(f) : f[0];
        y = FAR ? __builtin_nontemporal_load(f + 1) : f[1];
    }
    template <bool FAR = false>
    __device__ inline void store(float* p) const {
        f32x4_t* f = reinterpret_cast<f32x4_t*>(p);
        if (FAR) {
            __builtin_nontemporal_store(x, f);
            __builtin_nontemporal_store(y, f + 1);
        } else {
            f[0] = x;
            f[1] = y;
        }
    }
    __device__ inline void get(float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = x[i];
            f[4 + i] = y[i];
        }
    }
    __device__ inline void set(const float* f) {
        x = f32x4_t{f[0], f[1], f[2], f[3]};
        y = f32x4_t{f[4], f[5], f[6], f[7]};
    }
    __device__ inline void clear() { x = y = f32x4_t{0.f, 0.f, 0.f, 0.f}; }
};

__device__ inline float weight_at(const RopeKParams& p, int side, int i) {
    if (p.w_code == F32::code) return ((const float*)p.weight[side])[i];
    const uint16_t raw = ((const uint16_t*)p.weight[side])[i];
    return p.w_code == BF16::code ? BF16::to_float(raw) : F16::to_float(raw);
}

// Where a row of an append goes.
struct Place {
    bool owned;         // a sequence has the row
    int pos;            // its place in that sequence (negative: more rows than tokens)
    int64_t row;        // the cache row, -1: none
};
// Among the sequences by 64 offsets at a time, one per lane (an empty sequence's
// offset is the next one's: the last of equals owns the row).
__device__ inline Place find_place(const RopeKParams& p, int row, int lane) {
    int lo = 0, n = p.num_seqs;                        // the answer is in [lo, lo + n)
    while (n > 64) {
        const int step = (n + 63) / 64, i = min(lane * step, n - 1);
        const uint64_t le = __ballot(lane * step < n && p.cu[lo + i] <= row);
        const int l = le != 0 ? 63 - __builtin_clzll(le) : 0;
        lo += l * step;
        n = min(step, n - l * step);
    }
    const uint64_t le = __ballot(lane < n && p.cu[lo + min(lane, n - 1)] <= row);
    const int s = lo + (le != 0 ? 63 - __builtin_clzll(le) : 0);
    const SeqRange r = seq_range(p.cu, s, p.total);
    Place out{row >= r.start && row < r.end, 0, -1};
    if (!out.owned) return out;
    out.pos = kv_length(p.cu_kv, s) - (r.end - row);
    if (out.pos < 0) return out;
    const int col = out.pos / p.page_size;
    const int pg = col < p.bt_stride ? p.block_table[(int64_t)s * p.bt_stride + col] : -1;
    if (pg >= 0 && pg < p.num_pages) out.row = (int64_t)pg * p.page_size + (out.pos - col * p.page_size);
    return out;
}

// The two 8-element chunks of unit u of a head: halves of 8 pairs, or what passes.
template <bool INTER>
__device__ inline void unit_chunks(int u, int rot, int& a, int& b) {
    if (INTER || 16 * u >= rot) {
        a = 16 * u;
        b = a + 8;
    } else {
        a = 8 * u;
        b = a + rot / 2;
    }
}

// Rotates the 8 pairs that va and vb (a unit's chunks) hold.
template <bool INTER>
__device__ inline void rotate(float* va, float* vb, const float* cs, const float* sn) {
    if (INTER) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float* v = (i < 4 ? va : vb) + 2 * (i & 3);
            const float a = v[0], b = v[1];
            v[0] = fmaf(a, cs[i], -b * sn[i]);
            v[1] = fmaf(b, cs[i], a * sn[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = va[i], b = vb[i];
            va[i] = fmaf(a, cs[i], -b * sn[i]);
            vb[i] = fmaf(b, cs[i], a * sn[i]);
        }
    }
}

// A wave's table of cos and sin, a lane per frequency, and its lane's eight of each.
__device__ inline void wave_table(const RopeKParams& p, float* tab, int pos, int lane) {
    for (int i = lane; i < p.rot / 2; i += 64) turn(pos, p.inv_freq[i], p.scale, p.sign, tab[i], tab[kMaxD / 2 + i]);
    __builtin_amdgcn_wave_barrier();
}
__device__ inline void table_of(const float* tab, int u, int rot, float* cs, float* sn) {
    const float* t = tab + (16 * u < rot ? 8 * u : 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x4_t c = *reinterpret_cast<const f32x4_t*>(t + 4 * i);
        const f32x4_t s = *reinterpret_cast<const f32x4_t*>(t + kMaxD / 2 + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            cs[4 * i + j] = c[j];
            sn[4 * i + j] = s[j];
        }
    }
}

// Forward (and, without norms, backward: sign = -1), or an append. D and R are
// multiples of 16, rows 16-byte aligned. A lane holds 16 values of a head (its
// unit: both members of 8 pairs), 2^units_log2 lanes a head; a wave takes PP passes
// over its token's heads, whose loads are all under way before the angles. An append's
// rows go past the caches both ways (32 sequences of 1024 new tokens 155 -> 142 us, with a
// paged decode of them 180 -> 170; 16 of 512 41 -> 38, 50 -> 52). A rotation's are left in
// them, for the attention (32768 tokens 118 -> 110 us past them, but with the attention
// 407 -> 412), and come past them where FAR_IN says so (past_caches), but with
// norms, whose rows the backward reads again.
template <typename T, bool INTER, bool NORM, bool APPEND, int PP, bool FAR_IN>
__global__ __launch_bounds__(kWaves * 64) void rope_kernel(RopeKParams p) {
    __shared__ __attribute__((aligned(16))) float s_tab[kWaves][kMaxD];
    __shared__ __attribute__((aligned(16))) float s_w[NORM ? 2 * kMaxD : 4];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t item = (p.wg0 + blockIdx.x) * kWaves + w;
    const int64_t tok = item / p.slices;
    const bool active = tok < p.total;
    const int64_t token = active ? tok : p.total - 1;
    const int pass0 = (int)(item - tok * p.slices) * PP;
    const int u = lane & ((1 << p.units_log2) - 1), hl = lane >> p.units_log2, hpw = 64 >> p.units_log2;
    const bool unit = 16 * u < p.d;
    int ea, eb;
    unit_chunks<INTER>(u, p.rot, ea, eb);
    const bool turns = 16 * u < p.rot;

    Row8<T> xa[PP], xb[PP];
    int part[PP], hd[PP];
#pragma unroll
    for (int i = 0; i < PP; ++i) {
        const int head = (pass0 + i) * hpw + hl;
        part[i] = head < p.hq ? 0 : head < p.hq + p.hkv ? 1 : 2;
        hd[i] = head - (part[i] == 0 ? 0 : part[i] == 1 ? p.hq : p.hq + p.hkv);
        xa[i].clear();
        xb[i].clear();
        if (head >= p.heads || !unit || !active) {
            part[i] = -1;
            continue;
        }
        const typename T::raw* x =
            (const typename T::raw*)p.in[part[i]] + token * p.in_rs[part[i]] + (int64_t)hd[i] * p.d;
        xa[i].template load<FAR_IN>(x + ea);
        xb[i].template load<FAR_IN>(x + eb);
    }
    Place at{true, 0, 0};
    if (APPEND) at = find_place(p, (int)token, lane);
    if (NORM) {
        for (int i = threadIdx.x; i < 2 * p.d; i += kWaves * 64) {
            const int side = i >= p.d ? 1 : 0;
            s_w[side * kMaxD + i - side * p.d] = p.weight[side] != nullptr ? weight_at(p, side, i - side * p.d) : 0.f;
        }
    }
    float cs[8], sn[8];
    if (p.rot > 0) {
        wave_table(p, s_tab[w], p.positions != nullptr ? p.positions[token] : at.pos, lane);
        table_of(s_tab[w], u, p.rot, cs, sn);
    }
    if (NORM) __syncthreads();
#pragma unroll
    for (int i = 0; i < PP; ++i) {
        if (NORM || !APPEND || part[i] != 2) {
            float va[8], vb[8];
            xa[i].get(va);
            xb[i].get(vb);
            if (NORM) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) sum = fmaf(va[j], va[j], fmaf(vb[j], vb[j], sum));
                for (int o = 1; o < 1 << p.units_log2; o <<= 1) sum += __shfl_xor(sum, o);
                const float r = 1.f / sqrtf(fmaf(sum, p.inv_d, p.eps));
                const float* wt = s_w + (part[i] == 0 ? 0 : kMaxD);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    va[j] *= r * wt[(unit ? ea : 0) + j];
                    vb[j] *= r * wt[(unit ? eb : 0) + j];
                }
            }
            if (turns) rotate<INTER>(va, vb, cs, sn);
            if (part[i] != 2 && (NORM || turns)) {
                xa[i].set(va);
                xb[i].set(vb);
            }
        }
        if (part[i] < 0) continue;
        int64_t row = token;
        if (APPEND) {
            if (part[i] > 0) row = at.row;
            if (row < 0) continue;
            if (part[i] == 0 && !at.owned) {
                xa[i].clear();
                xb[i].clear();
            }
        }
        typename T::raw* y = (typename T::raw*)p.out[part[i]] + row * p.out_rs[part[i]] + (int64_t)hd[i] * p.d;
        xa[i].template store<APPEND>(y + ea);
        xb[i].template store<APPEND>(y + eb);
    }
}

// The sums of a workgroup's waves, in their order: acc holds, per lane, what its elements
// of the weights' gradients are (e(j): the element of value j, -1: none).
template <int N, typename E>
__device__ inline void store_part(const RopeKParams& p, float (*s_sum)[2][kMaxD], const float (&acc)[2][N], E e, bool first,
                                  int w) {
    if (first) {
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (e(j) >= 0) s_sum[w][side][e(j)] = acc[side][j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.d; i += kWaves * 64) {
        const int side = i >= p.d ? 1 : 0;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) sum += s_sum[k][side][i - side * p.d];
        p.part[(int64_t)blockIdx.x * 2 * p.d + i] = sum;
    }
}

// Backward with norms, on the same units: dy and x in, dx out. A wave goes through
// every (workgroups * kWaves)-th token, the passes over its query heads, then over its
// kv heads, the next pass's rows under way meanwhile (the next two: 120 us against 112);
// its share of dw stays in registers, and one more launch adds the workgroups' sums (no
// atomics: the same result every time). With few tokens the waves of a token share its
// passes. Rows of 16 bits come and go past the caches (16384 tokens of 32/8 heads, D = 128: 104
// -> 92 us, all displaced 112 -> 100; 2048: 21 -> 24, displaced 30 -> 23; 16384 of 16/16, D = 64:
// 47 -> 49, 56 -> 51); those of fp32 do not, whose neighbouring 16 bytes are two loads, so that
// a line would come twice (16384 of 16/16, D = 80: 176 us past them, 117 not). All lane moves
// of dw's sums are under way together (one value's after another's: 4 us more at every size).
template <typename T, bool INTER>
__global__ __launch_bounds__(kWaves * 64) void rope_bwd_kernel(RopeKParams p) {
    constexpr bool FAR = T::code != F32::code;
    __shared__ __attribute__((aligned(16))) float s_tab[kWaves][kMaxD];
    __shared__ __attribute__((aligned(16))) float s_w[2 * kMaxD];
    __shared__ float s_sum[kWaves][2][kMaxD];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int u = lane & ((1 << p.units_log2) - 1), hl = lane >> p.units_log2, hpw = 64 >> p.units_log2;
    const bool unit = 16 * u < p.d, turns = 16 * u < p.rot;
    int ea, eb;
    unit_chunks<INTER>(u, p.rot, ea, eb);
    const int q_passes = (p.hq + hpw - 1) / hpw, passes = q_passes + (p.hkv + hpw - 1) / hpw;
    struct Rows {
        Row8<T> ga, gb, xa, xb;
    };
    auto head_of = [&](int pass) { return (pass < q_passes ? pass : pass - q_passes) * hpw + hl; };
    auto load = [&](int64_t token, int pass, Rows& r) {
        const int side = pass < q_passes ? 0 : 1, hd = head_of(pass);
        r.ga.clear(); r.gb.clear(); r.xa.clear(); r.xb.clear();
        if (unit && hd < (side == 0 ? p.hq : p.hkv)) {
            const typename T::raw* g = (const typename T::raw*)p.in[side] + token * p.in_rs[side] + (int64_t)hd * p.d;
            const typename T::raw* x = (const typename T::raw*)p.x[side] + token * p.x_rs[side] + (int64_t)hd * p.d;
            r.ga.template load<FAR>(g + ea);
            r.gb.template load<FAR>(g + eb);
            r.xa.template load<FAR>(x + ea);
            r.xb.template load<FAR>(x + eb);
        }
    };
    float dw[2][16] = {};
    const int64_t wave = (int64_t)blockIdx.x * kWaves + w, step = (int64_t)gridDim.x * kWaves / p.slices;
    const int slice = (int)(wave % p.slices), first = slice * passes / p.slices, end = (slice + 1) * passes / p.slices;
    int64_t token = wave / p.slices;
    Rows now;
    int pos = 0;
    if (token < p.total) {
        load(token, first, now);
        if (p.rot > 0) pos = p.positions[token];
    }
    for (int i = threadIdx.x; i < 2 * p.d; i += kWaves * 64) {
        const int side = i >= p.d ? 1 : 0;
        s_w[side * kMaxD + i - side * p.d] = weight_at(p, side, i - side * p.d);
    }
    __syncthreads();
    while (token < p.total) {
        float cs[8], sn[8];
        if (p.rot > 0) {
            __builtin_amdgcn_wave_barrier();
            wave_table(p, s_tab[w], pos, lane);
            table_of(s_tab[w], u, p.rot, cs, sn);
            pos = p.positions[min(token + step, p.total - 1)];
        }
#pragma unroll 1
        for (int pass = first; pass < end; ++pass) {
            const bool last = pass + 1 == end;
            const int64_t next = last ? token + step : token;
            Rows then;
            if (next < p.total) load(next, last ? first : pass + 1, then);
            const int side = pass < q_passes ? 0 : 1, hd = head_of(pass);
            float va[8], vb[8], fa[8], fb[8];
            now.ga.get(va);
            now.gb.get(vb);
            now.xa.get(fa);
            now.xb.get(fb);
            if (turns) rotate<INTER>(va, vb, cs, sn);
            const float* wt = s_w + side * kMaxD;
            float sum = 0.f, dot = 0.f;
            float wa[8], wb[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                wa[j] = wt[(unit ? ea : 0) + j];
                wb[j] = wt[(unit ? eb : 0) + j];
                sum = fmaf(fa[j], fa[j], fmaf(fb[j], fb[j], sum));
                dot = fmaf(va[j] * wa[j], fa[j], fmaf(vb[j] * wb[j], fb[j], dot));
            }
            for (int o = 1; o < 1 << p.units_log2; o <<= 1) {
                sum += __shfl_xor(sum, o);
                dot += __shfl_xor(dot, o);
            }
            // (lanes without a head hold zeros: their r could be infinite, and the sums of dw take
            // every lane)
            const bool there = unit && hd < (side == 0 ? p.hq : p.hkv);
            const float r = there ? 1.f / sqrtf(fmaf(sum, p.inv_d, p.eps)) : 0.f;
            const float m = dot * r * p.inv_d * r;                     // mean(w g xn) r
            auto add = [&](float (&d)[16]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    d[j] = fmaf(va[j], fa[j] * r, d[j]);
                    d[8 + j] = fmaf(vb[j], fb[j] * r, d[8 + j]);
                }
            };
            if (side == 0) add(dw[0]);
            else add(dw[1]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                va[j] = r * fmaf(va[j], wa[j], -fa[j] * m);
                vb[j] = r * fmaf(vb[j], wb[j], -fb[j] * m);
            }
            if (there) {
                now.ga.set(va);
                now.gb.set(vb);
                typename T::raw* y = (typename T::raw*)p.out[side] + token * p.out_rs[side] + (int64_t)hd * p.d;
                now.ga.template store<FAR>(y + ea);
                now.gb.template store<FAR>(y + eb);
            }
            now = then;
        }
        token += step;
    }
    for (int o = 1 << p.units_log2; o < 64; o <<= 1)   // (all values' moves under way together)
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int j = 0; j < 16; ++j) dw[side][j] += __shfl_xor(dw[side][j], o);
    store_part<16>(p, s_sum, dw, [&](int j) { return unit ? (j < 8 ? ea + j : eb + j - 8) : -1; }, hl == 0, w);
}

// Any D up to 256, any even R, rows of any alignment: a wave takes kAnyHeads heads of a
// token, one after the other, a lane per pair or passing element, one element at a time;
// the angles of the lane's pairs once per token. About a third of the other kernel's
// rate (16384 tokens of 32/8 heads, D = 128, bf16: 194 us, with norms 250, their backward
// 379; on aligned rows 58, 75 and 98).
constexpr int kAnyHeads = 8;
template <typename T, bool BWD>
__global__ __launch_bounds__(kWaves * 64, BWD ? 5 : 1) void rope_any_kernel(RopeKParams p, bool append) {
    constexpr int NS = kMaxD / 64;                     // slots of a lane: pairs (the first NP at most), then single elements
    constexpr int NP = NS / 2;
    __shared__ float s_sum[kWaves][2][kMaxD];
    using raw = typename T::raw;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int pairs = p.rot / 2, slots = p.d - pairs, groups = (p.heads + kAnyHeads - 1) / kAnyHeads;
    int ia[NS], ib[NP];                                // elements of a slot (ib -1: a single one, ia -1: none)
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        const int t = lane + 64 * j;
        ia[j] = t >= slots ? -1 : t >= pairs ? t + pairs : p.interleaved ? 2 * t : t;
        if (j < NP) ib[j] = t >= pairs ? -1 : p.interleaved ? 2 * t + 1 : t + pairs;
    }
    float wa[2][NS] = {}, wb[2][NP] = {};
    if (p.norm) {
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                if (p.weight[side] == nullptr) continue;
                if (ia[j] >= 0) wa[side][j] = weight_at(p, side, ia[j]);
                if (j < NP && ib[j] >= 0) wb[side][j] = weight_at(p, side, ib[j]);
            }
    }
    float dw[2][NS + NP] = {};
    const int64_t step = (int64_t)gridDim.x * kWaves, items = p.total * groups;
    for (int64_t item = (int64_t)blockIdx.x * kWaves + w; item < items; item += step) {
        const int64_t token = item / groups;
        const int head0 = (int)(item - token * groups) * kAnyHeads, head1 = min(head0 + kAnyHeads, p.heads);
        Place at{true, 0, 0};
        if (append) at = find_place(p, (int)token, lane);
        float cs[NP], sn[NP];
        if (p.rot > 0) {
            const int pos = p.positions != nullptr ? p.positions[token] : at.pos;
#pragma unroll
            for (int j = 0; j < NP; ++j)
                if (ib[j] >= 0) turn(pos, p.inv_freq[lane + 64 * j], p.scale, p.sign, cs[j], sn[j]);
        }
#pragma unroll 2
        for (int head = head0; head < head1; ++head) {
            const int part = head < p.hq ? 0 : head < p.hq + p.hkv ? 1 : 2;
            const int hd = head - (part == 0 ? 0 : part == 1 ? p.hq : p.hq + p.hkv);
            const int64_t row = append && part > 0 ? at.row : token;
            if (row < 0) continue;
            const raw* in = (const raw*)p.in[part] + token * p.in_rs[part] + (int64_t)hd * p.d;
            raw* y = (raw*)p.out[part] + row * p.out_rs[part] + (int64_t)hd * p.d;
            const raw* xr = BWD ? (const raw*)p.x[part] + token * p.x_rs[part] + (int64_t)hd * p.d : nullptr;
            raw ra[NS] = {}, rb[NP] = {}, xa[NS] = {}, xb[NP] = {};
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                if (ia[j] >= 0) ra[j] = in[ia[j]];
                if (j < NP && ib[j] >= 0) rb[j] = in[ib[j]];
                if (BWD && ia[j] >= 0) xa[j] = xr[ia[j]];
                if (BWD && j < NP && ib[j] >= 0) xb[j] = xr[ib[j]];
            }
            if (part == 2 || !at.owned) {
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    if (ia[j] >= 0) y[ia[j]] = part == 2 ? ra[j] : raw(0);
                    if (j < NP && ib[j] >= 0) y[ib[j]] = part == 2 ? rb[j] : raw(0);
                }
                continue;
            }
            float va[NS], vb[NP], fa[NS], fb[NP], sum = 0.f, r = 1.f;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                va[j] = T::to_float(ra[j]);
                fa[j] = BWD ? T::to_float(xa[j]) : va[j];
                sum = fmaf(fa[j], fa[j], sum);
                if (j < NP) {
                    vb[j] = T::to_float(rb[j]);
                    fb[j] = BWD ? T::to_float(xb[j]) : vb[j];
                    sum = fmaf(fb[j], fb[j], sum);
                }
            }
            if (p.norm) r = 1.f / sqrtf(fmaf(wave_sum(sum), p.inv_d, p.eps));
            // (every path of a side in registers: the index is a constant)
            auto w_a = [&](int j) { return part == 0 ? wa[0][j] : wa[1][j]; };
            auto w_b = [&](int j) { return part == 0 ? wb[0][j] : wb[1][j]; };
            if (!BWD && p.norm) {
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    va[j] *= r * w_a(j);
                    if (j < NP) vb[j] *= r * w_b(j);
                }
            }
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (ib[j] < 0) continue;
                const float a = va[j], b = vb[j];
                va[j] = fmaf(a, cs[j], -b * sn[j]);
                vb[j] = fmaf(b, cs[j], a * sn[j]);
            }
            if (BWD) {
                float dot = 0.f;
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    dot = fmaf(va[j] * w_a(j), fa[j], dot);
                    if (j < NP) dot = fmaf(vb[j] * w_b(j), fb[j], dot);
                }
                const float m = wave_sum(dot) * r * p.inv_d * r;
                auto add = [&](float (&d)[NS + NP]) {
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        d[j] = fmaf(va[j], fa[j] * r, d[j]);
                        if (j < NP) d[NS + j] = fmaf(vb[j], fb[j] * r, d[NS + j]);
                    }
                };
                if (part == 0) add(dw[0]);
                else add(dw[1]);
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    va[j] = r * fmaf(va[j], w_a(j), -fa[j] * m);
                    if (j < NP) vb[j] = r * fmaf(vb[j], w_b(j), -fb[j] * m);
                }
            }
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                // (what passes without a norm keeps its bits)
                const bool pair = j < NP && ib[j] >= 0;
                if (ia[j] >= 0) y[ia[j]] = !pair && !p.norm ? ra[j] : T::from_float(va[j]);
                if (pair) y[ib[j]] = T::from_float(vb[j]);
            }
        }
    }
    if constexpr (BWD)
        store_part<NS + NP>(p, s_sum, dw, [&](int j) { return j < NS ? ia[j] : ib[j - NS]; }, true, w);
}

// dw: the workgroups' sums, in their order within 64 interleaved runs and then by
// halves, in 64 bits; 4 columns a workgroup, so that all loads are under way at once.
__global__ __launch_bounds__(256) void rope_dw_kernel(const float* part, int n, int d, int w_code, void* dq, void* dk) {
    __shared__ double s_sum[64][4];
    const int c = threadIdx.x & 3, run = threadIdx.x >> 2, i = blockIdx.x * 4 + c;
    double sum = 0.;
    if (i < 2 * d) {
#pragma unroll 8
        for (int g = run; g < n; g += 64) sum += (double)part[(int64_t)g * 2 * d + i];
    }
    s_sum[run][c] = sum;
    for (int h = 32; h > 0; h >>= 1) {
        __syncthreads();
        if (run < h) s_sum[run][c] += s_sum[run + h][c];
    }
    if (run != 0 || i >= 2 * d) return;
    const float x = (float)s_sum[0][c];
    void* out = i < d ? dq : dk;
    const int e = i < d ? i : i - d;
    if (out == nullptr) return;
    if (w_code == F32::code) ((float*)out)[e] = x;
    else ((uint16_t*)out)[e] = w_code == BF16::code ? BF16::from_float(x) : F16::from_float(x);
}

RopeKParams params(const RopeArgs& a) {
    RopeKParams p{};
    for (int i = 0; i < 3; ++i) {
        p.in[i] = a.in[i];
        p.in_rs[i] = a.in_rs[i];
        p.out[i] = a.out[i];
        p.out_rs[i] = a.out_rs[i];
    }
    for (int i = 0; i < 2; ++i) {
        p.x[i] = a.x[i];
        p.x_rs[i] = a.x_rs[i];
        p.weight[i] = a.weight[i];
    }
    p.w_code = a.w_dtype;
    p.positions = a.positions;
    p.inv_freq = a.inv_freq;
    p.scale = a.scale;
    p.eps = a.eps;
    p.inv_d = 1.f / (float)a.d;
    p.sign = a.backward ? -1.f : 1.f;
    p.interleaved = a.interleaved;
    p.norm = a.weight[0] != nullptr || a.weight[1] != nullptr;
    p.hq = a.hq;
    p.hkv = a.hkv;
    p.heads = a.hq + (a.append ? 2 : 1) * a.hkv;
    p.d = a.d;
    p.rot = a.rot;
    p.total = a.total;
    p.cu = a.cu;
    p.cu_kv = a.cu_kv;
    p.block_table = a.block_table;
    p.bt_stride = a.bt_stride;
    p.num_seqs = a.num_seqs;
    p.page_size = a.page_size;
    p.num_pages = a.num_pages;
    p.part = a.part;
    while (16 << p.units_log2 < a.d) ++p.units_log2;
    return p;
}

// Workgroups of the backward with norms, in one round: two per CU of the unit kernel, which its
// registers hold at every type, five of the other one. 32/8 heads, D = 128, us: 16384 tokens
// bf16 103, fp16 102, fp32 192; three per CU 98, 111, 210 (registers of bf16 alone hold those),
// four 108 in bf16; 4096 tokens bf16 33.6, fp16 34.3; three 34.5, 37.
int unit_part_wgs(int64_t total, int slices) {
    return (int)std::max<int64_t>(1, std::min<int64_t>((total * slices + kWaves - 1) / kWaves, 2 * (int64_t)device_cus()));
}
// Waves that share a token's passes: 2 or 4 where the workgroups above have the waves (16
// tokens of 32/8 heads, D = 128, bf16: 9.6 us with the sums, with one each 13.8; 512: 13.2
// and 15.2; 8 waves the same from 64 tokens on).
int bwd_slices(int64_t total) {
    const int64_t waves = 2 * (int64_t)device_cus() * kWaves;
    return 4 * total <= waves ? 4 : 2 * total <= waves ? 2 : 1;
}
int any_part_wgs(int64_t total, int heads) {
    const int64_t items = total * ((heads + kAnyHeads - 1) / kAnyHeads);
    return (int)std::max<int64_t>(1, std::min<int64_t>((items + kWaves - 1) / kWaves, 5 * (int64_t)device_cus()));
}

// Rows that the unit kernels take: 16-byte aligned, D and R multiples of 16.
bool whole_units(const RopeArgs& a, int es) {
    if (a.d % 16 != 0 || a.rot % 16 != 0) return false;
    for (int i = 0; i < (a.append ? 3 : 2); ++i) {
        if (i == 0 && a.hq == 0) continue;
        if ((uintptr_t)a.in[i] % 16 != 0 || (uintptr_t)a.out[i] % 16 != 0 || a.in_rs[i] * es % 16 != 0 ||
            a.out_rs[i] * es % 16 != 0)
            return false;
        if (i < 2 && a.x[i] != nullptr && ((uintptr_t)a.x[i] % 16 != 0 || a.x_rs[i] * es % 16 != 0)) return false;
    }
    return true;
}

template <typename T, bool INTER, bool NORM, bool APPEND, int PP, bool FAR_IN>
hipError_t launch_units(RopeKParams p, int passes, hipStream_t st) {
    p.slices = (passes + PP - 1) / PP;
    const int64_t wgs = (p.total * p.slices + kWaves - 1) / kWaves;
    constexpr int64_t kMost = (int64_t(1) << 32) / (kWaves * 64) - 1;  // (a grid has fewer than 2^32 threads)
    for (; p.wg0 < wgs; p.wg0 += kMost) {
        hipLaunchKernelGGL((rope_kernel<T, INTER, NORM, APPEND, PP, FAR_IN>), dim3((unsigned)std::min(wgs - p.wg0, kMost)),
                           dim3(kWaves * 64), 0, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Rows in of a rotation without norms come past the caches where they and the rows out are
// more than the last cache holds (256 MiB), rows of 16 bits only. Just written by another
// kernel and with that one, bf16, 32/8 heads, D = 128: 16384 tokens (336 MB) 129 -> 123 us,
// displaced 71 -> 66 alone; 12288 (252 MB) 88 -> 92, 4096 30.8 -> 31.4, 16384 of 16/16, D = 80
// (168 MB) 36 -> 41, though displaced rows would gain there too (8192 41 -> 38). fp32: a line
// would come twice (see the backward; 16384 of 16/16, D = 80 80 -> 99, of 32/8, D = 128 122 -> 130).
bool past_caches(const RopeKParams& p, int es) {
    constexpr double kLastCache = 256.0 * (1 << 20);
    return 2.0 * (double)p.total * (p.hq + p.hkv) * p.d * es > kLastCache;
}

// Two passes per wave from 8192 passes on (2048 tokens of 32/8 heads, D = 128, bf16: 10.0 us, with
// one 11.0; 16384 appended tokens with norms 76 against 83), one below, for the waves (1024
// with norms 7.6 us, with two 7.9; 16 3.7 against 4.5). More than two were slower.
template <typename T, bool INTER, bool NORM, bool APPEND>
hipError_t launch_passes(const RopeKParams& p, hipStream_t st) {
    const int hpw = 64 >> p.units_log2, passes = (p.heads + hpw - 1) / hpw;
    if constexpr (!NORM && !APPEND && T::code != F32::code) {
        if (past_caches(p, sizeof(typename T::raw))) return launch_units<T, INTER, NORM, APPEND, 2, true>(p, passes, st);
    }
    if (p.total * passes <= 8192) return launch_units<T, INTER, NORM, APPEND, 1, APPEND>(p, passes, st);
    return launch_units<T, INTER, NORM, APPEND, 2, APPEND>(p, passes, st);
}

template <typename T>
hipError_t launch_typed(const RopeArgs& a, hipStream_t st) {
    RopeKParams p = params(a);
    const bool norm_bwd = a.backward && p.norm;
    if (norm_bwd) p.slices = bwd_slices(a.total);
    const bool units = whole_units(a, sizeof(typename T::raw));
    const int part_wgs = units ? unit_part_wgs(a.total, p.slices) : any_part_wgs(a.total, p.heads);
    if (a.total > 0) {
        if (!units) {
            const int64_t items = a.total * ((p.heads + kAnyHeads - 1) / kAnyHeads);
            const int64_t wgs = norm_bwd ? part_wgs : std::min<int64_t>((items + kWaves - 1) / kWaves, 1 << 20);
            if (norm_bwd) hipLaunchKernelGGL((rope_any_kernel<T, true>), dim3((unsigned)wgs), dim3(kWaves * 64), 0, st, p, false);
            else hipLaunchKernelGGL((rope_any_kernel<T, false>), dim3((unsigned)wgs), dim3(kWaves * 64), 0, st, p, a.append);
        } else if (norm_bwd) {
            if (a.interleaved) hipLaunchKernelGGL((rope_bwd_kernel<T, true>), dim3(part_wgs), dim3(kWaves * 64), 0, st, p);
            else hipLaunchKernelGGL((rope_bwd_kernel<T, false>), dim3(part_wgs), dim3(kWaves * 64), 0, st, p);
        } else {
            hipError_t e;
            if (a.append) {
                if (p.norm) e = a.interleaved ? launch_passes<T, true, true, true>(p, st) : launch_passes<T, false, true, true>(p, st);
                else e = a.interleaved ? launch_passes<T, true, false, true>(p, st) : launch_passes<T, false, false, true>(p, st);
            } else if (p.norm) {
                e = a.interleaved ? launch_passes<T, true, true, false>(p, st) : launch_passes<T, false, true, false>(p, st);
            } else {
                e = a.interleaved ? launch_passes<T, true, false, false>(p, st) : launch_passes<T, false, false, false>(p, st);
            }
            if (e != hipSuccess) return e;
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (norm_bwd && (a.dw[0] != nullptr || a.dw[1] != nullptr)) {
        hipLaunchKernelGGL(rope_dw_kernel, dim3((unsigned)((2 * a.d + 3) / 4)), dim3(256), 0, st, a.part,
                           a.total > 0 ? part_wgs : 0, a.d, a.w_dtype, a.dw[0], a.dw[1]);
    }
    return hipGetLastError();
}

}  // namespace

int rope_part_wgs(int64_t total) { return any_part_wgs(total, 1 << 17); }

hipError_t launch_rope(int dtype, const RopeArgs& a, hipStream_t st) {
    if (dtype == MTLATTN_DTYPE_BF16) return launch_typed<BF16>(a, st);
    if (dtype == MTLATTN_DTYPE_F16) return launch_typed<F16>(a, st);
    if (dtype == MTLATTN_DTYPE_F32) return launch_typed<F32>(a, st);
    return hipErrorInvalidValue;
}

}  // namespace mtlattn
