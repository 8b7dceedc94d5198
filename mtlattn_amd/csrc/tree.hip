// Attention of a tree of drafted tokens over a paged K/V cache, fp16/bf16; no
// counterpart in the reference. A sequence's n drafted tokens are its last n logical
// tokens; query i sees the keys before them and those drafted ones that row i of the
// mask names:
//
//   S[i, j] = scale * q_i . k_j,  P = softmax over the seen j,  O_i = sum_j P[i, j] v_j
//
// With few rows (drafted tokens times the heads of a GQA group) the cache's stream
// bounds it, with many the matrix cores do.
//   * A unit of work is up to ROWS = 32 RW of the rows n * g that share a kv head,
//     against all keys of the sequence, in tiles of KT. All units' tiles are numbered in one line, cut
//     into equal pieces, one per workgroup that the GPU holds, from the offsets on
//     the device (no host read): a piece may end one unit and begin the next. Units
//     inside one piece are written directly; of the others each piece leaves
//     normalised fp32 rows and their LSEs, two at most (of the unit that an earlier
//     piece began, of the one that begins here and goes on), for the merge kernel.
//   * 4 waves share the tiles in LDS: RW of them take other rows, KW = 4 / RW other
//     keys of a tile (their results meet in LDS at the end of the unit), so that few
//     rows still keep four waves at the stream.
//   * K and V go from the pages into LDS by direct loads, 16 keys (one page, one
//     lookup) at a time per wave, one tile ahead. Products and softmax are those of
//     the flash forward (fwd.hip): S^T = K Q^T, O^T += V^T P^T on 32x32x16 matrix
//     instructions, softmax statistics and sums in fp32, P rounded to the type of q
//     for the second product (half a step of each weight: less than the output's own
//     rounding; the row sum adds the rounded weights).
//   * Keys before the tree are seen by every row: their tiles have no masks. The
//     tree's tiles take 32 bits per row and 32 keys, and there nothing of a key that
//     a row does not see reaches it, infinities and NaN of V included (a product with 0
//     would let them in).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "../../include/mtlattn_capi.h"

namespace mtlattn {

namespace {

constexpr int kWaves = 4;
constexpr int kMaskWords = kTreeMaxCols / 32 + 1;      // of a token's mask; the last one is 0

struct TreeKParams {
    const uint16_t* q; const uint16_t* k; const uint16_t* v;
    uint16_t* o; float* lse;
    const int* cu_q; const int* cu_kv; const int* block_table;
    const uint8_t* mask; int64_t mask_rs;
    int64_t q_rs, k_rs, v_rs, bt_stride, total_q;
    int num_seqs, hq, hkv, g, mask_cols;
    int page_size, page_log2, num_pages;               // page_log2: -1 where the page is no power of two
    float scale_log2;                                  // > 0; q's bits are changed by (x & q_and) ^ q_xor
    uint32_t q_and, q_xor;
    int4* desc;                                        // per piece: sequence, kv head, row tile and pieces of the
                                                       // unit that it begins and leaves to others (0: none)
    float* part_lse; float* part_o;                    // [pieces][2][ROWS], [pieces][2][ROWS][D]
};

// Shortest piece, in tiles.
constexpr int kMinPiece = 1;

// What the units of a sequence are.
struct SeqWork {
    int q0, n, len, tiles, rows;                       // first query, queries, keys, key tiles, row tiles
    int64_t work;                                      // of all its units, in key tiles
};
template <int ROWS, int KT>
__device__ inline SeqWork seq_work(const TreeKParams& p, int s) {
    const SeqRange r = seq_range(p.cu_q, s, p.total_q);
    SeqWork w;
    w.q0 = r.start;
    w.n = r.end - r.start;
    w.len = kv_length(p.cu_kv, s);
    w.tiles = max(1, (w.len + KT - 1) / KT);           // (without keys: rows of 0)
    w.rows = (w.n * p.g + ROWS - 1) / ROWS;
    w.work = (int64_t)w.tiles * w.rows * p.hkv;
    return w;
}
__device__ inline int64_t wave_sum64(int64_t x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor((long long)x, o);
    return x;
}
__device__ inline int64_t lane_value64(int64_t x, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, l), hi = __builtin_amdgcn_readlane((int)(x >> 32), l);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// 32 bits of a token's mask for the keys from node `base` of the tree on (keys before the tree: 1).
__device__ inline uint32_t mask_bits(const uint32_t* words, int base) {
    if (base <= -32) return ~0u;
    if (base < 0) return words[0] << -base | ((1u << -base) - 1u);
    if (base >= kTreeMaxCols) return 0u;
    const int i = base >> 5, sh = base & 31;
    return (uint32_t)(((uint64_t)words[i + 1] << 32 | words[i]) >> sh);
}

// Both 16-bit halves of w where they are not finite, as masks of 16 ones.
template <typename T>
__device__ inline uint32_t not_finite(uint32_t w) {
    constexpr uint32_t top = T::code == BF16::code ? 0x7f80u : 0x7c00u;
    const uint32_t lo = (w & 0x7fffu) >= top ? 0xffffu : 0u, hi = (w >> 16 & 0x7fffu) >= top ? 0xffff0000u : 0u;
    return lo | hi;
}
// 1 for inf, 128 for -inf, 16384 for NaN, else 0, as T: sums of at most 127 of each tell which there are.
template <typename T>
__device__ inline uint32_t kind_of(uint32_t h) {
    constexpr bool bf = T::code == BF16::code;
    constexpr uint32_t top = bf ? 0x7f80u : 0x7c00u;
    if ((h & 0x7fffu) < top) return 0u;
    if ((h & 0x7fffu) > top) return bf ? 0x4680u : 0x7400u;
    return (h & 0x8000u) != 0 ? (bf ? 0x4300u : 0x5800u) : (bf ? 0x3f80u : 0x3c00u);
}

template <typename T, int D, int RW, int KT, int NBUF>
__global__ __launch_bounds__(kWaves * 64, NBUF * KT * D * 4 <= 72 * 1024 ? 2 : 1) void tree_kernel(TreeKParams p) {
    constexpr int KW = kWaves / RW, ROWS = 32 * RW;
    constexpr int NKB = KT / 32 / KW;                  // 32-key blocks of a wave
    constexpr int NPC = 2 * NKB;                       // 16-key chunks of P
    constexpr int DC = D / 16, DB = D / 32;
    constexpr int TILE = KT * D * 2, STAGE = 2 * TILE;
    constexpr int NI = 16 * D * 2 / 1024;              // direct loads of 16 rows
    constexpr int NB = KT / 16 / kWaves;               // 16-key blocks that a wave stages
    constexpr int AHEAD = NBUF - 1, LOADS = 2 * NI * NB;
    static_assert(KT % (32 * KW) == 0 && KT % (16 * kWaves) == 0, "a tile's keys over the waves");
    static_assert((KW - 1) * RW * (DB * 4096 + 512) <= NBUF * STAGE, "the waves' results meet in the ring");
    __shared__ __attribute__((aligned(1024))) char smem[NBUF * STAGE];
    __shared__ uint32_t s_mask[ROWS][kMaskWords];

    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, hi = lane >> 5, rw = w % RW, kw = w / RW;
    const int pieces = (int)gridDim.x, id = xcd_remap((int)blockIdx.x, pieces);

    // the piece: all work, then where this piece's share begins
    SeqWork mine{};
    int64_t sum = 0, base = 0, total = 0;
    for (int g0 = 0; g0 < p.num_seqs; g0 += 64) {
        const SeqWork x = seq_work<ROWS, KT>(p, min(g0 + lane, p.num_seqs - 1));
        total += wave_sum64(g0 + lane < p.num_seqs ? x.work : 0);
    }
    total = lane_value64(total, 0);
    const int64_t piece = max((int64_t)kMinPiece, (total + pieces - 1) / pieces);
    int64_t at = id * piece;
    const int64_t end = min(total, at + piece);
    if (at >= end) {
        if (threadIdx.x == 0) p.desc[id] = int4{0, 0, 0, 0};
        return;
    }
    int s = 0;
    for (int g0 = 0; g0 < p.num_seqs; g0 += 64) {
        mine = seq_work<ROWS, KT>(p, min(g0 + lane, p.num_seqs - 1));
        const int64_t x = g0 + lane < p.num_seqs ? mine.work : 0;
        sum = x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t y = __shfl_up((long long)sum, o);
            if (lane >= o) sum += y;
        }
        const uint64_t past = __ballot(base + sum > at);
        if (past != 0) {
            const int l = __builtin_ctzll(past);
            s = g0 + l;
            base += lane_value64(sum - x, l);
            break;
        }
        base += lane_value64(sum, 63);
    }
    s = __builtin_amdgcn_readfirstlane(s);

    // where this lane's rows of a 16-key block lie: byte offsets of its direct loads
    uint32_t koff[NI], voff[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        using St = TileStager<D, 16, 1>;
        koff[j] = St::lane_off(j, lane, St::row_of(j, lane), (uint32_t)(2 * p.k_rs));
        voff[j] = St::lane_off(j, lane, St::row_of(j, lane), (uint32_t)(2 * p.v_rs));
    }
    const uint32_t rbase = row_base<D>(l32, hi), tbase = tr_base<D>(lane);
    const float c2 = p.scale_log2;
    constexpr float kRescale = std::is_same<T, F16>::value ? 15.f : 32.f;     // (as in the flash forward)
    int4 begun{0, 0, 0, 0};

    while (at < end && s < p.num_seqs) {
        const SeqWork q = seq_work<ROWS, KT>(p, s);
        if (q.work == 0 || at >= base + q.work) {      // (sequences without queries)
            base += q.work;
            ++s;
            continue;
        }
        const int64_t in = at - base;
        const int unit = __builtin_amdgcn_readfirstlane((int)(in / q.tiles));
        const int t0 = __builtin_amdgcn_readfirstlane((int)(in - (int64_t)unit * q.tiles));
        const int hk = __builtin_amdgcn_readfirstlane(unit / q.rows), rt = unit - hk * q.rows;
        const int t1 = __builtin_amdgcn_readfirstlane((int)min((int64_t)q.tiles, t0 + (end - at)));
        const int len = __builtin_amdgcn_readfirstlane(q.len), ctx = len - q.n, n_rows = q.n * p.g;
        const bool whole = t0 == 0 && t1 == q.tiles;
        if (t0 == 0 && !whole) begun = int4{s, hk, rt, (int)((at + q.tiles - 1) / piece) - id + 1};

        // Q^T operands: lane holds row l32 of the wave's, d = 16 kc + 8 hi + (0..7)
        const int row = rt * ROWS + 32 * rw + l32;
        const int rc = min(row, n_rows - 1), tok = rc / p.g, head = hk * p.g + rc - tok * p.g;
        const uint16_t* qp = p.q + (int64_t)(q.q0 + tok) * p.q_rs + (int64_t)head * D + 8 * hi;
        u32x4_t qf[DC];
#pragma unroll
        for (int kc = 0; kc < DC; ++kc) qf[kc] = ld16(qp + 16 * kc);

        // the masks of the unit's tokens, where this piece reaches the tree
        const int tok0 = rt * ROWS / p.g;
        if ((int64_t)t1 * KT > ctx) {
            const int toks = (min(rt * ROWS + ROWS, n_rows) - 1) / p.g - tok0 + 1, cols = min(q.n, p.mask_cols);
            for (int c = 0; c < kMaskWords; c += 2) {
                const int j = 32 * c + lane;
                constexpr int U = 8;
                for (int i0 = w; i0 < toks; i0 += U * kWaves) {
                    uint8_t b[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int i = min(i0 + u * kWaves, toks - 1);
                        b[u] = j < cols ? p.mask[(int64_t)(q.q0 + tok0 + i) * p.mask_rs + j] : 0;
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const uint64_t bits = __ballot(b[u] != 0);
                        const int i = i0 + u * kWaves;
                        if (lane < 2 && i < toks && c + lane < kMaskWords)
                            s_mask[i][c + lane] = (uint32_t)(lane == 0 ? bits : bits >> 32);
                    }
                }
            }
        }
#pragma unroll
        for (int kc = 0; kc < DC; ++kc)
#pragma unroll
            for (int j = 0; j < 4; ++j) qf[kc][j] = (qf[kc][j] & p.q_and) ^ p.q_xor;
        wait_vmcnt<0>();

        const uint16_t* kh = p.k + (int64_t)hk * D;
        const uint16_t* vh = p.v + (int64_t)hk * D;
        const int* bt = p.block_table + (int64_t)s * p.bt_stride;
        const int last_col = (int)min(p.bt_stride, (int64_t)0x7fffffff) - 1;
        const int n_tiles = len > 0 ? t1 - t0 : 0;
        // 16 keys of a tile at a time; past the last key, its block again, rows that repeat it
        auto stage = [&](int it) {
            char* buf = smem + it % NBUF * STAGE;
            const int kt = (t0 + it) * KT;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int blk = w + b * kWaves;
                const int key = min(kt + 16 * blk, (len - 1) & ~15);
                const int col = p.page_log2 >= 0 ? key >> p.page_log2 : key / p.page_size;
                const int off = key - col * p.page_size;
                const int pg = min(max(bt[min(col, last_col)], 0), p.num_pages - 1);
                const int64_t row0 = (int64_t)pg * p.page_size + off;
                const char* ks = reinterpret_cast<const char*>(kh + row0 * p.k_rs);
                const char* vs = reinterpret_cast<const char*>(vh + row0 * p.v_rs);
                char* kd = buf + blk * NI * 1024;
                const int rmax = len - 1 - key;
                if (rmax >= 15) {
#pragma unroll
                    for (int j = 0; j < NI; ++j) lds_dma16s(ks, koff[j], kd + j * 1024);
#pragma unroll
                    for (int j = 0; j < NI; ++j) lds_dma16s(vs, voff[j], kd + TILE + j * 1024);
                } else {
                    using St = TileStager<D, 16, 1>;
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        lds_dma16s(ks, St::lane_off(j, lane, min(St::row_of(j, lane), rmax), (uint32_t)(2 * p.k_rs)),
                                   kd + j * 1024);
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        lds_dma16s(vs, St::lane_off(j, lane, min(St::row_of(j, lane), rmax), (uint32_t)(2 * p.v_rs)),
                                   kd + TILE + j * 1024);
                }
            }
        };

        float m_run = kNegInf, l_run = 0.f;
        f32x16_t oacc[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[db] = f32x16_t{};
        auto step = [&](int it, auto masked) {
            constexpr bool MASKED = decltype(masked)::value;
            if (AHEAD > 1 && it + 1 < n_tiles) wait_vmcnt<LOADS>(); else wait_vmcnt<0>();
            __syncthreads();
            if (it + AHEAD < n_tiles) stage(it + AHEAD);
            const char* buf = smem + it % NBUF * STAGE;
            const char* kb_ = opaque(buf + rbase) + kw * NKB * 32 * 2 * D;
            const char* vtb = opaque(buf + TILE + tbase) + kw * NKB * 32 * 2 * D;
            f32x16_t sacc[NKB];
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb) sacc[kb] = f32x16_t{};
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kc = 0; kc < DC; ++kc)
#pragma unroll
                for (int kb = 0; kb < NKB; ++kb)
                    sacc[kb] = mfma32<T>(row_operand<D>(kb_, kc, 32 * kb), qf[kc], sacc[kb]);
            pipe_reads<1, NKB * DC, 4>();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            uint32_t bits[NKB];
            if constexpr (MASKED) {
#pragma unroll
                for (int kb = 0; kb < NKB; ++kb) {
                    // (bit 8 (r / 4) + r % 4 is then the key of register r)
                    bits[kb] = mask_bits(s_mask[tok - tok0], (t0 + it) * KT + 32 * (kw * NKB + kb) - ctx) >> (4 * hi);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        sacc[kb][r] = (bits[kb] >> (8 * (r >> 2) + (r & 3)) & 1u) != 0 ? sacc[kb][r] : kNegInf;
                }
            }
            float mx = kNegInf;
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sacc[kb][r]);
            mx = pair_max(mx * c2);
            const float m_new = mx > m_run + kRescale ? mx : m_run;
            if (__any(m_new != m_run)) {
                const float corr = __builtin_amdgcn_exp2f(m_run - (m_new == kNegInf ? 0.f : m_new));
                l_run *= corr;
#pragma unroll
                for (int db = 0; db < DB; ++db) oacc[db] *= corr;
            }
            m_run = m_new;
            const float m_use = m_run == kNegInf ? 0.f : m_run;
            u32x4_t pf[NPC];
#pragma unroll
            for (int c = 0; c < NPC; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 8 * (c & 1) + 2 * j;
                    const float a = __builtin_amdgcn_exp2f(fmaf(sacc[c >> 1][r], c2, -m_use));
                    const float b = __builtin_amdgcn_exp2f(fmaf(sacc[c >> 1][r + 1], c2, -m_use));
                    pf[c][j] = T::pack2(a, b);
                    l_run = dot2_ones<T>(pf[c][j], l_run);
                }
            bool odd = false;
            if constexpr (MASKED) {
                uint32_t any = 0;
#pragma unroll
                for (int c = 0; c < NPC; ++c)
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const u32x4_t v = tr_operand<D>(vtb, c, db);
#pragma unroll
                        for (int j = 0; j < 4; ++j) any |= not_finite<T>(v[j]);
                    }
                odd = __any(any != 0);
            }
            if (MASKED && odd) {
                // finite values by products; of the others, which kinds a row sees
#pragma unroll 1
                for (int c = 0; c < NPC; ++c) {
                    u32x4_t one;
                    const uint32_t cb = bits[NKB == 1 ? 0 : c >> 1] >> (16 * (c & 1));
                    constexpr uint32_t k1 = T::code == BF16::code ? 0x3f80u : 0x3c00u;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int b = 8 * (j >> 1) + 2 * (j & 1);
                        one[j] = (cb >> b & 1u ? k1 : 0u) | (cb >> (b + 1) & 1u ? k1 << 16 : 0u);
                    }
                    u32x4_t pc = pf[0];
#pragma unroll
                    for (int i = 1; i < NPC; ++i) pc = c == i ? pf[i] : pc;
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const u32x4_t v = tr_operand<D>(vtb, c, db);
                        u32x4_t fin, kind;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            fin[j] = v[j] & ~not_finite<T>(v[j]);
                            kind[j] = kind_of<T>(v[j] & 0xffffu) | kind_of<T>(v[j] >> 16) << 16;
                        }
                        oacc[db] = mfma32<T>(fin, pc, oacc[db]);
                        const f32x16_t seen = mfma32<T>(kind, one, f32x16_t{});
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int x = (int)seen[r];
                            const bool pos = (x & 127) != 0, neg = (x >> 7 & 127) != 0, nan = x >= 16384 || (pos && neg);
                            const float add = nan ? __uint_as_float(0x7fc00000u) : pos ? kPosInf : neg ? kNegInf : 0.f;
                            oacc[db][r] = x != 0 ? oacc[db][r] + add : oacc[db][r];
                        }
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < NPC; ++c)
#pragma unroll
                    for (int db = 0; db < DB; ++db) oacc[db] = mfma32<T>(tr_operand<D>(vtb, c, db), pf[c], oacc[db]);
            }
        };
        if (n_tiles > 0) stage(0);
        if (AHEAD > 1 && n_tiles > 1) stage(1);
        // tiles that end before the tree
        const int plain = min(n_tiles, max(0, ctx / KT - t0));
        int it = 0;
        for (; it < plain; ++it) step(it, std::false_type{});
        for (; it < n_tiles; ++it) step(it, std::true_type{});

        float lt = pair_sum(l_run);
        if (KW > 1) {
            // the waves of other keys leave theirs in the ring, lane by lane
            __syncthreads();
            char* mine_ = smem + ((kw - 1) * RW + rw) * (DB * 4096 + 512);
            if (kw > 0) {
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int rg = 0; rg < 4; ++rg)
                        *reinterpret_cast<f32x4_t*>(mine_ + (db * 4 + rg) * 1024 + lane * 16) =
                            f32x4_t{oacc[db][4 * rg], oacc[db][4 * rg + 1], oacc[db][4 * rg + 2], oacc[db][4 * rg + 3]};
                *reinterpret_cast<float*>(mine_ + DB * 4096 + lane * 4) = m_run;
                *reinterpret_cast<float*>(mine_ + DB * 4096 + 256 + lane * 4) = lt;
            }
            __syncthreads();
            if (kw == 0) {
#pragma unroll 1
                for (int i = 1; i < KW; ++i) {
                    const char* other = smem + ((i - 1) * RW + rw) * (DB * 4096 + 512);
                    const float m2 = *reinterpret_cast<const float*>(other + DB * 4096 + lane * 4);
                    const float l2 = *reinterpret_cast<const float*>(other + DB * 4096 + 256 + lane * 4);
                    const float m = nan_max(m2, m_run), mu = m == kNegInf ? 0.f : m;
                    const float a = __builtin_amdgcn_exp2f(m_run - mu), b = __builtin_amdgcn_exp2f(m2 - mu);
                    lt = lt * a + l2 * b;
                    m_run = m;
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int rg = 0; rg < 4; ++rg) {
                            const f32x4_t o =
                                *reinterpret_cast<const f32x4_t*>(other + (db * 4 + rg) * 1024 + lane * 16);
#pragma unroll
                            for (int e = 0; e < 4; ++e) oacc[db][4 * rg + e] = oacc[db][4 * rg + e] * a + o[e] * b;
                        }
                }
            }
        }
        // (NaN is not <= 0; rows that see nothing: 0 and -inf)
        if (kw == 0 && row < n_rows) {
            const float inv = !(lt <= 0.f) ? 1.f / lt : 0.f;
            const float lse = !(lt <= 0.f) ? m_run * kLn2 + logf(lt) : kNegInf;
            if (whole) {
                const int64_t rh = (int64_t)(q.q0 + tok) * p.hq + head;
                uint16_t* op = p.o + rh * D;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int rg = 0; rg < 4; ++rg)
                        st8(op + 32 * db + 8 * rg + 4 * hi,
                            u32x2_t{T::pack2(oacc[db][4 * rg] * inv, oacc[db][4 * rg + 1] * inv),
                                    T::pack2(oacc[db][4 * rg + 2] * inv, oacc[db][4 * rg + 3] * inv)});
                if (p.lse != nullptr && hi == 0) p.lse[rh] = lse;
            } else {
                const int64_t pr = (int64_t)(2 * id + (t0 == 0 ? 1 : 0)) * ROWS + 32 * rw + l32;
                float* op = p.part_o + pr * D;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int rg = 0; rg < 4; ++rg)
                        *reinterpret_cast<f32x4_t*>(op + 32 * db + 8 * rg + 4 * hi) =
                            f32x4_t{oacc[db][4 * rg] * inv, oacc[db][4 * rg + 1] * inv, oacc[db][4 * rg + 2] * inv,
                                    oacc[db][4 * rg + 3] * inv};
                if (hi == 0) p.part_lse[pr] = lse;
            }
        }
        at += t1 - t0;
        __syncthreads();                               // (the ring and the masks are free again)
    }
    if (threadIdx.x == 0) p.desc[id] = begun;
}

// The rows of a unit that several pieces share: half a wave per row, its lanes over
// the head dim, O = sum_z w_z O_z / sum_z w_z, w_z = exp(lse_z - max lse), in the
// pieces' order.
template <typename T, int D, int ROWS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeKParams p) {
    const int a = blockIdx.x;
    const int4 d = p.desc[a];
    if (d.w == 0) return;
    const SeqRange r = seq_range(p.cu_q, d.x, p.total_q);
    const int rr = blockIdx.y * 8 + (threadIdx.x >> 5), l32 = threadIdx.x & 31;
    const int row = d.z * ROWS + rr;
    if (row >= (r.end - r.start) * p.g) return;
    const int tok = row / p.g, head = d.y * p.g + row - tok * p.g;
    // piece z of the unit: the first one's second place, the others' first
    auto place = [&](int z) { return (int64_t)(z == 0 ? 2 * a + 1 : 2 * (a + z)) * ROWS + rr; };
    float m = kNegInf;
    for (int z = l32; z < d.w; z += 32) m = nan_max(p.part_lse[place(z)], m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = nan_max(m, __shfl_xor(m, o));
    constexpr int NE = D / 32;                         // columns of a lane
    float acc[NE] = {}, sum = 0.f;
    if (m != kNegInf) {
#pragma unroll 4
        for (int z = 0; z < d.w; ++z) {
            const int64_t pr = place(z);
            const float l = p.part_lse[pr], wgt = l == kNegInf ? 0.f : __expf(l - m);
            const float* op = p.part_o + pr * D + NE * l32;
            sum += wgt;
#pragma unroll
            for (int e = 0; e < NE; ++e) acc[e] += l == kNegInf ? 0.f : wgt * op[e];
        }
    }
    const float inv = !(sum <= 0.f) ? 1.f / sum : 0.f;
    const int64_t rh = (int64_t)(r.start + tok) * p.hq + head;
    uint32_t* out = reinterpret_cast<uint32_t*>(p.o + rh * D + NE * l32);
#pragma unroll
    for (int e = 0; e < NE; e += 2) out[e / 2] = T::pack2(acc[e] * inv, acc[e + 1] * inv);
    if (p.lse != nullptr && l32 == 0) p.lse[rh] = !(sum <= 0.f) ? m + logf(sum) : kNegInf;
}

template <typename T, int D, int RW, int KT, int NBUF>
hipError_t launch_rows(const TreeArgs& a, TreeKParams p, hipStream_t st) {
    constexpr int ROWS = 32 * RW;
    char* ws = (char*)a.workspace;
    const size_t grid = (size_t)a.plan.grid;
    p.desc = (int4*)ws;
    p.part_lse = (float*)(ws + grid * sizeof(int4));
    p.part_o = p.part_lse + grid * 2 * ROWS;
    hipLaunchKernelGGL((tree_kernel<T, D, RW, KT, NBUF>), dim3((unsigned)grid), dim3(kWaves * 64), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((tree_merge_kernel<T, D, ROWS>), dim3((unsigned)grid, ROWS / 8), dim3(256), 0, st, p);
    return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_typed(const TreeArgs& a, hipStream_t st) {
    const Geometry& g = a.geo;
    TreeKParams p{};
    p.q = (const uint16_t*)a.q; p.k = (const uint16_t*)a.k; p.v = (const uint16_t*)a.v;
    p.o = (uint16_t*)a.o; p.lse = a.lse;
    p.cu_q = g.cu_q; p.cu_kv = g.cu_kv; p.block_table = a.block_table;
    p.mask = a.mask; p.mask_rs = a.mask_rs; p.mask_cols = a.mask_cols;
    p.q_rs = a.q_rs; p.k_rs = a.k_rs; p.v_rs = a.v_rs;
    p.bt_stride = a.bt_stride; p.total_q = g.total_q;
    p.num_seqs = g.num_seqs; p.hq = g.hq; p.hkv = g.hkv; p.g = g.g;
    p.page_size = a.page_size; p.num_pages = a.num_pages;
    p.page_log2 = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctz(a.page_size) : -1;
    // the raw maximum needs a positive factor: a negative one turns q's signs, 0 makes q 0
    p.scale_log2 = (g.scale == 0.f ? 1.f : fabsf(g.scale)) * kLog2e;
    p.q_and = g.scale == 0.f ? 0u : ~0u;
    p.q_xor = g.scale < 0.f ? 0x80008000u : 0u;
    if (a.plan.rows == 32) return launch_rows<T, D, 1, 128, 2>(a, p, st);
    if (a.plan.rows == 64) return launch_rows<T, D, 2, 64, 2>(a, p, st);
    return launch_rows<T, D, 4, 64, 2>(a, p, st);
}

}  // namespace

TreePlan make_tree_plan(const Geometry& g, int max_q, int64_t max_kv, int cus) {
    TreePlan plan;
    const int64_t rows = (int64_t)std::max(max_q, 1) * g.g;
    plan.rows = rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    const int kt = plan.rows == 32 ? 128 : 64;
    // every tile of every unit by the bounds; a grid that those fill
    const int64_t units = ((int64_t)g.num_seqs * g.hkv) * ((rows + plan.rows - 1) / plan.rows);
    const int64_t tiles = std::max<int64_t>(1, (max_kv + kt - 1) / kt);
    const int64_t full = (int64_t)cus * (plan.rows == 32 && g.d == 128 ? 1 : 2);
    const int64_t most = units > full ? full : units * std::min<int64_t>(tiles, full);
    plan.grid = (int)std::max<int64_t>(1, std::min(full, most));
    plan.bytes = (size_t)plan.grid * (16 + 2 * (size_t)plan.rows * ((size_t)g.d + 1) * sizeof(float));
    return plan;
}

hipError_t launch_tree(int dtype, const TreeArgs& a, hipStream_t st) {
    const int d = a.geo.d;
    if (dtype == MTLATTN_DTYPE_BF16) {
        if (d == 128) return launch_typed<BF16, 128>(a, st);
        if (d == 64) return launch_typed<BF16, 64>(a, st);
    } else if (dtype == MTLATTN_DTYPE_F16) {
        if (d == 128) return launch_typed<F16, 128>(a, st);
        if (d == 64) return launch_typed<F16, 64>(a, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace mtlattn
