// Attention of a tree of drafted tokens over a paged K/V cache, fp16/bf16; no
// counterpart in the reference. A sequence's n drafted tokens are its last n logical
// tokens; query i sees the keys before them and those drafted ones that row i of the
// mask names:
//
//   S[i, j] = scale * q_i . k_j,  P = softmax over the seen j,  O_i = sum_j P[i, j] v_j
//
// With few rows (drafted tokens times the heads of a GQA group) the cache's stream
// bounds it, with many the matrix cores and their softmax do. Measured, bf16, D = 128:
// 64 sequences of 2 to 8 drafted tokens over 1024 to 16384 keys, 32/8 heads, 380 us,
// 5.9 TB/s; 4 of 64 over 32768 to 98304, 64/8 heads, 688 us, where the matrix cores
// run at 1.15 PFLOP/s, 63% of their cycles at the 1.74 GHz that the GPU then holds; one of
// 16 over 700, 15 us.
//   * A unit of work is up to ROWS = 32 RW of the rows n * g that share a kv head,
//     against all keys of the sequence, in tiles of KT. All units' tiles are numbered in
//     one line, cut into equal pieces, from the offsets on the device (no host read): a
//     piece may end one unit and begin the next. Units inside one piece are written
//     directly; of the others each piece leaves normalised fp32 rows and their LSEs, two
//     at most (of the unit that an earlier piece began, of the one that begins here and
//     goes on), for the merge kernel. A workgroup takes a piece for one kv head; those of
//     all heads run side by side.
//   * NW waves share the tiles in LDS: RW of them take other rows, KW = NW / RW other
//     keys of a tile (their results meet in LDS at the end of the unit), so that few
//     rows still keep four waves at the stream, two workgroups a CU.
//   * K and V go from the pages into a ring of two tiles in LDS by direct loads, 16 keys
//     (one page) at a time per wave, whose rows were looked up 64 blocks of 16 keys at a
//     time (one lookup per tile, in front of its loads, cost 20% of a stream). The loads
//     leave nothing in the caches (the 64 sequences 418 -> 381 us; 119 MB of cache that
//     nothing else displaced since the last call 45 -> 50, displaced 49 -> 47). Products
//     and softmax are those of the flash forward (fwd.hip): S^T = K Q^T, O^T += V^T P^T
//     on 32x32x16 matrix instructions, operands read four ahead (two the same), softmax
//     statistics and sums in fp32.
//   * P enters the second product as the sum of two numbers of q's type, itself rounded
//     and what that left: 16 bits of it in bf16, 22 in fp16, far below the rounding of the
//     result. (Rounded once, results were off by 2.1-2.3e-3 of their norm in bf16 where
//     1.7e-3 is their own rounding. Its second part takes half as many products again,
//     which the streams hide, 377 -> 380 us; few rows 43 -> 45; the long trees, at the matrix
//     cores' rate, 512 -> 688.)
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

constexpr int kMaskWords = kTreeMaxCols / 32 + 1;      // of a token's mask; the last one is 0
// Beginning a unit after another one in a piece takes as long as this many tiles (the last
// stores, a page lookup and the first tile's loads, one after the other, where the GPU streams:
// 16 sequences of 8 to 32 drafted tokens over 128 to 4096 keys, 32/8 heads, D = 128: 47.5 us
// without, 45.2 with 4, 45.9 with 7; 12 of 512 to 16384 keys, 16 heads, D = 64: 89, 80, 79;
// one of 16 over 700: 16.3, 15.0, 16.1).
constexpr int kUnitCost = 4;

struct TreeKParams {
    const uint16_t* q; const uint16_t* k; const uint16_t* v;
    uint16_t* o; float* lse;
    const int* cu_q; const int* cu_kv; const int* block_table;
    const uint8_t* mask; int64_t mask_rs;
    int64_t q_rs, k_rs, v_rs, bt_stride, total_q;
    int num_seqs, hq, hkv, g, mask_cols;
    int page_size, page_log2, num_pages;               // page_log2: -1 where the page is no power of two
    int pieces, side;                                  // workgroups: pieces * hkv * side (row tiles side by side)
    float scale_log2;                                  // > 0; q's bits are changed by (x & q_and) ^ q_xor
    uint32_t q_and, q_xor;
    int4* desc;                                        // per workgroup: first query, rows, row tile and pieces of the
                                                       // unit that it begins and leaves to others (pieces 0: none)
    float* part_lse; float* part_o;                    // [workgroups][2][ROWS], [workgroups][2][ROWS][D]
};

// The kernel reads its parameters where they lie: a fresh pointer keeps the compiler
// from holding all of them in scalar registers through the loops (which it then puts
// into lanes of vector registers, and those into memory).
typedef const __attribute__((address_space(4))) TreeKParams CParams;
__device__ inline CParams* params() {
    uint64_t a = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return (CParams*)a;
}

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline const char* uniform(const char* x) {
    const uint64_t a = (uint64_t)x;
    return (const char*)((uint64_t)(uint32_t)uniform((int)(a >> 32)) << 32 | (uint32_t)uniform((int)(uint32_t)a));
}

// The units of a sequence: first query, queries, keys, key tiles, rounds of row tiles (`side`
// of them at a time), and the work of one of the workgroups side by side in key tiles.
struct SeqWork {
    int q0, n, len, tiles, rounds;
    int64_t work;
};
template <int D, int ROWS, int KT>
__device__ inline SeqWork seq_work(CParams* p, int s) {
    const SeqRange r = seq_range(p->cu_q, s, p->total_q);
    SeqWork w;
    w.q0 = r.start;
    w.n = r.end - r.start;
    w.len = kv_length(p->cu_kv, s);
    w.tiles = max(1, (w.len + KT - 1) / KT);           // (without keys: rows of 0)
    w.rounds = ((w.n * p->g + ROWS - 1) / ROWS + p->side - 1) / p->side;
    w.work = (int64_t)(w.tiles + kUnitCost) * w.rounds;
    return w;
}
__device__ inline int64_t lane_value64(int64_t x, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, l), hi = __builtin_amdgcn_readlane((int)(x >> 32), l);
    return (int64_t)((uint64_t)hi << 32 | lo);
}
// x + the value `ctrl` moves here from another lane (0 where there is none).
template <int CTRL, int ROWS_MASK>
__device__ inline int add_dpp(int x) {
    return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS_MASK, 0xf, false);
}
// Sums over the lanes up to and with each one: by lane moves in 32 bits where they hold it.
__device__ inline int64_t wave_scan64(int64_t x, int lane) {
    if (!__any(x >= (1 << 24))) {
        int y = (int)x;
        y = add_dpp<0x111, 0xf>(y);                    // row_shr 1, 2, 4, 8: within 16 lanes
        y = add_dpp<0x112, 0xf>(y);
        y = add_dpp<0x114, 0xf>(y);
        y = add_dpp<0x118, 0xf>(y);
        y = add_dpp<0x142, 0xa>(y);                    // row_bcast 15: into the second and the fourth 16
        y = add_dpp<0x143, 0xc>(y);                    // row_bcast 31: into the upper 32
        return y;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up((long long)x, o);
        if (lane >= o) x += y;
    }
    return x;
}
// a / b of non-negative numbers, in 32 bits where those hold them.
__device__ inline int64_t quotient(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// 32 bits of a token's mask for the keys from node `base` of the tree on (keys before the tree: 1).
__device__ inline uint32_t mask_bits(const uint32_t* words, int base) {
    if (base <= -32) return ~0u;
    if (base < 0) return words[0] << -base | ((1u << -base) - 1u);
    if (base >= kTreeMaxCols) return 0u;
    const int i = base >> 5, sh = base & 31;
    return (uint32_t)(((uint64_t)words[i + 1] << 32 | words[i]) >> sh);
}

// Ones in the halves of w that are finite.
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
template <typename T>
constexpr uint32_t kInf16 = T::code == BF16::code ? 0x7f80u : 0x7c00u;
template <typename T>
__device__ inline uint32_t finite_halves(uint32_t w) {
    return ((w & 0x7fffu) >= kInf16<T> ? 0u : 0xffffu) | ((w >> 16 & 0x7fffu) >= kInf16<T> ? 0u : 0xffff0000u);
}

// The bits of the tokens' masks of a row tile, a wave per token: bytes in, ballots out.
template <int NW>
__device__ inline void load_masks(CParams* p, uint32_t (*s_mask)[kMaskWords], int64_t first, int toks, int cols, int w,
                                  int lane) {
    constexpr int U = 8;
    const uint8_t* mask = p->mask + first * p->mask_rs;
    const int64_t rs = p->mask_rs;
    for (int i0 = w; i0 < toks; i0 += U * NW) {
        for (int c = 0; c < kMaskWords; c += 2) {
            const int j = 32 * c + lane;
            uint8_t b[U];
#pragma unroll
            for (int u = 0; u < U; ++u) b[u] = j < cols ? mask[min(i0 + u * NW, toks - 1) * rs + j] : 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t bits = __ballot(b[u] != 0);
                const int i = i0 + u * NW;
                if (lane < 2 && i < toks && c + lane < kMaskWords) s_mask[i][c + lane] = (uint32_t)(bits >> (32 * lane));
            }
        }
    }
}

template <typename T, int D, int NW, int RW, int KT>
__global__ __launch_bounds__(NW * 64, NW == 4 ? 2 : 1) void tree_kernel(TreeKParams) {
    constexpr int KW = NW / RW, ROWS = 32 * RW;
    constexpr int NKB = KT / 32 / KW;                  // 32-key blocks of a wave
    constexpr int NPC = 2 * NKB;                       // 16-key chunks of P
    constexpr int DC = D / 16, DB = D / 32;
    constexpr int TILE = KT * D * 2, STAGE = 2 * TILE;
    constexpr int NI = 16 * D * 2 / 1024;              // direct loads of 16 rows
    constexpr int NU = 2 * KT / 16 / NW;               // 16-row blocks of K or V that a wave stages
    constexpr int LOADS = NU * NI, NS = NKB * DC;      // of a wave and tile: direct loads, products of S
    constexpr int kShare = DB * 4096 + 2 * 256;        // bytes of a wave's O, maxima and sums
    constexpr bool SPREAD = LOADS <= NS;               // loads between the products
    using St = TileStager<D, 16, 1>;
    static_assert(KT % (32 * KW) == 0 && KT % (16 * NW) == 0, "a tile's keys over the waves");
    static_assert((KW - 1) * RW * kShare <= 2 * STAGE, "the waves' results meet in the ring");
    __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
    __shared__ uint32_t s_mask[ROWS][kMaskWords];
    __shared__ int s_odd;

    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
    const int l32 = lane & 31, hi = lane >> 5, rw = w % RW, kw = w / RW;

    // the piece: all work, and where this piece's share begins. The kv heads of a piece run
    // side by side, so that whole rows of the cache are read together, and so do `side` row
    // tiles of a head, which read the same.
    int id, piece_id, hk, rt0, s = 0;
    int64_t at, end, base = 0, piece;
    SeqWork sw;
    {
        CParams* p = params();
        id = xcd_remap((int)blockIdx.x, p->pieces * p->hkv * p->side);
        const int col = uniform(id / p->side);
        rt0 = id - col * p->side;
        piece_id = uniform(col / p->hkv);
        hk = col - piece_id * p->hkv;
        const int n = p->num_seqs;
        const SeqWork first = seq_work<D, ROWS, KT>(p, min(lane, n - 1));
        const int64_t sum0 = wave_scan64(lane < n ? first.work : 0, lane);
        int64_t total = lane_value64(sum0, 63);
        for (int g0 = 64; g0 < n; g0 += 64) {
            const SeqWork x = seq_work<D, ROWS, KT>(p, min(g0 + lane, n - 1));
            total += lane_value64(wave_scan64(g0 + lane < n ? x.work : 0, lane), 63);
        }
        piece = max((int64_t)1, quotient(total + p->pieces - 1, p->pieces));
        at = piece_id * piece;
        end = min(total, at + piece);
        if (at >= end) {
            if (threadIdx.x == 0) p->desc[id] = int4{0, 0, 0, 0};
            return;
        }
        for (int g0 = 0; g0 < n; g0 += 64) {
            int64_t sum = sum0;
            sw = first;
            if (g0 > 0) {
                sw = seq_work<D, ROWS, KT>(p, min(g0 + lane, n - 1));
                sum = wave_scan64(g0 + lane < n ? sw.work : 0, lane);
            }
            const uint64_t past = __ballot(g0 + lane < n && base + sum > at);
            if (past != 0) {
                const int l = __builtin_ctzll(past);
                s = g0 + l;
                base += lane_value64(sum - sw.work, l);
                sw.q0 = __builtin_amdgcn_readlane(sw.q0, l);
                sw.n = __builtin_amdgcn_readlane(sw.n, l);
                sw.len = __builtin_amdgcn_readlane(sw.len, l);
                sw.tiles = __builtin_amdgcn_readlane(sw.tiles, l);
                sw.work = lane_value64(sw.work, l);
                break;
            }
            base += lane_value64(sum, 63);
        }
    }

    // Where this lane's part of a 16-row block lies: instruction j loads row LR j + lane / (D / 8), at
    // the chunk that the swizzle puts there (TileStager::lane_off), which is its chunk of
    // instruction 0 with the swizzle of LR j rows on top
    constexpr int LR = 64 * 16 / (2 * D);              // rows of an instruction
    const uint32_t chunk0 = (uint32_t)((lane & (D / 8 - 1)) ^ row_swz<D>(lane / (D / 8))) * 16u;
    const uint32_t lane_krow = (uint32_t)(lane / (D / 8)) * (uint32_t)(2 * params()->k_rs);   // bytes, in K and in V
    const uint32_t lane_vrow = (uint32_t)(lane / (D / 8)) * (uint32_t)(2 * params()->v_rs);
    const uint32_t rbase = row_base<D>(l32, hi) + kw * NKB * 32 * 2 * D, tbase = TILE + tr_base<D>(lane) + kw * NKB * 32 * 2 * D;
    constexpr float kRescale = std::is_same<T, F16>::value ? 15.f : 32.f;     // (as in the flash forward)
    int4 begun{0, 0, 0, 0};

    while (at < end) {
        CParams* p = params();
        if (at >= base + sw.work) {                    // (this sequence is done, or has no queries)
            base += sw.work;
            if (++s >= p->num_seqs) break;
            sw = seq_work<D, ROWS, KT>(p, s);
            continue;
        }
        // (the line has kUnitCost places before a unit's tiles: a piece that begins a unit
        // after another one gets fewer tiles)
        const int len_v = sw.tiles + kUnitCost, round = uniform((int)quotient(at - base, len_v)), rt = round * p->side + rt0;
        const int64_t unit_at = base + (int64_t)round * len_v + kUnitCost;     // the unit's first tile
        const int t0 = uniform((int)max(at - unit_at, (int64_t)0));
        const int t1 = uniform((int)(min(unit_at + sw.tiles, end) - unit_at));
        const int len = uniform(sw.len), ctx = len - uniform(sw.n), n_rows = uniform(sw.n) * p->g, q0 = uniform(sw.q0);
        const bool whole = t0 == 0 && t1 == sw.tiles;
        at = min(unit_at + sw.tiles, end);
        // (a piece that ends before the first tile; the last round has fewer row tiles)
        if (t1 <= 0 || (int64_t)rt * ROWS >= n_rows) continue;
        if (t0 == 0 && !whole)
            begun = int4{q0, n_rows, rt, (int)quotient(unit_at + sw.tiles - 1, piece) - piece_id + 1};

        // 16 keys of a tile at a time; past the last key, its block again, rows that repeat it
        const int n_tiles = len > 0 ? t1 - t0 : 0;
        const int* bt = p->block_table + (int64_t)s * p->bt_stride;
        const int last_col = (int)min(p->bt_stride, (int64_t)0x7fffffff) - 1;
        const int page_log2 = p->page_log2, page_size = p->page_size, num_pages = p->num_pages;
        const int64_t k_rs = p->k_rs, v_rs = p->v_rs;
        const char* kh = reinterpret_cast<const char*>(p->k + (int64_t)hk * D);
        const char* vh = reinterpret_cast<const char*>(p->v + (int64_t)hk * D);
        // Cache rows of 64 blocks of 16 keys at a time (TPG tiles), a lane each, the next 64's
        // lookups under way meanwhile.
        constexpr int BPT = KT / 16, TPG = 64 / BPT;
        auto block_key = [&](int g) { return min((t0 + g * TPG) * KT + 16 * lane, (len - 1) & ~15); };
        auto block_col = [&](int key) { return page_log2 >= 0 ? key >> page_log2 : key / page_size; };
        auto lookup = [&](int g) { return bt[min(block_col(block_key(g)), last_col)]; };
        auto cache_row = [&](int pg, int g) {
            const int key = block_key(g);
            return min(max(pg, 0), num_pages - 1) * page_size + (key - block_col(key) * page_size);
        };
        int rows_now = 0, pages_next = 0;
        if (n_tiles > 0) {
            rows_now = cache_row(lookup(0), 0);
            pages_next = lookup(1);
        }
        // block i of this wave's in tile `it`, first those of K, then those of V: its first key, its source
        auto key_side = [](int i) { return i < NU / 2; };
        auto first_key = [&](int it, int i) __attribute__((always_inline)) {
            return min((t0 + it) * KT + 16 * ((w + i * NW) & (BPT - 1)), (len - 1) & ~15);
        };
        auto source = [&](int it, int i) __attribute__((always_inline)) {
            const int64_t row = __builtin_amdgcn_readlane(rows_now, it % TPG * BPT + ((w + i * NW) & (BPT - 1)));
            return uniform(key_side(i) ? kh + row * (2 * k_rs) : vh + row * (2 * v_rs));
        };
        auto next_rows = [&](int it) __attribute__((always_inline)) {      // before a tile's sources are taken
            if (it % TPG == 0 && it > 0) {
                rows_now = cache_row(pages_next, it / TPG);
                pages_next = lookup(it / TPG + 1);
            }
        };
        auto lane_off = [&](int i, int j) __attribute__((always_inline)) {
            uint32_t c = chunk0;                       // (one add per use, not a register held per load)
            asm volatile("" : "+v"(c));
            return (c ^ (uint32_t)(row_swz<D>(j * LR) * 16)) + (key_side(i) ? lane_krow : lane_vrow);
        };
        auto stage = [&](int it) __attribute__((always_inline)) {
            char* buf = smem + it % 2 * STAGE;
            next_rows(it);
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int key = first_key(it, i), rmax = len - 1 - key;
                const char* src = source(it, i);
                char* dst = buf + (w + i * NW) * NI * 1024;
                const uint32_t rs2 = (uint32_t)(2 * (key_side(i) ? k_rs : v_rs));
                if (rmax >= 15) {
#pragma unroll
                    for (int j = 0; j < NI; ++j) lds_dma16s_once(src + j * LR * (int64_t)rs2, lane_off(i, j), dst + j * 1024);
                } else {
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        lds_dma16s_once(src, St::lane_off(j, lane, min(St::row_of(j, lane), rmax), rs2), dst + j * 1024);
                }
            }
        };

        // Q^T operands: lane holds row l32 of the wave's, d = 16 kc + 8 hi + (0..7)
        const int row = rt * ROWS + 32 * rw + l32;
        const int tok = min(row, n_rows - 1) / p->g, head = hk * p->g + min(row, n_rows - 1) - tok * p->g;
        const int tok0 = rt * ROWS / p->g;
        u32x4_t qf[DC];
        {
            const uint16_t* qp = p->q + (int64_t)(q0 + tok) * p->q_rs + (int64_t)head * D + 8 * hi;
#pragma unroll
            for (int kc = 0; kc < DC; ++kc) qf[kc] = ld16(qp + 16 * kc);
            if (n_tiles > 0) stage(0);
            // the masks of the unit's tokens, where this piece reaches the tree
            if ((int64_t)t1 * KT > ctx)
                load_masks<NW>(p, s_mask, q0 + tok0, (min(rt * ROWS + ROWS, n_rows) - 1) / p->g - tok0 + 1,
                               min(uniform(sw.n), p->mask_cols), w, lane);
            const uint32_t q_and = p->q_and, q_xor = p->q_xor;
#pragma unroll
            for (int kc = 0; kc < DC; ++kc)
#pragma unroll
                for (int j = 0; j < 4; ++j) qf[kc][j] = (qf[kc][j] & q_and) ^ q_xor;
        }
        const float c2 = p->scale_log2;

        if (threadIdx.x == 0) s_odd = 0;               // a value of V in the tree's tiles is not finite
        float m_run = kNegInf, l_run = 0.f;
        f32x16_t oacc[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[db] = f32x16_t{};
        auto step = [&](int it, auto masked) __attribute__((always_inline)) {
            constexpr bool MASKED = decltype(masked)::value;
            wait_vmcnt<0>();
            __syncthreads();
            // (a tile that ends past the last key is staged at once, with its rows clamped)
            const bool more = it + 1 < n_tiles;
            const bool spread = SPREAD && !MASKED && more && (t0 + it + 2) * KT <= len;
            if (more && !spread) stage(it + 1);
            const char* kb_ = opaque(smem + it % 2 * STAGE + rbase);
            const char* vtb = opaque(smem + it % 2 * STAGE + tbase);
            f32x16_t sacc[NKB];
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb) sacc[kb] = f32x16_t{};
            __builtin_amdgcn_s_setprio(1);
            auto products = [&](auto with_loads) __attribute__((always_inline)) {
                const char* src[NU];
                char* dst = smem + (it + 1) % 2 * STAGE + w * NI * 1024;
                if (decltype(with_loads)::value) {
                    next_rows(it + 1);
#pragma unroll
                    for (int i = 0; i < NU; ++i) src[i] = source(it + 1, i);
                }
                u32x4_t ka[NS];
#pragma unroll
                for (int i = 0; i < 4 && i < NS; ++i) ka[i] = row_operand<D>(kb_, i / NKB, 32 * (i % NKB));
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    sacc[i % NKB] = mfma32<T>(ka[i], qf[i / NKB], sacc[i % NKB]);
                    if (i + 4 < NS) ka[i + 4] = row_operand<D>(kb_, (i + 4) / NKB, 32 * ((i + 4) % NKB));
                    if constexpr (decltype(with_loads)::value) {
                        constexpr int E = NS / LOADS;          // products per load
                        if (i % E == E - 1 && i / E < LOADS) {
                            const int x = i / E / NI, j = i / E % NI;
                            lds_dma16s_once(src[x] + j * LR * (2 * (key_side(x) ? k_rs : v_rs)), lane_off(x, j),
                                       dst + (x * NW * NI + j) * 1024);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            if constexpr (SPREAD && !MASKED) {
                if (spread) products(std::true_type{});
                else products(std::false_type{});
            } else {
                products(std::false_type{});
            }
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            if constexpr (MASKED) {
#pragma unroll
                for (int kb = 0; kb < NKB; ++kb) {
                    // (bit 8 (r / 4) + r % 4 is then the key of register r)
                    const uint32_t bits =
                        mask_bits(s_mask[tok - tok0], (t0 + it) * KT + 32 * (kw * NKB + kb) - ctx) >> (4 * hi);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        sacc[kb][r] = (bits >> (8 * (r >> 2) + (r & 3)) & 1u) != 0 ? sacc[kb][r] : kNegInf;
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
            u32x4_t pf[NPC], pl[NPC];                  // the weights rounded, and what that left of them
#pragma unroll
            for (int c = 0; c < NPC; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 8 * (c & 1) + 2 * j;
                    const float a = __builtin_amdgcn_exp2f(fmaf(sacc[c >> 1][r], c2, -m_use));
                    const float b = __builtin_amdgcn_exp2f(fmaf(sacc[c >> 1][r + 1], c2, -m_use));
                    l_run += a + b;
                    pf[c][j] = T::pack2(a, b);
                    pl[c][j] = T::pack2(a - lo16<T>(pf[c][j]), b - hi16<T>(pf[c][j]));
                }
            if constexpr (MASKED) {
                // this wave's share of the tile's V: what is not finite leaves the tile, and is
                // added below to the rows that see it
                char* vs = smem + it % 2 * STAGE + TILE + w * (TILE / NW) + lane * 16;
#pragma unroll
                for (int i = 0; i < TILE / NW / 1024; ++i) {
                    u32x4_t v = ld16(vs + i * 1024);
                    u16x2_t top{};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, v[j] & 0x7fff7fffu));
                    if (max(top[0], top[1]) >= kInf16<T>) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] &= finite_halves<T>(v[j]);
                        st16(vs + i * 1024, v);
                        s_odd = 1;
                    }
                }
                __syncthreads();
            }
            // (the operand reads four products ahead)
            constexpr int NV = NPC * DB;
            u32x4_t va[NV];
#pragma unroll
            for (int i = 0; i < 4; ++i) va[i] = tr_operand<D>(vtb, i / DB, i % DB);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                oacc[i % DB] = mfma32<T>(va[i], pf[i / DB], oacc[i % DB]);
                oacc[i % DB] = mfma32<T>(va[i], pl[i / DB], oacc[i % DB]);
                if (i + 4 < NV) va[i + 4] = tr_operand<D>(vtb, (i + 4) / DB, (i + 4) % DB);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // tiles that end before the tree
        const int plain = min(n_tiles, max(0, ctx / KT - t0));
        int it = 0;
#pragma unroll 1
        for (; it < plain; ++it) step(it, std::false_type{});
#pragma unroll 1
        for (; it < n_tiles; ++it) step(it, std::true_type{});

        // Where a seen value of V is not finite, the column is what such values add up to (an
        // infinity times the two parts of a weight can be NaN): this wave's keys, from the
        // cache, 64 at a time, those with such a value one after the other. In the tree's
        // tiles where V was found to have one, before them where a sum is not finite (of rows
        // with a weight that is NaN every column is).
        float lt = pair_sum(l_run), off = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) off = fmaf(oacc[db][r], 0.f, off);
        const bool odd = plain < n_tiles && uniform(s_odd) != 0, before = __any(off != off && lt == lt);
        if (odd || before) {
            const uint32_t* words = s_mask[tok - tok0];
            const int last = min(len, t1 * KT);
            auto value_row = [&](int key) {
                const int col = page_log2 >= 0 ? key >> page_log2 : key / page_size;
                const int pg = min(max(bt[min(col, last_col)], 0), num_pages - 1);
                return vh + ((int64_t)pg * page_size + (key - col * page_size)) * (2 * v_rs);
            };
            f32x16_t x[DB];
#pragma unroll
            for (int db = 0; db < DB; ++db) x[db] = f32x16_t{};
#pragma unroll 1
            for (int key0 = before ? t0 * KT : (t0 + plain) * KT; key0 < last; key0 += 64) {
                const int mine = min(key0 + lane, last - 1);
                const char* vp = value_row(mine);
                u16x2_t top{};
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    const u32x4_t v = ld16(vp + 16 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, v[j] & 0x7fff7fffu));
                }
                uint64_t todo = __ballot(key0 + lane < last && max(top[0], top[1]) >= kInf16<T> &&
                                         mine / 32 % (KT / 32) / NKB == kw);
#pragma unroll 1
                for (; todo != 0; todo &= todo - 1) {
                    const int key = key0 + __builtin_ctzll(todo), node = key - ctx;
                    const bool see = node < 0 || (node < kTreeMaxCols && (words[node >> 5] >> (node & 31) & 1u) != 0);
                    const char* kp = value_row(key) + 8 * hi;
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int rg = 0; rg < 4; ++rg) {
                            const u32x2_t y = ld8(kp + 2 * (32 * db + 8 * rg));
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float f = (e & 1) ? hi16<T>(y[e >> 1]) : lo16<T>(y[e >> 1]);
                                if (see && !(fabsf(f) < kPosInf)) x[db][4 * rg + e] += f;
                            }
                        }
                }
            }
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!(fabsf(x[db][r]) < kPosInf)) oacc[db][r] = x[db][r];
        }

        if (KW > 1) {
            // the waves of other keys leave theirs in the ring, lane by lane
            __syncthreads();
            if (kw > 0) {
                char* own = smem + ((kw - 1) * RW + rw) * kShare;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int rg = 0; rg < 4; ++rg)
                        *reinterpret_cast<f32x4_t*>(own + (db * 4 + rg) * 1024 + lane * 16) =
                            f32x4_t{oacc[db][4 * rg], oacc[db][4 * rg + 1], oacc[db][4 * rg + 2], oacc[db][4 * rg + 3]};
                float* sums = reinterpret_cast<float*>(own + DB * 4096) + lane;
                sums[0] = m_run;
                sums[64] = lt;
            }
            __syncthreads();
            if (kw == 0) {
#pragma unroll 1
                for (int i = 1; i < KW; ++i) {
                    const char* other = smem + ((i - 1) * RW + rw) * kShare;
                    const float* sums = reinterpret_cast<const float*>(other + DB * 4096) + lane;
                    const float m = nan_max(sums[0], m_run), mu = m == kNegInf ? 0.f : m;
                    const float a = __builtin_amdgcn_exp2f(m_run - mu), b = __builtin_amdgcn_exp2f(sums[0] - mu);
                    lt = lt * a + sums[64] * b;
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
        // (the row again, from the lane: nothing of it is held through the loops; NaN is not
        // <= 0; rows that see nothing: 0 and -inf)
        int l2 = l32;
        asm volatile("" : "+v"(l2));
        const int orow = rt * ROWS + 32 * rw + l2;
        if (kw == 0 && orow < n_rows) {
            CParams* p2 = params();
            const int otok = orow / p2->g, ohead = hk * p2->g + orow - otok * p2->g;
            const float inv = !(lt <= 0.f) ? 1.f / lt : 0.f;
            const float lse = !(lt <= 0.f) ? m_run * kLn2 + logf(lt) : kNegInf;
            if (whole) {
                const int64_t rh = (int64_t)(q0 + otok) * p2->hq + ohead;
                uint16_t* op = p2->o + rh * D;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int rg = 0; rg < 4; ++rg)
                        st8(op + 32 * db + 8 * rg + 4 * hi,
                            u32x2_t{T::pack2(oacc[db][4 * rg] * inv, oacc[db][4 * rg + 1] * inv),
                                    T::pack2(oacc[db][4 * rg + 2] * inv, oacc[db][4 * rg + 3] * inv)});
                if (p2->lse != nullptr && hi == 0) p2->lse[rh] = lse;
            } else {
                const int64_t pr = (int64_t)(2 * id + (t0 == 0 ? 1 : 0)) * ROWS + 32 * rw + l2;
                float* op = p2->part_o + pr * D;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int rg = 0; rg < 4; ++rg)
                        *reinterpret_cast<f32x4_t*>(op + 32 * db + 8 * rg + 4 * hi) =
                            f32x4_t{oacc[db][4 * rg] * inv, oacc[db][4 * rg + 1] * inv, oacc[db][4 * rg + 2] * inv,
                                    oacc[db][4 * rg + 3] * inv};
                if (hi == 0) p2->part_lse[pr] = lse;
            }
        }
        __syncthreads();                               // (the ring and the masks are free again)
    }
    if (threadIdx.x == 0) params()->desc[id] = begun;
}

// The rows of a unit that several pieces share: half a wave per row, its lanes over
// the head dim, O = sum_z w_z O_z / sum_z w_z, w_z = exp(lse_z - max lse), in the
// pieces' order. Bound by the latency of its loads: the rows of 8 pieces are under way
// before their weights are known. (Two or four rows per half wave, for fewer workgroups: 2
// and 4 us slower over 11 pieces.)
template <typename T, int D, int ROWS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeKParams p) {
    constexpr int NE = D / 32, U = 8;                  // columns of a lane, pieces at a time
    typedef float fe_t __attribute__((ext_vector_type(NE)));
    const int id = blockIdx.x;
    const int4 d = p.desc[id];
    const int rr = blockIdx.y * 8 + (threadIdx.x >> 5), l32 = threadIdx.x & 31;
    const int row = d.z * ROWS + rr, n = d.w;
    if (n == 0 || row >= d.y) return;
    // piece z of the unit: the first one's second place, the others' first
    auto place = [&](int z) { return (2 * (id + (int64_t)z * p.hkv * p.side) + (z == 0 ? 1 : 0)) * ROWS + rr; };
    float m = kNegInf, sum = 0.f;
    fe_t acc{};
    for (int z0 = 0; z0 < n; z0 += U) {
        float l[U];
        fe_t o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t pr = place(min(z0 + u, n - 1));
            l[u] = p.part_lse[pr];
            o[u] = *reinterpret_cast<const fe_t*>(p.part_o + pr * D + NE * l32);
        }
        float mz = m;
#pragma unroll
        for (int u = 0; u < U; ++u) mz = nan_max(z0 + u < n ? l[u] : kNegInf, mz);
        if (mz == kNegInf) continue;                   // (nothing seen so far)
        const float corr = m == kNegInf ? 0.f : __expf(m - mz);
        acc *= corr;
        sum *= corr;
        m = mz;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (z0 + u >= n || l[u] == kNegInf) continue;
            const float wgt = __expf(l[u] - m);
            sum += wgt;
            acc += wgt * o[u];
        }
    }
    const float inv = !(sum <= 0.f) ? 1.f / sum : 0.f;
    const int tok = row / p.g, head = id / p.side % p.hkv * p.g + row - tok * p.g;
    const int64_t rh = (int64_t)(d.x + tok) * p.hq + head;
    uint32_t* out = reinterpret_cast<uint32_t*>(p.o + rh * D + NE * l32);
#pragma unroll
    for (int e = 0; e < NE; e += 2) out[e / 2] = T::pack2(acc[e] * inv, acc[e + 1] * inv);
    if (p.lse != nullptr && l32 == 0) p.lse[rh] = !(sum <= 0.f) ? m + logf(sum) : kNegInf;
}

template <typename T, int D, int NW, int RW, int KT>
hipError_t launch_rows(const TreeArgs& a, TreeKParams p, hipStream_t st) {
    constexpr int ROWS = 32 * RW;
    char* ws = (char*)a.workspace;
    p.pieces = a.plan.pieces;
    p.side = a.plan.side;
    const size_t grid = (size_t)p.pieces * p.hkv * p.side;
    p.desc = (int4*)ws;
    p.part_lse = (float*)(ws + grid * sizeof(int4));
    p.part_o = p.part_lse + grid * 2 * ROWS;
    hipLaunchKernelGGL((tree_kernel<T, D, NW, RW, KT>), dim3((unsigned)grid), dim3(NW * 64), 0, st, p);
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
    if (a.plan.rows == 64) return launch_rows<T, D, 4, 2, 64>(a, p, st);
    if (a.plan.rows == 128) return launch_rows<T, D, 4, 4, 64>(a, p, st);
    return launch_rows<T, D, 8, 8, 128>(a, p, st);
}

}  // namespace

// Rows of a workgroup: the fewest that hold a sequence's max_q * g rows of a kv head,
// so that the others' matrix work is not done for nothing, from 64 up to 256. D = 128, us:
// 16 rows (16 sequences of 4 drafted tokens over 128 to 4096 keys, 32/8 heads) 35.4 with 64, 37.3
// with 128; 128 rows (8 of 32 over 16384 to 32768) 188 with 128, 290 with 256; 512 rows (4
// of 64 over 32768 to 98304, 64/8 heads) 678 with 256, 687 with 128, which read the cache
// twice as often. (32 rows against 128-key tiles, one workgroup a CU, while weights had one part:
// 64 sequences of 1024 to 16384 keys 388 against 392, one of 500 17.5 against 14.3: there are none.)
TreePlan make_tree_plan(const Geometry& g, int max_q, int64_t max_kv, int cus) {
    TreePlan plan;
    const int64_t rows = (int64_t)std::max(max_q, 1) * g.g;
    plan.rows = rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    const int kt = plan.rows == 256 ? 128 : 64;
    // row tiles of a head side by side, where most sequences have that many
    const int64_t most = (rows + plan.rows - 1) / plan.rows;
    const int64_t usual = ((g.total_q * g.g + g.num_seqs - 1) / g.num_seqs + plan.rows - 1) / plan.rows;
    plan.side = most <= 8 && 4 * usual >= 3 * most ? (int)most : 1;
    // as many pieces as the GPU holds workgroups for, or as there are tiles by the bounds
    const int64_t held = (int64_t)cus * (plan.rows == 256 ? 1 : 2);
    const int64_t full = std::max<int64_t>(1, held / ((int64_t)g.hkv * plan.side));
    const int64_t units = (int64_t)g.num_seqs * ((most + plan.side - 1) / plan.side);
    const int64_t tiles = std::max<int64_t>(1, (max_kv + kt - 1) / kt);
    plan.pieces = (int)(units >= full ? full : std::min(full, units * tiles));
    plan.bytes = (size_t)plan.pieces * g.hkv * plan.side * (16 + 2 * (size_t)plan.rows * ((size_t)g.d + 1) * sizeof(float));
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
