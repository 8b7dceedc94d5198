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
//   * P s_v, which spans fp32's range, goes into the P V product as the sum of three
//     bf16 values: all 24 bits of it. (Two of them, 16 bits, left results of up to 2^-18 of
//     sum P |v| off, which shows where weights next to each other cancel; the third costs
//     0.7% of a long stream's time (64 sequences of 8192-65536 keys, 785 -> 791 us) and 3%
//     of a short call's (16 of 128-2048, 18.4 -> 19.0). Up to 5 rows would have room for
//     the parts as columns of one product: no faster, its branch costs what it saves.)
//   * One wave takes one kv head, the waves of a workgroup neighbouring heads of
//     the same tokens, so that whole token rows are read at about the same time
//     (one head's 128 bytes of each row at a time stream at 5.0 TB/s, 8 heads' at
//     6.0; the arithmetic is hidden in both: without it the times are within 3%).
//     With fewer kv heads than waves the others take the next tiles.
//   * Tiles of 32 keys go straight from HBM into the wave's LDS (two of them in
//     turn, no workgroup barriers), K as rows for the operand reads, V for the
//     transposing reads (ds_read_b64_tr_b8). Page lookups and scales are fetched 64
//     blocks at a time, the next ones while the current tiles stream.
//   * The work is cut into equal pieces over all sequences, one per workgroup that
//     the GPU holds, found on the device from the offsets (no host read): a piece may
//     end one sequence and begin the next. A sequence inside one piece is written
//     directly, the others as normalised partials for the combine kernel.
#include "cache8.h"
#include "common.h"
#include "kernels.h"
#include "../../include/mtlattn_capi.h"

namespace mtlattn {

namespace {

struct Dec8Params {
    const uint16_t* q; int64_t q_rs;
    const uint8_t* k; const uint8_t* v; int64_t k_rs, v_rs;
    const float* k_scale; const float* v_scale;
    const int* block_table; int64_t bt_stride;
    int page_size, page_log2, block_log2, num_pages;   // page_log2: -1 where the page is no power of two
    const int* cu_q; const int* cu_kv;
    const float* bias; int64_t bias_qs, bias_hs, bias_cols, bias_ss, bias_rows;
    int64_t total_q, total_kv;
    int num_seqs, hq, hkv, g, hpb, n_hg;
    int hw_log2;        // kv heads of a workgroup
    int pieces;         // pieces of the work (0: a sequence each)
    int unit_log2;      // keys of a unit: 32 * waves that share a head
    int rpw;            // heads of a row that a workgroup of the combine takes
    float scale_log2;
    int causal, window, bias_v4;
    float* o_part; float* lse_part;     // [hkv][n_hg][pieces][2][16] rows: of the sequence that an earlier
                                        // piece began, of the one that begins in this piece and goes on
    uint16_t* out; float* lse_out;
};

// The kernels read their parameters where they lie. A fresh pointer (params) keeps
// the compiler from holding a loop's worth of them, and of what follows from them, in
// registers: it put up to 86 scalars into lanes of vector registers before the first
// load (32 sequences of up to 16384 keys, window 2048, 16 heads, D = 64: 34.8 us, 31.7
// with a fresh pointer). 32 to 54 still go there, by instance, none to memory.
typedef const __attribute__((address_space(4))) Dec8Params CParams;
__device__ inline CParams* params() {
    uint64_t a = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return (CParams*)a;
}

constexpr int kKT = 32;                 // keys per tile

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Lane l's pointer, as a scalar.
__device__ inline const uint8_t* lane_pointer(uint64_t p, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)p, l), hi = __builtin_amdgcn_readlane((int)(p >> 32), l);
    return (const uint8_t*)((uint64_t)hi << 32 | lo);
}

// The sequences [g0, g0 + 64), one per lane: keys, queries, first key that a query
// sees (rounded down to a tile), and units of work, with their sum up to and with
// each lane. Sequences without queries have no work.
struct SeqGroup {
    int k0, k1, q0, q1;                 // offsets, as they are read
    int len, q_start, q_len, lo, n, sum;
    __device__ inline void fetch(CParams* p, int s) {
        s = min(s, p->num_seqs - 1);
        k0 = p->cu_kv[s];
        k1 = p->cu_kv[s + 1];
        q0 = p->cu_q[s];
        q1 = p->cu_q[s + 1];
    }
    __device__ inline void finish(CParams* p) {
        const int tk = (int)p->total_kv, tq = (int)p->total_q;
        k0 = min(max(k0, 0), tk);
        q_start = min(max(q0, 0), tq);
        len = min(min(max(k1, k0), tk) - k0, 0x7fff0000);    // (room for a few tiles in an int)
        q_len = min(max(q1, q_start), tq) - q_start;
        // (64 bits: a window may be any positive int, and q_len longer than len)
        lo = p->window > 0 ? (int)max((int64_t)len - q_len - p->window + 1, (int64_t)0) & ~(kKT - 1) : 0;
        sum = n = q_len > 0 ? (len - lo + (1 << p->unit_log2) - 1) >> p->unit_log2 : 0;
    }
    __device__ inline void scan(CParams* p, int g0, int lane) {
        finish(p);
        if (g0 + lane >= p->num_seqs) n = 0;
        sum = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(sum, o);
            if (lane >= o) sum += y;
        }
    }
    __device__ inline void load(CParams* p, int g0, int lane) {
        fetch(p, g0 + lane);
        scan(p, g0, lane);
    }
    __device__ inline int total() const { return __builtin_amdgcn_readlane(sum, 63); }
};
__device__ inline int wave_sum(int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
    return uniform(x);
}

// The units of all sequences after the first group, whose own are `work`. Four groups'
// offsets are under way at once.
__device__ inline int all_units(CParams* p, int work, int lane) {
    int n = 0;
    for (int g0 = 64; g0 < p->num_seqs; g0 += 256) {
        SeqGroup more[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) more[i].fetch(p, g0 + 64 * i + lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            more[i].finish(p);
            n += g0 + 64 * i + lane < p->num_seqs ? more[i].n : 0;
        }
    }
    return work + (p->num_seqs > 64 ? wave_sum(n) : 0);
}
// Units of a piece: all work in p->pieces equal ones.
__device__ inline int piece_units(CParams* p, int work) { return max((work + p->pieces - 1) / p->pieces, 1); }

// Waits until at most N of this wave's vector memory operations are pending; LDS
// reads stay behind it.
template <int N>
__device__ inline void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// All of this wave's LDS reads are done.
__device__ inline void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// Direct loads of 16 bytes a lane into LDS from per-lane addresses (common.h).
__device__ inline void lds_dma16(const void* gptr, const char* lds) {
    const uint32_t a = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(gptr), "{m0}"(a) : "memory");
}

typedef int v2i32_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i32_t lds_v2i32_t;
// 8 rows x 16 columns of bytes transposed within each 16-lane group: lane 2 e + q
// addresses row e at columns 8 q .., lane i receives column i of the 8 rows.
__device__ inline u32x2_t read_tr8(const char* p) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i32_t*)p));
}

// max / sum over the lanes that share lane & 15
__device__ inline float quad_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ inline float quad_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// A tile of 32 keys of one kv head in LDS: rows of D codes, K then V, each row's
// 16-byte chunks XOR-swizzled so that what is read at once falls on distinct
// banks (256 bytes hold 256 / D rows): K operands read one chunk of rows 0 .. 15,
// V's transposing reads one chunk of rows {4 lg .. + 3, 16 + 4 lg .. + 3} of two
// neighbouring lg.
template <int D>
struct Tile8 {
    static constexpr int kBytes = 2 * kKT * D, kV = kKT * D;
    static constexpr int kLoadRows = 1024 / D;                   // rows of one direct load
    static constexpr int kPerBlock = 16 / kLoadRows;             // loads of a 16-key block
    static constexpr int kLoads = 4 * kPerBlock;                 // of a tile, K and V
    __device__ static inline int swz_k(int row) { return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
    __device__ static inline int swz_v(int row) {
        return D == 128 ? ((row >> 1) & 3) | ((row >> 4) << 2) : ((row >> 2) & 1) | ((row >> 4) << 1);
    }
};

template <typename T, typename C, int D, bool BIAS, int NW>
// (D = 64, 8 waves: two workgroups on a CU)
__global__ __launch_bounds__(NW * 64, D == 64 && NW == 8 ? 4 : 2) void decode8_kernel(Dec8Params) {
    CParams* p = params();
    using Tile = Tile8<D>;
    constexpr int KB = 2, NC = D / 64, DB = D / 16;
    constexpr int TPV = 64 / KB;                     // tiles whose lookups are fetched at once
    constexpr int OROW = D * 4 + 16;                 // bytes of an fp32 O row in LDS (padded)
    constexpr int TB = Tile::kBytes + (BIAS ? KB * 1024 : 0);
    constexpr int LOADS = Tile::kLoads + (BIAS ? KB : 0);        // direct loads of a tile
    constexpr int WB = 2 * TB + 3 * 256;             // per wave: two tiles, page table, scales of K and V
    static_assert(2 * TB >= 16 * OROW, "the rows of O take the tiles' place");
    __shared__ __attribute__((aligned(256))) char smem[NW * WB + NW * 32 * 4];
    float* ml = reinterpret_cast<float*>(smem + NW * WB);        // [NW][16] row max (log2), [NW][16] row sum

    const int w = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n16 = lane & 15, lg = lane >> 4;

    // 8 neighbouring pieces on the 8 XCDs, the heads of a piece one after the other on its own
    const int piece = 8 * blockIdx.z + blockIdx.x;
    if (piece >= (p->pieces > 0 ? p->pieces : p->num_seqs)) return;
    SeqGroup grp;                                    // (offsets under way, lane constants meanwhile)
    grp.fetch(p, p->pieces > 0 ? lane : piece);
    const int hw_log2 = p->hw_log2, hw = 1 << hw_log2, TW = NW >> hw_log2, hkgs = p->hkv >> hw_log2;
    const int hgi = p->n_hg == 1 ? 0 : blockIdx.y / hkgs;
    const int hk = ((int)blockIdx.y - hgi * hkgs) * hw + (w & (hw - 1)), tw = w >> hw_log2;   // head; tiles tw, tw + TW, ..

    const uint8_t* kbase = p->k + (int64_t)hk * D;
    const uint8_t* vbase = p->v + (int64_t)hk * D;
    const int bt_last = (int)min(p->bt_stride, (int64_t)0x7fffffff) - 1;
    // direct loads: lane l fills chunk position l % (D / 16) of row l / (D / 16)
    const uint32_t k_rs = (uint32_t)p->k_rs, v_rs = (uint32_t)p->v_rs;
    const int64_t k_half = Tile::kLoadRows * p->k_rs, v_half = Tile::kLoadRows * p->v_rs;
    const int lrow = lane / (D / 16), lpos = lane % (D / 16);
    uint32_t koff[Tile::kPerBlock], voff[KB];
#pragma unroll
    for (int i = 0; i < Tile::kPerBlock; ++i)
        koff[i] = (uint32_t)lrow * k_rs + 16u * (uint32_t)(lpos ^ Tile::swz_k(Tile::kLoadRows * i + lrow));
#pragma unroll
    for (int b = 0; b < KB; ++b) voff[b] = (uint32_t)lrow * v_rs + 16u * (uint32_t)(lpos ^ Tile::swz_v(16 * b + lrow));
    char* tiles = smem + w * WB;
    char* look = tiles + 2 * TB;                     // page table entries, s_k, s_v: 64 each
    // operand reads, from a tile's start
    const int kread = n16 * D + 16 * (lg ^ Tile::swz_k(n16));    // chunk lg; lg + 4 is this ^ 64
    const int ve = (lane & 15) >> 1, vkey = ve < 4 ? 4 * lg + ve : 12 + 4 * lg + ve;
    const int vread = Tile::kV + vkey * D + 16 * Tile::swz_v(vkey) + 8 * (lane & 1);   // chunk 0; db is this ^ 16 db

    // units [u, u_end) of the work, from sequence group g0 on (`before` units before it)
    int g0 = 0, before = 0, u, u_end;
    if (p->pieces > 0) {
        grp.scan(p, 0, lane);
        const int work = all_units(p, grp.total(), lane), units = piece_units(p, work);
        if ((int64_t)piece * units >= work) return;
        u = piece * units;
        u_end = min(work - u, units) + u;
        while (before + grp.total() <= u && g0 + 64 < p->num_seqs) {
            before += grp.total();
            g0 += 64;
            grp.load(p, g0, lane);
        }
    } else {
        g0 = piece;                                  // (every lane holds the sequence)
        grp.finish(p);
        u = 0;
        u_end = max(1, uniform(grp.n));
    }

    while (u < u_end) {
        p = params();
        // the sequence of unit u
        int l = 0;
        if (p->pieces > 0) {
            uint64_t past = __ballot(before + grp.sum > u);
            while (past == 0 && g0 + 64 < p->num_seqs) {
                before += grp.total();
                g0 += 64;
                grp.load(p, g0, lane);
                past = __ballot(before + grp.sum > u);
            }
            if (past == 0) break;
            l = __builtin_ctzll(past);
        }
        const int s = g0 + l, kv_len = __builtin_amdgcn_readlane(grp.len, l), n_units = __builtin_amdgcn_readlane(grp.n, l);
        const int q_len = __builtin_amdgcn_readlane(grp.q_len, l), q_start = __builtin_amdgcn_readlane(grp.q_start, l);
        const int lo = __builtin_amdgcn_readlane(grp.lo, l);
        const int t0 = p->pieces > 0 ? before + __builtin_amdgcn_readlane(grp.sum, l) - n_units : 0;
        const bool begins = u == t0, whole = p->pieces == 0 || (begins && t0 + n_units <= u_end);
        const int ks = lo + ((u - t0) << p->unit_log2);
        const int ke = min(kv_len, lo + (min(n_units, u_end - t0) << p->unit_log2));
        u = p->pieces > 0 ? t0 + n_units : u_end;
        if (q_len == 0) continue;
        const int coff = kv_len - q_len;

        // Row n of the 16 columns: head hh = n / q_len of this group, query n % q_len.
        // (columns past the rows repeat row 0; nothing reads them)
        const int rows = min(p->hpb * q_len, 16);
        const bool row_ok = n16 < rows;
        const int hh = row_ok ? (q_len == 1 ? n16 : n16 / q_len) : 0;
        const int qi = row_ok ? n16 - hh * q_len : 0;
        const int head = hk * p->g + hgi * p->hpb + hh;
        const int64_t grow = q_start + qi;
        // keys [first, first + width) are the row's
        const int first = p->window > 0 ? (int)max((int64_t)qi + coff - p->window + 1, (int64_t)ks) : ks;
        const uint32_t width = (uint32_t)max(0, (p->causal ? min(ke, qi + coff + 1) : ke) - first);

        // operand kc = 2 c + h: codes 64 c + 16 lg + 8 h .. + 7 of a row
        u32x4_t qf[2 * NC];
        {
            const uint16_t* qp = p->q + grow * p->q_rs + (int64_t)head * D + 16 * lg;
#pragma unroll
            for (int kc = 0; kc < 2 * NC; ++kc) qf[kc] = ld16(qp + 64 * (kc >> 1) + 8 * (kc & 1));
        }
        const float* brow = nullptr;
        if (BIAS)
            brow = p->bias + bias_row_offset(grow, s, q_start, p->bias_qs, p->bias_ss, p->bias_rows) +
                   (int64_t)head * p->bias_hs;

        const int n_tiles = ke > ks ? (ke - ks + kKT - 1) / kKT : 0;
        const int n_my = n_tiles > tw ? (n_tiles - tw + TW - 1) >> (NW == 8 ? 3 - hw_log2 : 2 - hw_log2) : 0;
        const int* bt = p->block_table + (int64_t)s * p->bt_stride;

        // Lookups of tiles [i0, i0 + TPV): lane l has block l % KB of tile i0 + l / KB
        // (blocks past the item's end: its last block). Addresses of the block's first
        // row of this head from its page, and the scales, which arrive in LDS.
        uint64_t vkp = 0, vvp = 0;
        float vks = 0.f, vvs = 0.f;
        bool inf_scale = false;                          // one of V's was an infinity
        auto lookup_key = [&](int i0) { return min(ks + (tw + (i0 + lane / KB) * TW) * kKT + 16 * (lane % KB), ke - 1) & ~15; };
        auto page_of = [&](int key) { return p->page_log2 >= 0 ? key >> p->page_log2 : key / p->page_size; };
        auto table_entry = [&](int i0) { return bt + min(page_of(lookup_key(i0)), bt_last); };
        auto find_rows = [&](int i0, int page) {
            const int key = lookup_key(i0);
            const int row = (min(max(page, 0), p->num_pages - 1) - page_of(key)) * p->page_size + key;
            vkp = (uint64_t)(kbase + (int64_t)row * p->k_rs);
            vvp = (uint64_t)(vbase + (int64_t)row * p->v_rs);
            const int64_t sc = (int64_t)(row >> p->block_log2) * p->hkv + hk;
            lds_dma4(p->k_scale + sc, look + 256);
            lds_dma4(p->v_scale + sc, look + 512);
        };
        // starts the loads of tile i of this wave into buf
        auto load = [&](int i, char* buf) __attribute__((always_inline)) {
            const int kt = ks + (tw + i * TW) * kKT;
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const uint8_t* kp = lane_pointer(vkp, (i % TPV) * KB + b);
                const uint8_t* vp = lane_pointer(vvp, (i % TPV) * KB + b);
                char* kd = buf + b * 16 * D;
                char* vd = buf + Tile::kV + b * 16 * D;
                if (kt + kKT <= ke) {
#pragma unroll
                    for (int m = 0; m < Tile::kPerBlock; ++m) {
                        lds_dma16s(kp + m * k_half, koff[m], kd + m * 1024);
                        lds_dma16s(vp + m * v_half, voff[b], vd + m * 1024);
                    }
                } else {
                    // rows past the end: the last one again (masked to P = 0)
                    const int last = ke - 1 - min(kt + 16 * b, (ke - 1) & ~15);
#pragma unroll
                    for (int m = 0; m < Tile::kPerBlock; ++m) {
                        const uint32_t r = (uint32_t)min(Tile::kLoadRows * m + lrow, last) - (uint32_t)lrow;
                        lds_dma16s(kp, koff[m] + r * k_rs, kd + m * 1024);
                        lds_dma16s(vp, voff[b] + r * v_rs, vd + m * 1024);
                    }
                }
                // the lane's 4 keys of the block, where the tile lies within the columns
                if (BIAS)
                    lds_dma16(p->bias_v4 && kt + kKT <= p->bias_cols ? (const void*)(brow + kt + 16 * b + 4 * lg) : (const void*)kp,
                              buf + Tile::kBytes + b * 1024);
            }
        };

        float m_run = kNegInf, l_run = 0.f;
        f32x4_t oacc[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};

        auto step = [&](int i, const char* buf) __attribute__((always_inline)) {
            const int kt = ks + (tw + i * TW) * kKT;
            // (all of the tile's LDS reads at once: V's are not waited for before P)
            u32x4_t kc[KB][NC];
            u32x2_t vc[DB];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int c = 0; c < NC; ++c) kc[b][c] = ld16(buf + b * 16 * D + (kread ^ (64 * c)));
#pragma unroll
            for (int db = 0; db < DB; ++db) vc[db] = read_tr8(buf + (vread ^ (16 * db)));
            // S^T = K Q^T, 16 keys at a time
            f32x4_t sc[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                sc[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const u32x4_t k = kc[b][c];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const u32x2_t a = C::template unpack4<T>(k[2 * h]), a2 = C::template unpack4<T>(k[2 * h + 1]);
                        sc[b] = mfma16<T>(u32x4_t{a[0], a[1], a2[0], a2[1]}, qf[2 * c + h], sc[b]);
                    }
                }
            }
            float vs[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int at = (i % TPV) * KB + b;
                const float k_sc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vks), at));
                vs[b] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vvs), at));
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[b][r] *= k_sc;
                if (BIAS) {
                    f32x4_t bb = *reinterpret_cast<const f32x4_t*>(buf + Tile::kBytes + b * 1024 + 16 * lane);
                    if (!(p->bias_v4 && kt + kKT <= p->bias_cols)) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int64_t key = kt + 16 * b + 4 * lg + r;
                            bb[r] = key < p->bias_cols ? brow[key] : 0.f;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[b][r] = fmaf(bb[r], kLog2e, sc[b][r]);
                }
            }
            // (rows' window bands start at qi + coff - W + 1 <= coff + q_len - W)
            if ((kt + kKT > ke) || (p->causal && kt + kKT - 1 > coff) || (p->window > 0 && kt < coff + q_len - p->window)) {
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    bool sees = false;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool in = (uint32_t)(kt + 16 * b + 4 * lg + r - first) < width;
                        sees = sees || in;
                        sc[b][r] = in ? sc[b][r] : kNegInf;
                    }
                    vs[b] = sees ? vs[b] : 0.f;
                }
                // (0 * NaN: the keys before a window may lie in pages of another use by now)
                if (C::code == E4M3::code) {
                    uint32_t nan = 0;
#pragma unroll
                    for (int db = 0; db < DB; ++db) nan |= E4M3::nans(vc[db][0]) | E4M3::nans(vc[db][1]);
                    if (__any(nan != 0)) {
                        // Rows that see a NaN become one, by the count of those they see in each
                        // column; the codes themselves become 0.
                        u32x4_t see;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = kt + 16 * (e >> 1) + 4 * lg + 2 * (e & 1) - first;
                            see[e] = ((uint32_t)key < width ? 0x3f80u : 0u) | ((uint32_t)key + 1 < width ? 0x3f800000u : 0u);
                        }
#pragma unroll
                        for (int db = 0; db < DB; ++db) {
                            const uint32_t x = E4M3::nans(vc[db][0]), y = E4M3::nans(vc[db][1]);
                            const u32x2_t a = E4M3::unpack4<BF16>(x * 0x38u), b = E4M3::unpack4<BF16>(y * 0x38u);
                            const f32x4_t count = mfma16<BF16>(u32x4_t{a[0], a[1], b[0], b[1]}, see, f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                            for (int r = 0; r < 4; ++r) oacc[db][r] = count[r] > 0.f ? __builtin_nanf("") : oacc[db][r];
                            vc[db] &= ~u32x2_t{x * 0xffu, y * 0xffu};
                        }
                    }
                }
            }
            float mx = kNegInf;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[b][r]);
            mx = quad_max(mx);
            if (__any(mx > m_run)) {
                const float m_new = fmaxf(m_run, mx);
                const float corr = __builtin_amdgcn_exp2f(m_run - (m_new == kNegInf ? 0.f : m_new));
                m_run = m_new;
                l_run *= corr;
#pragma unroll
                for (int db = 0; db < DB; ++db) oacc[db] *= corr;
            }
            const float m_use = m_run == kNegInf ? 0.f : m_run;
            // P^T operand, slots j < 4: key 4 lg + j, then 16 + 4 lg + j - 4, in three parts of 8
            // bits each: the upper half of a float, of what it leaves (exact), and so on
            float wt[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] - m_use);
                l_run += x;
                wt[e] = x * vs[e >> 2];
            }
            u32x4_t pt[3];
#pragma unroll
            for (int i = 0; i < 3; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = __float_as_uint(wt[2 * e]), y = __float_as_uint(wt[2 * e + 1]);
                    pt[i][e] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                    wt[2 * e] -= __uint_as_float(x & 0xffff0000u);
                    wt[2 * e + 1] -= __uint_as_float(y & 0xffff0000u);
                }
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const u32x2_t x = C::template unpack4<BF16>(vc[db][0]), y = C::template unpack4<BF16>(vc[db][1]);
                const u32x4_t va = u32x4_t{x[0], x[1], y[0], y[1]};
#pragma unroll
                for (int i = 0; i < 3; ++i) oacc[db] = mfma16<BF16>(va, pt[i], oacc[db]);
            }
        };

        int page = n_my > 0 ? *table_entry(0) : 0;
        // nothing that the compiler counts stays pending (q, the page): its waits in
        // the loop would wait for the direct loads too, which it does not count
        wait_vmcnt<0>();
        // Two tiles of LDS in turn: tile i is computed while tile i + 1 is in flight, then
        // its place is loaded with tile i + 2. (Lookups between them are waited for early.)
#pragma clang loop unroll(disable)
        for (int i = -2; i < n_my; ++i) {
            char* buf = tiles + (i & 1) * TB;
            if (i >= 0) {
                if (i + 1 < n_my) wait_loads<LOADS>(); else wait_loads<0>();
                if (i % TPV == 0) {
                    vks = *reinterpret_cast<const float*>(look + 256 + 4 * lane) * p->scale_log2;
                    vvs = *reinterpret_cast<const float*>(look + 512 + 4 * lane);
                    // (infinite ones come in after the loop)
                    inf_scale = inf_scale || __any(fabsf(vvs) == kPosInf);
                    vvs = fabsf(vvs) == kPosInf ? 0.f : vvs;
                }
                step(i, buf);
                wait_lds();
            }
            if (i + 2 < n_my) {
                if ((i + 2) % TPV == 0) {
                    if (i >= 0) {
                        page = *reinterpret_cast<const int*>(look + 4 * lane);
                        wait_lds();
                    }
                    find_rows(i + 2, page);
                    if (i + 2 + TPV < n_my) lds_dma4(table_entry(i + 2 + TPV), look);
                }
                load(i + 2, buf);
            }
        }

        p = params();
        // A caller's own scales of V that are infinities: each key of theirs that a row sees
        // adds its codes times the infinity, whatever its weight but 0.
        if (inf_scale) {
#pragma clang loop unroll(disable)
            for (int j = 0; j < KB * n_my; ++j) {
                const int k0 = ks + (tw + j / KB * TW) * kKT + 16 * (j % KB);
                if (k0 >= ke) break;
                const int pg = min(max(bt[min(page_of(k0), bt_last)], 0), p->num_pages - 1);
                const int row = (pg - page_of(k0)) * p->page_size + k0;
                const float inf = p->v_scale[(int64_t)(row >> p->block_log2) * p->hkv + hk];
                if (fabsf(inf) != kPosInf) continue;
#pragma clang loop unroll(disable)
                for (int key = k0; key < min(k0 + 16, ke); ++key) {
                    if ((uint32_t)(key - first) >= width) continue;
                    float x = inf;
                    if (BIAS) x *= key < p->bias_cols && brow[key] == kNegInf ? 0.f : 1.f;
                    const uint8_t* vp = vbase + (int64_t)(row + key - k0) * p->v_rs + 4 * lg;
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        float f[4];
                        C::to_float4(*reinterpret_cast<const uint32_t*>(vp + 16 * db), f);
#pragma unroll
                        for (int r = 0; r < 4; ++r) oacc[db][r] += f[r] * x;
                    }
                }
            }
        }
        const float lt = quad_sum(l_run);
        // where row n of this wave's head goes: the output, or a partial
        auto out_row = [&](int n) {
            const int h2 = q_len == 1 ? n : n / q_len;
            return (int64_t)(q_start + n - h2 * q_len) * p->hq + hk * p->g + hgi * p->hpb + h2;
        };
        auto part_row = [&](int n) {
            return (((int64_t)(hk * p->n_hg + hgi) * p->pieces + piece) * 2 + (begins ? 1 : 0)) * 16 + n;
        };
        auto put_lse = [&](int n, float m, float lsum) {
            const float lse = !(lsum <= 0.f) ? m * kLn2 + logf(lsum) : kNegInf;
            if (!whole) p->lse_part[part_row(n)] = lse;
            else if (p->lse_out != nullptr) p->lse_out[out_row(n)] = lse;
        };
        if (TW == 1) {
            if (row_ok) {
                const float inv = !(lt <= 0.f) ? 1.f / lt : 0.f;
                if (whole) {
                    uint16_t* o = p->out + out_row(n16) * D + 4 * lg;
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const f32x4_t x = oacc[db] * inv;
                        st8(o + 16 * db, u32x2_t{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])});
                    }
                } else {
                    float* o = p->o_part + part_row(n16) * D + 4 * lg;
#pragma unroll
                    for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4_t*>(o + 16 * db) = oacc[db] * inv;
                }
                if (lg == 0) put_lse(n16, m_run, lt);
            }
        } else {
            // the waves of a head meet in LDS, in their tiles' place
            if (row_ok) {
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    *reinterpret_cast<f32x4_t*>(tiles + n16 * OROW + (16 * db + 4 * lg) * 4) = oacc[db];
                if (lg == 0) {
                    ml[w * 16 + n16] = m_run;
                    ml[(NW + w) * 16 + n16] = lt;
                }
            }
            __syncthreads();
            // one lane per row and 4 columns; the reads of all TW waves at once
            for (int t = tw * 64 + lane; t < rows * (D / 4); t += TW * 64) {
                const int n = t / (D / 4), d = 4 * (t % (D / 4));
                float mw[NW], lw[NW], m = kNegInf, lsum = 0.f;
                f32x4_t ow[NW], o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    const int v = (w & (hw - 1)) + (i < TW ? i : 0) * hw;
                    mw[i] = ml[v * 16 + n];
                    lw[i] = ml[(NW + v) * 16 + n];
                    ow[i] = *reinterpret_cast<const f32x4_t*>(smem + v * WB + n * OROW + d * 4);
                }
#pragma unroll
                for (int i = 0; i < NW; ++i) m = nan_max(mw[i], m);
                const float m_use = m == kNegInf ? 0.f : m;
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    const float wgt = __builtin_amdgcn_exp2f(mw[i] - m_use);
                    if (i < TW) {
                        lsum += wgt * lw[i];
                        o += wgt * ow[i];
                    }
                }
                o *= !(lsum <= 0.f) ? 1.f / lsum : 0.f;
                if (whole) st8(p->out + out_row(n) * D + d, u32x2_t{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])});
                else *reinterpret_cast<f32x4_t*>(p->o_part + part_row(n) * D + d) = o;
                if (d == 0) put_lse(n, m, lsum);
            }
            if (u < u_end) __syncthreads();
        }
        // rows past the 16 that max_seqlen_q promised: NaN (the combine's, of pieces)
        if (p->pieces == 0) {
            const int more = p->hpb * q_len - 16;
            for (int64_t t = threadIdx.x; t < (int64_t)more * hw * D; t += NW * 64) {
                const int64_t r = t / D;
                const int hs = (int)(r % hw), n = 16 + (int)(r / hw), d = (int)(t % D), h2 = n / q_len;
                const int64_t rh = (int64_t)(q_start + n - h2 * q_len) * p->hq + (hk - (w & (hw - 1)) + hs) * p->g + hgi * p->hpb + h2;
                p->out[rh * D + d] = T::from_float(__builtin_nanf(""));
                if (p->lse_out != nullptr && d == 0) p->lse_out[rh] = __builtin_nanf("");
            }
        }
    }
}

// Merges the partials of the pieces of a row's sequence with their LSEs: D / 4 lanes
// to a partial, the 1024 / D such groups of a workgroup on p->rpw heads of one row,
// the groups of a head taking its partials in turn with four loads of each in
// flight. Many rows have few pieces each (one head to a group: 4096 rows of about 5
// pieces 13 -> 8 us), few rows many (one wave that walked the 256 of a sequence of
// 131071 keys took 30 us). Rows of a sequence inside one piece are there already;
// rows of no sequence are left as they were.
template <typename T, int D, int NT>
__global__ __launch_bounds__(NT) void combine8_kernel(Dec8Params) {
    CParams* p = params();
    constexpr int TPR = D / 4, G = NT / TPR, U = 4;
    __shared__ __attribute__((aligned(16))) float so[G][D];
    __shared__ float sm[G], sl[G];
    const int tid = threadIdx.x, lane = tid & 63, split = G / p->rpw, per = p->hq / p->rpw;
    const int row = blockIdx.x / per, head = (blockIdx.x - row * per) * p->rpw + tid / (TPR * split);
    // the row's sequence, the units before it, and all work (four groups of 64 sequences
    // at once after the first: 1024 sequences of up to 4096 keys 830 -> 819 us)
    int s = -1, q_len = 0, q_start = 0, n_units = 0, t0 = 0, work = 0;
    auto take = [&](SeqGroup& grp, int at) __attribute__((always_inline)) {
        grp.finish(p);
        const int n = at < p->num_seqs ? grp.n : 0, behind = row - grp.q_start;
        work += n;
        t0 += behind >= grp.q_len ? n : 0;
        if (at < p->num_seqs && behind >= 0 && behind < grp.q_len) {
            s = at;
            q_len = grp.q_len;
            q_start = grp.q_start;
            n_units = n;
        }
    };
    SeqGroup grp;
    grp.fetch(p, lane);
    take(grp, lane);
    for (int g0 = 64; g0 < p->num_seqs; g0 += 256) {
        SeqGroup more[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) more[i].fetch(p, g0 + 64 * i + lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) take(more[i], g0 + 64 * i + lane);
    }
    const uint64_t in = __ballot(s >= 0);
    if (in == 0) return;
    const int own = __builtin_ctzll(in);
    q_len = __builtin_amdgcn_readlane(q_len, own);
    q_start = __builtin_amdgcn_readlane(q_start, own);
    n_units = __builtin_amdgcn_readlane(n_units, own);
    work = wave_sum(work);
    t0 = wave_sum(t0);
    const int units = piece_units(p, work);
    // (offsets that overlap may make more units than an int holds, here or in the decode:
    // whatever the sums, no partial but the workspace's)
    const int first = min(max(t0 / units, 0), p->pieces - 1);
    const int count = n_units > 0 ? min((t0 + n_units - 1) / units - first + 1, p->pieces - first) : 0;
    const int qi = row - q_start, hk = head / p->g, hh_full = head - hk * p->g;
    const int hgi = hh_full / p->hpb, n = (hh_full - hgi * p->hpb) * q_len + qi;
    // its partials: the second of `first`, then the first ones of the following pieces
    const int64_t base = (((int64_t)(hk * p->n_hg + hgi) * p->pieces + first) * 2) * 16 + n;
    const int g = tid / TPR, d = 4 * (tid % TPR);
    float m = kNegInf, l = 0.f;
    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int i0 = g % split; i0 < (n < 16 && count > 1 ? count : 0); i0 += split * U) {
        float li[U];
        f32x4_t oi[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(i0 + u * split, count - 1);
            const int64_t at = base + (int64_t)(i == 0 ? 1 : 2 * i) * 16;
            li[u] = p->lse_part[at];
            oi[u] = *reinterpret_cast<const f32x4_t*>(p->o_part + at * D + d);
        }
        float m_new = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            li[u] = i0 + u * split < count ? li[u] * kLog2e : kNegInf;
            m_new = nan_max(li[u], m_new);          // (a piece of NaN must not look empty)
        }
        const float m_use = m_new == kNegInf ? 0.f : m_new;
        const float corr = __builtin_amdgcn_exp2f(m - m_use);
        l *= corr;
        acc *= corr;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float wgt = __builtin_amdgcn_exp2f(li[u] - m_use);
            l += wgt;
            if (i0 + u * split < count) acc += wgt * oi[u];
        }
        m = m_new;
    }
    *reinterpret_cast<f32x4_t*>(&so[g][d]) = acc;
    if (d == 0) {
        sm[g] = m;
        sl[g] = l;
    }
    __syncthreads();
    if (g % split != 0 || (count == 1 && n < 16)) return;
    const int64_t rh = (int64_t)row * p->hq + head;
    float mt = kNegInf;
#pragma unroll
    for (int i = 0; i < G; ++i) mt = i < split ? nan_max(sm[(g + i) % G], mt) : mt;
    const float m_use = mt == kNegInf ? 0.f : mt;
    float lt = 0.f;
    f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < G; ++i) {
        if (i >= split) continue;
        const float wgt = __builtin_amdgcn_exp2f(sm[(g + i) % G] - m_use);
        lt += wgt * sl[(g + i) % G];
        o += wgt * *reinterpret_cast<const f32x4_t*>(&so[(g + i) % G][d]);
    }
    o *= !(lt <= 0.f) ? 1.f / lt : 0.f;
    float lse = !(lt <= 0.f) ? mt * kLn2 + logf(lt) : kNegInf;
    if (n >= 16) {                                  // more rows than max_seqlen_q promised
        lse = __builtin_nanf("");
        o = f32x4_t{lse, lse, lse, lse};
    }
    st8(p->out + rh * D + d, u32x2_t{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])});
    if (p->lse_out != nullptr && d == 0) p->lse_out[rh] = lse;
}

template <typename T, typename C, int D>
hipError_t launch_typed(Dec8Params p, hipStream_t st) {
    // the combine: groups of D / 4 lanes for a head's pieces (on average), eight each
    const int groups = 1024 / D;
    const bool many = p.pieces > 8 * groups * (int64_t)p.num_seqs;
    p.rpw = many ? 1 : groups;
    while (p.rpw > 1 && (p.hq % p.rpw != 0 || (int64_t)groups / p.rpw * 8 * p.num_seqs < p.pieces)) p.rpw /= 2;
    const int64_t octs = ((p.pieces > 0 ? p.pieces : p.num_seqs) + 7) / 8;
    const int64_t per = (int64_t)(p.hkv >> p.hw_log2) * p.n_hg, rh = p.total_q * p.hq;
    if (octs > 65535 || per > 65535 || rh > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid(8, (unsigned)per, (unsigned)octs);
    if (p.bias != nullptr) hipLaunchKernelGGL((decode8_kernel<T, C, D, true, 4>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((decode8_kernel<T, C, D, false, 8>), grid, dim3(512), 0, st, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.pieces == 0) return e;
    const dim3 cgrid((unsigned)(rh / p.rpw));
    if (many) hipLaunchKernelGGL((combine8_kernel<T, D, 1024>), cgrid, dim3(1024), 0, st, p);
    else hipLaunchKernelGGL((combine8_kernel<T, D, 256>), cgrid, dim3(256), 0, st, p);
    return hipGetLastError();
}

template <typename T, typename C>
hipError_t launch_dim(const Dec8Params& p, int d, hipStream_t st) {
    if (d == 128) return launch_typed<T, C, 128>(p, st);
    if (d == 64) return launch_typed<T, C, 64>(p, st);
    return hipErrorInvalidValue;
}

}  // namespace

Dec8Plan make_dec8_plan(const Geometry& g, int max_q, int64_t max_kv, int cus) {
    Dec8Plan plan;
    int hpb = 16 / (max_q > 0 ? max_q : 1);         // heads per 16-row group: largest divisor of g that fits
    if (hpb < 1) hpb = 1;
    if (hpb > g.g) hpb = g.g;
    while (g.g % hpb != 0) --hpb;
    plan.hpb = hpb;
    const int n_hg = g.g / hpb;
    // (with a bias, whose tiles are larger, 8 waves do not fit the LDS)
    plan.waves = g.bias != nullptr ? 4 : 8;
    if (g.window > 0) max_kv = std::min<int64_t>(max_kv, (int64_t)g.window + max_q - 1 + kKT - 1);
    auto heads = [&](int want) {                    // of a workgroup: at most `want`, a divisor of hkv
        int hw = std::min(want, plan.waves);
        while (g.hkv % hw != 0) hw /= 2;
        return hw;
    };
    const int64_t seq_heads = (int64_t)g.num_seqs * g.hkv * n_hg;
    if ((max_kv <= 1024 || (max_kv <= 2048 && seq_heads > 32)) && g.num_seqs <= 8 * 65535) {
        // One workgroup per sequence, no second launch; as many of its waves on a head as
        // the CUs have room for: a wave takes about 1 us per tile, which a bandwidth-bound
        // stream hides. bf16, D = 128, 32/8 heads, up to 1024 keys: 16 sequences 12.1 us
        // with 8 waves on a head, 17.4 with 4, 47.7 with 1; 64 26.0 / 22.9 / 50.5, 256
        // 84.7 / 69.3 / 66.4. Pieces took 16.8, 26.4 and 67.6; of up to 2048 keys (16, 64,
        // 256 sequences) 19.0, 37.9 and 136 against 18.7, 36.1 and 136-140, of up to 4096
        // (64) 62 against 69.
        int hw = 1;
        while (seq_heads > (int64_t)cus * hw && hw < plan.waves) hw *= 2;
        plan.hw = heads(hw);
    } else {
        // Pieces for every workgroup that the CUs hold, of whole token rows (8 heads); few
        // tiles (under 4 a wave) on fewer heads and more waves each, with fewer partials: one
        // sequence of 2048 keys 12.3 us with 2 heads, 17.4 with 8, 17.6 as a whole; four of
        // 4096 16.1 and 16.8.
        const double tiles = (double)g.num_seqs * (double)max_kv / kKT * g.hkv * n_hg;
        plan.hw = heads(tiles < cus * 8 * 4 ? 2 : 8);
        const int resident = g.bias == nullptr ? (g.d == 64 ? 2 : 1) : (g.d == 64 ? 3 : 1);
        // (a multiple of 8 where there are as many: a piece's workgroups share an XCD)
        const int per = g.hkv / plan.hw * n_hg, slots = cus * resident;
        plan.pieces = slots / 8 >= per ? slots / 8 / per * 8 : std::max(1, slots / per);
    }
    plan.rows = (int64_t)g.hkv * n_hg * plan.pieces * 2 * 16;
    return plan;
}

hipError_t launch_decode8(int dtype, int code, const Dec8Args& a, hipStream_t st) {
    const Geometry& g = a.geo;
    if (a.block_table == nullptr || a.block < 16 || a.plan.hw < 1 || a.plan.hpb < 1) return hipErrorInvalidValue;
    Dec8Params p;
    p.q = (const uint16_t*)a.q; p.q_rs = a.q_rs;
    p.k = a.k; p.v = a.v; p.k_rs = a.k_rs; p.v_rs = a.v_rs;
    p.k_scale = a.k_scale; p.v_scale = a.v_scale;
    p.block_table = a.block_table; p.bt_stride = a.bt_stride;
    p.page_size = a.page_size; p.num_pages = a.num_pages;
    p.page_log2 = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctz(a.page_size) : -1;
    p.block_log2 = __builtin_ctz(a.block);
    p.cu_q = g.cu_q; p.cu_kv = g.cu_kv;
    p.bias = g.bias; p.bias_qs = g.bias_qs; p.bias_hs = g.bias_hs; p.bias_cols = g.bias_cols;
    p.bias_ss = g.bias_ss; p.bias_rows = g.bias_rows;
    p.total_q = g.total_q; p.total_kv = g.total_kv;
    p.num_seqs = g.num_seqs; p.hq = g.hq; p.hkv = g.hkv; p.g = g.g;
    p.hpb = a.plan.hpb;
    p.n_hg = g.g / p.hpb;
    p.hw_log2 = __builtin_ctz(a.plan.hw);
    p.pieces = a.plan.pieces;
    p.unit_log2 = __builtin_ctz(kKT * (a.plan.waves / a.plan.hw));
    p.scale_log2 = g.scale * kLog2e;
    p.causal = g.causal;
    p.window = g.window;
    p.bias_v4 = g.bias != nullptr && ((uintptr_t)g.bias % 16 == 0) && g.bias_qs % 4 == 0 && g.bias_hs % 4 == 0 &&
                (g.bias_ss < 0 || g.bias_ss % 4 == 0);
    p.o_part = a.o_part;
    p.lse_part = a.lse_part;
    p.out = (uint16_t*)a.o;
    p.lse_out = a.lse;
    const bool e4m3 = code == MTLATTN_CODE_E4M3;
    if (dtype == MTLATTN_DTYPE_BF16)
        return e4m3 ? launch_dim<BF16, E4M3>(p, g.d, st)
                    : launch_dim<BF16, I8>(p, g.d, st);
    if (dtype == MTLATTN_DTYPE_F16)
        return e4m3 ? launch_dim<F16, E4M3>(p, g.d, st)
                    : launch_dim<F16, I8>(p, g.d, st);
    return hipErrorInvalidValue;
}

}  // namespace mtlattn
