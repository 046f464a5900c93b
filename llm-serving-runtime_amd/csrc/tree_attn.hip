// Attention of several new tokens per row over the paged cache for gfx950: the nodes of a tree of drafted
// tokens, or a chain of tokens, attend over the row's context and their own ancestors. (The reference drafts
// and verifies one token after the other through its decode path, runtime/phase2/worker_server.py:1010-1075.)
//
// out[b, i, h] = sum_j p_j v_j, p = softmax over the visible j of scale * q[b, h, i] . k_j. Token j of row b is
// visible to node i where j < ctx (ctx = seq_lens[b] - counts[b]), or where it is node j - ctx and mask[b, i, j - ctx] is
// set (no mask: j - ctx <= i).
//
// Bound: few query rows read K and V from HBM (4 D bytes a token and head); 256 query rows need as long for the products,
// and there the softmax, the addresses and the exchange through LDS come on top, since the waves of a SIMD hide little of each other's.
// Measured, a call: 32 rows of U[128, 4096] tokens with 16 nodes (G 4, D 128, 279 MB) 65 us, 4.3 TB/s; one row of 131,071
// tokens with 25 nodes (537 MB) 113 us, 4.7 TB/s; 8 rows of U[4096, 8192] tokens with 64 nodes (52 GFLOP) 80 us, 645 TFLOP/s;
// two chunks of 509 tokens over U[2048, 4096] (55 GFLOP) 79 us, 700 TFLOP/s; one row of 705 tokens with 5 nodes 16 us.
//
// Work decomposition. The G * T query rows of a (row, kv-head) share its K and V. A segment is a (row, kv-head,
// tile of R query rows), heads of a node next to each other; it holds ceil(visible tokens / 64) tiles. All segments form
// one sequence of tiles that is cut into equal ranges, one per workgroup, so that the chip drains evenly whatever
// the lengths are. A segment that one workgroup holds whole is written as output; of the others the pieces leave
// (m, l, output / l) in fp32 in the workspace (two slots per workgroup: its first piece and its last) and a second launch joins them.
//
// A workgroup is RW waves over the query rows (each RT tiles of 16) times TW waves over a tile's tokens. K and V of
// 64 tokens at a time are staged in LDS, double buffered, as rows whose 16-byte chunks are permuted by the row
// (chunk ^ row), which spreads the reads below over all banks. Scores are computed transposed (K rows as the A operand of
// v_mfma_f32_16x16x32, query rows as B): lane l holds the scores of tokens 4 * (l / 16) + [0, 4) of row l % 16 of two
// 16-token tiles, which is the k order of the B operand of the second product if V^T's columns are taken in that
// order too. ds_read_b64_tr_b16 gives them so: a group of 16 lanes reads 4 tokens x 16 dims and each lane gets one
// dim of the 4 tokens. So probabilities never leave their lane, and V needs no transposed copy.
//
// The softmax is the online one in fp32 on the exp2 scale; the reference maximum moves only when it would rise by more than
// 2^8. p enters the second product rounded to the element type, the only operand that the matrix cores take beside such V (in 32 bits
// a product runs at a sixteenth of the rate), and l sums the rounded values, so the weights still add up to 1: 2.2e-4 to 2.8e-4
// of the outputs' norm off in fp16 and 1.8e-3 to 2.2e-3 in bf16, where rounding the output alone is 2.1e-4 and 1.7e-3.
//
// Masked places have no effect whatever they hold: scores of invisible tokens are replaced by -inf, V of tokens past the end or
// of blocks outside the pool is staged as 0, and V of a drafted token that is not finite reaches only
// the rows that see it (nf_step below).
#include <type_traits>

#include "common.h"
#include "elt.h"

namespace mx {
namespace tree {

constexpr int kTok = 64;  // tokens per tile
// A segment counts for its tiles and this many more: its query rows, its masked tiles, its output (13,000 cycles next to a tile's
// 5,000, and the memory rests). 32 rows of U[128, 4096] tokens with 16 nodes each take 80 us where it counts for nothing (the
// ranges over the shortest rows hold six segments and end last), 70, 66, 64, 59, 56, 56, 58 with 1, 2, 3, 4, 6, 8, 10; 8 rows of
// 64 nodes 74, 72, 71, 69, 69, 67, 70, 71.
constexpr int kPieceTiles = 6;
constexpr int kCus = 256;
constexpr int kXcds = 8;
constexpr float kLazyLog2 = 8.0f;  // rescale only when the running max rises by more than 2^8
// The reference of the exponentials stands this much below the maximum it was taken from: p reaches 2^15 and no more, so an fp16 p
// loses nothing of a token that counts 2^-21 of the largest, and 2^-32 at most of one that counts less. (At the maximum
// itself 10^5 tokens of 2^-25 each, 0.4 %, would be rounded to 0.)
constexpr float kHeadLog2 = 7.0f;
constexpr float kLowest = -3.4028235e38f;
constexpr int kMfma = 0x8, kDsRead = 0x100;  // kinds of instructions, for the compiler's scheduler

struct Params {
    const _Float16* q;
    int64_t q_sb, q_sh, q_st;
    const _Float16* k;
    const _Float16* v;
    int64_t kv_sblk, kv_shead;
    const int32_t* bt;
    int64_t bt_sb;
    int max_blocks, bs_shift;
    const int32_t* seq_lens;
    const uint8_t* mask;  // null: a chain
    int64_t mask_sb, mask_st;
    const int32_t* counts;  // null: T
    int B, T, Hkv, G;
    int num_blocks;
    float scale_log2e;
    _Float16* out;
    int64_t o_sb, o_st, o_sh;
    float* part;  // [2 * workers][R][D + 4]: output / l, m, l
    int2* pieces;  // [segments]: 2 * the worker of a segment's first piece (+ 1: its last one), and how many pieces
    int* err;
    int workers;
    int nrt;  // tiles of query rows per (row, kv-head)
    int R;    // query rows per tile
};

// A pointer to memory on the device (and not, as far as the compiler can tell of one read from memory, to LDS).
template <typename T>
using global = __attribute__((address_space(1))) T;
template <typename T>
__device__ __forceinline__ global<T>* as_global(T* p) {
    return (global<T>*)p;
}

// What a row of the batch attends over.
struct Row {
    int len;    // tokens that its table holds
    int ctx;    // token of node 0 (below 0 where the row is shorter than its nodes)
    int count;  // nodes
};

__device__ __forceinline__ Row row_of(const Params& p, int b) {
    Row w;
    const int s0 = as_global(p.seq_lens)[b], s = s0 > 0 ? s0 : 0, cap = p.max_blocks << p.bs_shift;
    int c = p.counts ? as_global(p.counts)[b] : p.T;
    c = c < 0 ? 0 : c < p.T ? c : p.T;
    w.count = c;
    w.ctx = s - c;
    w.len = s < cap ? s : cap;
    return w;
}

// Tokens that a tile of query rows attends over: all of the row's (tree) or those up to its last node (chain).
__device__ __forceinline__ int visible_end(const Params& p, const Row& w, int rt) {
    const int first = rt * p.R / p.G;
    if (first >= w.count) return 0;
    if (p.mask) return w.len;
    int last = (rt * p.R + p.R - 1) / p.G;
    last = last < w.count ? last : w.count - 1;
    const int64_t end = (int64_t)w.ctx + last + 1;
    return end < 0 ? 0 : end < w.len ? (int)end : w.len;
}
__device__ __forceinline__ int seg_tiles(const Params& p, const Row& w, int rt) {
    return (visible_end(p, w, rt) + kTok - 1) / kTok;
}
// What a segment counts for when the whole is cut into ranges.
__device__ __forceinline__ int seg_units(const Params& p, const Row& w, int rt) {
    const int n = seg_tiles(p, w, rt);
    return n == 0 ? 0 : n + kPieceTiles;
}
// ... and one kv-head of a row.
__device__ __forceinline__ int head_units(const Params& p, const Row& w) {
    int n = 0;
    for (int rt = 0; rt < p.nrt; ++rt) n += seg_units(p, w, rt);
    return n;
}

__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(v, o);
        if (lane >= o) v += t;
    }
    return v;
}

struct Seg {
    int b, kvh, rt, tile;
};

// The rows of a batch as a wave holds them: up to 64 in its lanes, read once; of more, each when it is asked for.
struct Rows {
    Row mine;   // row `lane` (B <= 64)
    int units;  // of it
    int incl;   // of it and those before it
    int total;  // of all (below 2^30, checked on the host)
    __device__ __forceinline__ void read(const Params& p, int lane) {
        mine = Row{0, 0, 0};
        total = 0;
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            if (b0 + lane < p.B) mine = row_of(p, b0 + lane);
            units = b0 + lane < p.B ? head_units(p, mine) * p.Hkv : 0;
            incl = wave_scan(units, lane);
            total += __builtin_amdgcn_readlane(incl, 63);
        }
    }
    __device__ __forceinline__ Row at(const Params& p, int b) const {
        if (p.B > 64) return row_of(p, b);
        return Row{__builtin_amdgcn_readlane(mine.len, b), __builtin_amdgcn_readlane(mine.ctx, b),
                   __builtin_amdgcn_readlane(mine.count, b)};
    }
    // The segment that holds unit x of all (x < total), and x's index in it: a tile, or behind the last one.
    __device__ __forceinline__ Seg locate(const Params& p, int x, int lane) const {
        int n = units, up = incl;
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            if (p.B > 64) {
                n = b0 + lane < p.B ? head_units(p, row_of(p, b0 + lane)) * p.Hkv : 0;
                up = wave_scan(n, lane);
            }
            const int sum = __builtin_amdgcn_readlane(up, 63);
            if (x < sum) {
                const int bl = __builtin_popcountll(__builtin_amdgcn_ballot_w64(up <= x));
                Seg s;
                s.b = b0 + bl;
                const int here = __builtin_amdgcn_readlane(n, bl);
                x -= __builtin_amdgcn_readlane(up, bl) - here;
                const int per = (unsigned)here / (unsigned)p.Hkv;
                s.kvh = (unsigned)x / (unsigned)per;
                x -= s.kvh * per;
                s.rt = 0;
                if (p.nrt > 1) {
                    const Row w = at(p, s.b);
                    for (int m; s.rt + 1 < p.nrt && x >= (m = seg_units(p, w, s.rt)); ++s.rt) x -= m;
                }
                s.tile = x;
                return s;
            }
            x -= sum;
        }
        return Seg{0, 0, 0, 0};  // unreachable for x < total
    }
};

__device__ __forceinline__ int workers_of(const Params& p, int total) { return p.workers < total ? p.workers : total; }
// a / b, in 32 bits where they do (64-bit division is a long sequence, and every workgroup begins with two).
__device__ __forceinline__ int quotient(uint64_t a, int b) {
    return a >> 32 ? (int)(a / (uint32_t)b) : (int)((uint32_t)a / (uint32_t)b);
}
__device__ __forceinline__ int range_lo(int w, int total, int workers) { return quotient((uint64_t)w * total, workers); }
// The worker that holds unit x.
__device__ __forceinline__ int worker_of(int x, int total, int workers) {
    return quotient((uint64_t)(x + 1) * workers - 1, total);
}

// N times 16 bytes per lane from memory to LDS: load i's of lane l, at from[i], to `to` + 1024 i + 16 l (`to` the same in all
// lanes). As a builtin the loads would be waited for ahead of every later read of LDS, whatever that reads; so the caller
// waits (vmcnt) before the barrier that hands the tile over. Nothing is written to a register. An instruction's offset counts
// on both sides, so M0, which holds the place in LDS, is set once, and left as it was. STREAM: past the caches.
#define MX_LOADS_TO_LDS(NT)                                                                                               \
    if constexpr (N == 1)                                                                                                 \
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off" NT "\n\t"       \
                     "s_mov_b32 m0, %0"                                                                                   \
                     : "=&s"(was)                                                                                         \
                     : "s"(at), "v"(from[0])                                                                              \
                     : "memory");                                                                                         \
    else if constexpr (N == 2)                                                                                            \
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off" NT "\n\t"       \
                     "global_load_lds_dwordx4 %3, off offset:%4" NT "\n\ts_mov_b32 m0, %0"                                \
                     : "=&s"(was)                                                                                         \
                     : "s"(at), "v"(from[0]), "v"(from[1] - 1024), "n"(1024)                                              \
                     : "memory");                                                                                         \
    else                                                                                                                  \
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off" NT "\n\t"       \
                     "global_load_lds_dwordx4 %3, off offset:%6" NT                                                       \
                     "\n\tglobal_load_lds_dwordx4 %4, off offset:%7" NT                                                   \
                     "\n\tglobal_load_lds_dwordx4 %5, off offset:%8" NT "\n\ts_mov_b32 m0, %0"                            \
                     : "=&s"(was)                                                                                         \
                     : "s"(at), "v"(from[0]), "v"(from[1] - 1024), "v"(from[2] - 2 * 1024), "v"(from[3] - 3 * 1024),          \
                       "n"(1024), "n"(2 * 1024), "n"(3 * 1024)                                                            \
                     : "memory")
template <int N, bool STREAM>
__device__ __forceinline__ void load_to_lds(const char* const (&from)[N], uint32_t to) {
    static_assert(N == 1 || N == 2 || N == 4, "offsets are below 4096");
    uint32_t was;
    const int at = __builtin_amdgcn_readfirstlane((int)to);
    if constexpr (STREAM) {
        MX_LOADS_TO_LDS(" nt");
    } else {
        MX_LOADS_TO_LDS("");
    }
}
#undef MX_LOADS_TO_LDS

typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef int i32x2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4v lds_s16x4;
__device__ __forceinline__ s16x4v read_tr(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
}

// Elements that are not finite set to 0 in x; whether there were any.
template <bool BF16>
__device__ __forceinline__ bool drop_special(u32x4v& x) {
    constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool lo = (x[i] & E) == E, hi = (x[i] & (E << 16)) == (E << 16);
        x[i] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
        any |= lo || hi;
    }
    return any;
}

#define MX_INLINE __attribute__((always_inline))

// The kernel's arguments read again from where the launch left them. What the loop over tiles does not use would otherwise stay
// in scalar registers across it (or, as there are not enough of them, in lanes of vector registers, at a v_readlane each).
__device__ __forceinline__ Params reload() {
    uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    args = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)args) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(args >> 32)) << 32;
    const auto* from = (const __attribute__((address_space(4))) uint64_t*)args;
    static_assert(sizeof(Params) % 8 == 0, "read in words");
    uint64_t words[sizeof(Params) / 8];
#pragma unroll
    for (size_t i = 0; i < sizeof(Params) / 8; ++i) words[i] = from[i];
    Params p;
    __builtin_memcpy(&p, words, sizeof p);
    return p;
}

typedef short s16x8v __attribute__((ext_vector_type(8)));

// A tile and its segment, the same in all lanes.
struct Tile {
    Seg seg;
    int end, ntiles;  // of the segment: tokens that it attends over, tiles

    __device__ __forceinline__ void enter(const Params& p, const Rows& rows) {
        end = visible_end(p, rows.at(p, seg.b), seg.rt);
        ntiles = (end + kTok - 1) / kTok;
    }
    // To the next segment that holds a tile; there is one.
    __device__ __forceinline__ void next_segment(const Rows& rows) {
        const Params p = reload();
        seg.tile = 0;
        do {
            if (++seg.rt == p.nrt) {
                seg.rt = 0;
                if (++seg.kvh == p.Hkv) {
                    seg.kvh = 0;
                    ++seg.b;
                }
            }
            enter(p, rows);
        } while (ntiles == 0);
    }
    // Every node of the segment sees every token below this (if its block is one of the pool).
    __device__ __forceinline__ int open(const Params& p, const Row& row) const {
        const int64_t n = (int64_t)row.ctx + (p.mask ? 0 : seg.rt * p.R / p.G + 1);
        return n < end ? n > 0 ? (int)n : 0 : end;
    }
};

// Tiles on their way from the pool to LDS, WAVES waves sharing them. The loads go without a register: a lane's 16 bytes land at 16
// times the lane behind the instruction's place, so the permutation of a token's chunks is in the addresses that the lanes
// read from. Block ids are held 64 at a time, one a lane (an instruction's 1 KiB holds tokens of two blocks at most), and read
// ahead of the tile that needs them: ids read a tile at a time, by scalar loads, took 1300 of a tile's 5600 cycles.
template <int D, int WAVES, bool STREAM>
struct Loader {
    static constexpr int CH = D / 8;                // 16-byte chunks per token
    static constexpr int RPL = 64 / CH;             // tokens per load instruction of a wave
    static constexpr int P = kTok / RPL / WAVES;    // load instructions per wave and tile, of K and of V each
    static constexpr int IPL = RPL / 4;             // blocks per instruction, at most
    static_assert(P * RPL * WAVES == kTok, "tile split");
    Tile x;           // the next one to load
    int64_t head;     // elements before its kv-head in a block
    int ids, coming;  // the 64 block ids around it, and those to take their place
    bool change;
    int left;         // units of the range from this tile on

    __device__ __forceinline__ void look_up(const Params& p, int lane) {
        head = (int64_t)x.seg.kvh * p.kv_shead;
        const int i = (x.seg.tile * kTok >> p.bs_shift & ~63) + lane, last = (x.end - 1) >> p.bs_shift;
        coming = as_global(p.bt)[(int64_t)x.seg.b * p.bt_sb + (i < last ? i : last)];  // past the end: the last one again
        change = true;
    }
    __device__ __forceinline__ void advance(const Rows& rows, int bs_shift, int lane) {
        --left;
        if (++x.seg.tile >= x.ntiles) {
            left -= kPieceTiles;
            if (left <= 0) return;
            x.next_segment(rows);
        }
        if (left <= 0) return;
        if ((x.seg.tile * kTok >> bs_shift & 63) == 0) look_up(reload(), lane);
    }
    // The tile to ks_at and vs_at; returns whether a block lies outside the pool (its tokens read block 0).
    __device__ __forceinline__ bool issue(const Params& p, uint32_t ks_at, uint32_t vs_at, int wave, int lane) {
        if (change) {
            ids = coming;
            asm volatile("" : "+v"(ids));  // waited for in this branch
            change = false;
        }
        const int last = x.end - 1, bs = 1 << p.bs_shift;
        const _Float16 *kb = p.k + head, *vb = p.v + head;
        bool bad = false;
        constexpr int N = P < 4 ? P : 4;
#pragma unroll
        for (int i0 = 0; i0 < P; i0 += N) {
            const char *kf[N], *vf[N];
#pragma unroll
            for (int i = i0; i < i0 + N; ++i) {
                int64_t blk[IPL];
#pragma unroll
                for (int j = 0; j < IPL; ++j) {
                    const int tok = x.seg.tile * kTok + (wave * P + i) * RPL + 4 * j;
                    const int id = __builtin_amdgcn_readlane(ids, tok >> p.bs_shift & 63);
                    const bool inside = (unsigned)id < (unsigned)p.num_blocks;
                    bad |= !inside;
                    blk[j] = (inside ? id : 0) * p.kv_sblk;
                }
                const int rr = (wave * P + i) * RPL + lane / CH;
                int tok = x.seg.tile * kTok + rr;
                tok = tok < last ? tok : last;
                const int at = (tok & (bs - 1)) * D + 8 * (lane % CH ^ (rr & (CH - 1)));
                const int64_t off = (IPL == 2 && (lane / CH & 4) ? blk[IPL - 1] : blk[0]) + at;
                kf[i - i0] = reinterpret_cast<const char*>(kb + off);
                vf[i - i0] = reinterpret_cast<const char*>(vb + off);
            }
            const uint32_t at = (uint32_t)(wave * P + i0) * 1024;
            load_to_lds<N, STREAM>(kf, ks_at + at);
            load_to_lds<N, STREAM>(vf, vs_at + at);
        }
        if (bad && p.err) atomicOr(p.err, 4);
        return bad;
    }
};

// The query rows of a wave (RT tiles of 16) and what they have gathered, over NTT 16-token tiles at a time.
template <int D, bool BF16, int RT, int NTT>
struct Queries {
    using E = Elt<BF16>;
    static constexpr int KC = D / 32;  // 32-dim steps of a score
    static constexpr int DT = D / 16;  // 16-dim output tiles
    static constexpr int CH = D / 8;   // 16-byte chunks per token
    half8v q[RT][KC];                  // lane l: dims 32 c + 8 (l / 16) + [0, 8) of row l % 16 of each tile
    // (vectors: of arrays here the compiler keeps some in memory)
    int node __attribute__((ext_vector_type(RT)));  // -1: no such row
    float m __attribute__((ext_vector_type(RT)));
    float4v l[RT], acc[DT][RT];        // (l's four are the same)

    // Rows row0 .. of the segment.
    __device__ __forceinline__ void load(const Params& p, const Seg& seg, int count, int row0, int lane) {
        const int g = lane >> 4, r = lane & 15;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int rr = row0 + t * 16 + r;
            const int n = rr / p.G, h = seg.kvh * p.G + (rr - n * p.G);
            node[t] = n < count ? n : -1;
            const auto* qp = as_global(p.q) + (int64_t)seg.b * p.q_sb + (int64_t)h * p.q_sh + (int64_t)n * p.q_st + 8 * g;
#pragma unroll
            for (int kk = 0; kk < KC; ++kk)
                q[t][kk] = node[t] >= 0 ? __builtin_bit_cast(half8v, *(const global<u32x4v>*)(qp + 32 * kk)) : half8v{};
            m[t] = 0.0f;
            l[t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d][t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // Scores of the tokens from `first` of the tile whose K begins at byte `at` of k. A row's chunks are permuted by an exclusive
    // or, and so are the addresses of one lane's reads; rows 16 apart are permuted alike. (The empty asm keeps the
    // compiler from holding all addresses in registers.)
    __device__ __forceinline__ void scores(const char* k, uint32_t at, int first, int lane, float4v (&s)[NTT][RT]) const {
        const int g = lane >> 4, r = lane & 15;
        uint32_t ka = at + (uint32_t)(first + r) * D * 2 + ((g ^ (r & (CH - 1))) << 4);
        asm volatile("" : "+v"(ka));
#pragma unroll
        for (int kk = 0; kk < KC; ++kk)
#pragma unroll
            for (int i = 0; i < NTT; ++i) {
                const half8v a = __builtin_bit_cast(half8v, *reinterpret_cast<const u32x4v*>(k + (ka ^ (kk << 6)) + 16 * i * D * 2));
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    s[i][t] = E::mma32(a, q[t][kk], kk ? s[i][t] : float4v{0.0f, 0.0f, 0.0f, 0.0f});
            }
        // Reads a step ahead of the products that use them: left to itself the compiler waits for each pair of reads.
        __builtin_amdgcn_sched_group_barrier(kDsRead, NTT, 0);
#pragma unroll
        for (int kk = 0; kk + 1 < KC; ++kk) {
            __builtin_amdgcn_sched_group_barrier(kDsRead, NTT, 0);
            __builtin_amdgcn_sched_group_barrier(kMfma, NTT * RT, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, NTT * RT, 0);
    }
    // -inf where words (of nodes from `node0` on) say that a token is not visible.
    __device__ __forceinline__ void hide(const uint64_t* words, int node0, int first, int lane, float4v (&s)[NTT][RT]) const {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            uint64_t seen = node[t] >= 0 ? words[node[t] - node0] : 0;
            seen >>= first + 4 * (lane >> 4);
#pragma unroll
            for (int i = 0; i < 4 * NTT; ++i)
                if (!(seen >> (16 * (i >> 2) + (i & 3)) & 1)) s[i >> 2][t][i & 3] = -__builtin_huge_valf();
        }
    }
    // Scores to probabilities: m moved where it has to be, what was gathered with it.
    __device__ __forceinline__ void softmax(float scale_log2e, float4v (&s)[NTT][RT], half8v (&pr)[NTT / 2][RT]) {
        // What a score's exponential is taken of, score * scale - m; the maximum of these says whether m has to move. (It
        // begins where the row's first visible scores are, wherever that is.)
        bool move = false;
        float top[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int i = 0; i < 4 * NTT; ++i) s[i >> 2][t][i & 3] = __builtin_fmaf(s[i >> 2][t][i & 3], scale_log2e, -m[t]);
            top[t] = fmaxf(s[0][t][0], s[0][t][1]);
#pragma unroll
            for (int i = 2; i < 4 * NTT; i += 2) top[t] = fmaxf(fmaxf(top[t], s[i >> 2][t][i & 3]), s[i >> 2][t][(i & 3) + 1]);
            move |= top[t] > (l[t][0] == 0.0f ? -__builtin_huge_valf() : kLazyLog2 + kHeadLog2);
        }
        if (__builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const bool fresh = l[t][0] == 0.0f;
                const float up = xor_max_16_32(top[t]) - kHeadLog2;
                const float by = (fresh || up > 0.0f) && up > -__builtin_huge_valf() ? up : 0.0f;
                const float f = fresh ? 1.0f : __builtin_amdgcn_exp2f(-by);
                m[t] += by;
                l[t] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d][t] *= f;
#pragma unroll
                for (int i = 0; i < 4 * NTT; ++i) s[i >> 2][t][i & 3] -= by;
            }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < 4 * NTT; ++i) pr[i >> 3][t][i & 7] = E::round(__builtin_amdgcn_exp2f(s[i >> 2][t][i & 3]));
    }
    // P.V of the same tokens, V beginning at byte `at` of v; l sums the rounded probabilities by a product with ones, which
    // adds up a row's four lanes as well.
    __device__ __forceinline__ void gather(const char* v, uint32_t at, int first, int lane, const half8v (&pr)[NTT / 2][RT]) {
        const int g = lane >> 4, r = lane & 15, vr = first + 4 * g + (r >> 2);
        uint32_t va = at + (uint32_t)vr * D * 2 + ((((r & 3) >> 1) ^ (vr & (CH - 1))) << 4) + 8 * (r & 1);
        asm volatile("" : "+v"(va));
        half8v ones;
#pragma unroll
        for (int i = 0; i < 8; ++i) ones[i] = E::round(1.0f);
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < NTT / 2; ++u) l[t] = E::mma32(ones, pr[u][t], l[t]);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int u = 0; u < NTT / 2; ++u) {
                // V^T: dim 16 d + r of tokens 32 u + 4 g + [0, 4) and that + 16
                const char* src = v + (va ^ (d << 5)) + 32 * u * D * 2;
                const s16x4v x0 = read_tr(src), x1 = read_tr(src + 16 * D * 2);
                const half8v a = __builtin_bit_cast(half8v, (s16x8v)__builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[d][t] = E::mma32(a, pr[u][t], acc[d][t]);
            }
        // Reads two dim tiles ahead.
        __builtin_amdgcn_sched_group_barrier(kDsRead, 2 * NTT, 0);
        __builtin_amdgcn_sched_group_barrier(kMfma, RT * NTT / 2, 0);
#pragma unroll
        for (int d = 0; d + 2 < DT; ++d) {
            __builtin_amdgcn_sched_group_barrier(kMfma, RT * NTT / 2, 0);
            __builtin_amdgcn_sched_group_barrier(kDsRead, NTT, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, RT * NTT, 0);
    }
    // V of drafted tokens that is not finite was staged as 0 where a node does not see every token of the tile (0 * inf would be
    // NaN for it): it counts for the rows that see it, whose probability of it is above 0. Tiles [from, to) of x's segment.
    __device__ __forceinline__ void add_special(const Params& p, const Tile& x, const Row& row, int from, int to, int lane) {
        const int open = x.open(p, row) / kTok;
        int tok = (from > open ? from : open) * kTok;
        tok = tok > row.ctx ? tok : row.ctx;
        for (; tok < to * kTok && tok < x.end; ++tok) {
            const int id = as_global(p.bt)[(int64_t)x.seg.b * p.bt_sb + (tok >> p.bs_shift)], n = tok - row.ctx;
            if ((unsigned)id >= (unsigned)p.num_blocks) continue;
            const auto* vp = as_global(p.v) + (int64_t)x.seg.kvh * p.kv_shead + id * p.kv_sblk +
                             (tok & ((1 << p.bs_shift) - 1)) * D + 4 * (lane >> 4);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const bool see = node[t] >= 0 && (p.mask ? as_global(p.mask)[(int64_t)x.seg.b * p.mask_sb +
                                                                             (int64_t)node[t] * p.mask_st + n] != 0
                                                         : n <= node[t]);
                if (see)
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const half4v v = *(const global<half4v>*)(vp + 16 * d);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float f = E::widen(v[i]);
                            if (!(__builtin_fabsf(f) < __builtin_huge_valf())) acc[d][t][i] += f;
                        }
                    }
            }
        }
    }
    // Rows row0 .. of the segment (the sums ls): as output where the piece is the whole segment, else to rows part0 .. of the
    // partials.
    __device__ __forceinline__ void store(const Params& p, const Seg& seg, bool complete, int row0, int64_t part0, const float (&ls)[RT],
                                          int lane) const {
        const int g = lane >> 4, r = lane & 15;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float inv = ls[t] == 0.0f ? 0.0f : 1.0f / ls[t];
            if (complete) {
                const int rr = row0 + t * 16 + r, n = rr / p.G, h = seg.kvh * p.G + (rr - n * p.G);
                if (n >= p.T) continue;
                auto* dst = as_global(p.out) + (int64_t)seg.b * p.o_sb + (int64_t)n * p.o_st + (int64_t)h * p.o_sh + 4 * g;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    half4v o;
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = ls[t] == 0.0f ? (_Float16)0.0f : E::round(acc[d][t][i] * inv);
                    *(global<half4v>*)(dst + 16 * d) = o;
                }
            } else {
                auto* dst = as_global(p.part) + (part0 + t * 16 + r) * (D + 4);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    *(global<float4v>*)(dst + 16 * d + 4 * g) = ls[t] == 0.0f ? float4v{} : acc[d][t] * inv;
                if (g == 0) *(global<f32x2v>*)(dst + D) = f32x2v{m[t], ls[t]};
            }
        }
    }
};

// A tile that some node does not see whole, by tid of NT threads in whole waves. V (at vt): 0 where there is no token, and
// where a drafted token's is not finite; returns whether there was one. And who sees what, a bit a token: a wave takes a
// node at a time, a lane a token, so the bytes of a mask row come in one load (as loads of each lane's own bytes two such
// tiles at a row's end took 20 us).
template <int D, bool BF16, int NT>
__device__ __forceinline__ bool clean_tile(const Tile& x, const Rows& rows, bool bad, uint64_t* words, _Float16* vt, int tid) {
    constexpr int CH = D / 8, WAVES = NT / 64;
    const Params p = reload();
    const Row row = rows.at(p, x.seg.b);
    const auto* bt = as_global(p.bt) + (int64_t)x.seg.b * p.bt_sb;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), t0 = x.seg.tile * kTok;
    const int first_node = x.seg.rt * p.R / p.G, last_node = (x.seg.rt * p.R + p.R - 1) / p.G;
    const int nodes = (last_node < row.count ? last_node + 1 : row.count) - first_node;
    const int tok = t0 + lane, n = tok - row.ctx;
    bool there = tok < x.end;
    if (bad && there) there = (unsigned)bt[tok >> p.bs_shift] < (unsigned)p.num_blocks;
    const bool drafted = there && n >= 0;
    constexpr int U = 8;
    for (int i0 = wave; i0 < nodes; i0 += U * WAVES) {
        uint8_t see[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * WAVES;
            see[u] = 1;
            if (p.mask && drafted && i < nodes)
                see[u] = as_global(p.mask)[(int64_t)x.seg.b * p.mask_sb + (int64_t)(first_node + i) * p.mask_st + n];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * WAVES;
            const uint64_t word = __builtin_amdgcn_ballot_w64(there && see[u] != 0 && (p.mask || n <= first_node + i));
            if (lane == 0 && i < nodes) words[i] = word;
        }
    }
    bool special = false;
    const int drop = t0 + kTok > x.open(p, row) ? row.ctx : x.end;  // from this token on
    for (int i = tid; i < kTok * CH; i += NT) {
        const int tok = t0 + i / CH;
        u32x4v* at = reinterpret_cast<u32x4v*>(vt) + i;
        u32x4v v = *at;
        if (tok >= x.end || (bad && (unsigned)bt[tok >> p.bs_shift] >= (unsigned)p.num_blocks)) v = u32x4v{0, 0, 0, 0};
        else if (tok < drop || !drop_special<BF16>(v)) continue;
        else special = true;
        *at = v;
    }
    return special;
}

__device__ __forceinline__ void wait_for_loads() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
}

// The units of a workgroup.
struct Range {
    int w, lo, hi, total, workers;
    // Consecutive ranges on one XCD (workgroups go round the 8 XCDs): the tiles of query rows of a kv-head meet in its L2.
    __device__ __forceinline__ Range(const Params& p, int total) : total(total), workers(workers_of(p, total)) {
        const int per = (workers + kXcds - 1) / kXcds;
        w = (int)blockIdx.x % kXcds * per + (int)blockIdx.x / kXcds;
        lo = hi = 0;
        if ((int)blockIdx.x / kXcds >= per || w >= workers) return;
        lo = range_lo(w, total, workers), hi = range_lo(w + 1, total, workers);
    }
};

// Tiles [t0, t1) of x's segment, which begin `first` units into the range, as wave rw over query rows has them (with the sums ls);
// and, with the first of them, how many pieces the segment has, for the launch that joins them.
template <int D, bool BF16, int RT, int NTT>
__device__ __forceinline__ void store_piece(const Params& p, const Queries<D, BF16, RT, NTT>& rs, const Tile& x, int t0, int t1,
                                            const Range& range, int first, int rw, int tid, const float (&ls)[RT]) {
    const int slot = 2 * range.w + (first == 0 ? 0 : 1);
    rs.store(p, x.seg, t0 == 0 && t1 == x.ntiles, x.seg.rt * p.R + rw * RT * 16, (int64_t)slot * p.R + rw * RT * 16, ls, tid & 63);
    if (t0 == 0 && tid == 0) {
        const int pieces = worker_of(range.lo + first + x.ntiles - 1, range.total, range.workers) - range.w + 1;
        *(global<i32x2v>*)(as_global(p.pieces) + ((int64_t)x.seg.b * p.Hkv + x.seg.kvh) * p.nrt + x.seg.rt) = i32x2v{slot, pieces};
    }
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// D: head dim. RT: 16-row query tiles per wave. RW x TW: waves over query rows and over a tile's tokens. STREAM: K and V are read
// past the caches.
template <int D, bool BF16, int RT, int RW, int TW, bool STREAM>
__global__ __launch_bounds__(64 * RW * TW, RW * TW == 2 ? 1 : 2) void tree_attn_kernel(Params p) {
    constexpr int NT = 64 * RW * TW;
    constexpr int NTT = kTok / 16 / TW;  // 16-token tiles per wave
    constexpr int R = 16 * RT * RW, TB = kTok * D * 2;
    static_assert(NTT % 2 == 0, "tile split");
    __shared__ __attribute__((aligned(16))) _Float16 ks[2][kTok * D];
    __shared__ __attribute__((aligned(16))) _Float16 vs[2][kTok * D];
    __shared__ uint64_t words[R];  // of a masked tile: bit j of word n: token j is visible to the n-th node of the query rows
    __shared__ float2 xml[TW > 1 ? RW * RT * 64 : 1];
    __shared__ int bad_step[2];  // the last step whose tile has a token of a block outside the pool
    __shared__ int nf_step;      // ... a drafted token whose V is not finite

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RW, tw = wave / RW;
    const int lane = tid & 63;

    // Waves 4 .. 7 share the four SIMDs with waves 0 .. 3: they issue their loads behind the scores, when the others have the
    // matrix cores, and not ahead of them (8 rows of 64 nodes: 73 against 75 us).
    const bool late = RW * TW == 8 && wave >= 4;
    Rows rows;
    rows.read(p, lane);
    const Range range(p, rows.total);
    if (range.lo >= range.hi) return;
    if (tid < 2) bad_step[tid] = 0;
    if (tid == 0) nf_step = 0;
    int step = 1;  // number of the tile at work, buffer step & 1
    const uint32_t ks_at = lds_address(&ks[0][0]), vs_at = lds_address(&vs[0][0]);

    Loader<D, RW * TW, STREAM> ahead;
    ahead.x.seg = rows.locate(p, range.lo, lane);
    ahead.x.enter(p, rows);
    ahead.left = range.hi - range.lo;
    if (ahead.x.seg.tile >= ahead.x.ntiles) {
        ahead.left -= ahead.x.ntiles + kPieceTiles - ahead.x.seg.tile;
        if (ahead.left <= 0) return;
        ahead.x.next_segment(rows);
    }
    ahead.look_up(p, lane);
    Tile cur = ahead.x;
    int left = ahead.left;  // units from the tile at work on
    __syncthreads();  // bad_step
    auto issue = [&](int st) MX_INLINE {  // tile number st
        if (ahead.issue(p, ks_at + (st & 1) * TB, vs_at + (st & 1) * TB, wave, lane)) bad_step[st & 1] = st;
        ahead.advance(rows, p.bs_shift, lane);
    };
    // The compiler does not track those loads.
    auto arrived = [&]() MX_INLINE {
        wait_for_loads();
        __syncthreads();
    };
    issue(step);
    arrived();

    // A piece after the other: the tiles of one segment in this range. The first tile of the next one is on its way already.
    for (;;) {
        const int t0 = cur.seg.tile, t1 = cur.ntiles - t0 < left ? cur.ntiles : t0 + left, step0 = step;
        const int first = range.hi - range.lo - left;
        Queries<D, BF16, RT, NTT> rs;
        int open;
        {
            const Params p = reload();
            const Row row = rows.at(p, cur.seg.b);
            open = cur.open(p, row);
            rs.load(p, cur.seg, row.count, cur.seg.rt * R + rw * RT * 16, lane);
            // Waited for here: in the loop the wait would be there every time, and for the loads of the next tile.
            wait_for_loads();
        }
        for (;;) {
            if (ahead.left > 0 && !late) issue(step + 1);
            const int buf = step & 1;
            const bool bad = bad_step[buf] == step, masked = cur.seg.tile * kTok + kTok > open || bad;
            if (masked) {
                if (clean_tile<D, BF16, NT>(cur, rows, bad, words, &vs[buf][0], tid)) nf_step = step;
                __syncthreads();
            }
            float4v s[NTT][RT];
            half8v pr[NTT / 2][RT];
            rs.scores(reinterpret_cast<const char*>(&ks[0][0]), buf * TB, tw * (kTok / TW), lane, s);
            if (ahead.left > 0 && late) issue(step + 1);
            if (masked) rs.hide(words, cur.seg.rt * R / reload().G, tw * (kTok / TW), lane, s);
            rs.softmax(p.scale_log2e, s, pr);
            rs.gather(reinterpret_cast<const char*>(&vs[0][0]), buf * TB, tw * (kTok / TW), lane, pr);
            if (cur.seg.tile + 1 == t1) break;
            arrived();
            ++cur.seg.tile, ++step;
        }

        float ls[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) ls[t] = rs.node[t] < 0 ? 0.0f : rs.l[t][0];
        // The waves over tokens meet in the buffers of the last tile (the others may be loading).
        if constexpr (TW > 1) {
            static_assert(TW == 2 && RW <= 2 && sizeof(ks[0]) >= sizeof(float4v) * 64 * RT * (D / 16), "exchange");
            float4v* xch = reinterpret_cast<float4v*>(rw == 0 ? &ks[step & 1][0] : &vs[step & 1][0]) + lane;
            __syncthreads();
            if (tw == 1) {
#pragma unroll
                for (int t = 0; t < RT; ++t) {
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) xch[(d * RT + t) * 64] = rs.acc[d][t];
                    xml[(rw * RT + t) * 64 + lane] = float2{rs.m[t], ls[t]};
                }
            }
            __syncthreads();
            if (tw == 0) {
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const float2 other = xml[(rw * RT + t) * 64 + lane];
                    // A wave that has seen nothing has no reference.
                    const float ma = ls[t] == 0.0f ? kLowest : rs.m[t], mb = other.y == 0.0f ? kLowest : other.x;
                    rs.m[t] = fmaxf(ma, mb);
                    const float fa = __builtin_amdgcn_exp2f(ma - rs.m[t]), fb = __builtin_amdgcn_exp2f(mb - rs.m[t]);
                    ls[t] = ls[t] * fa + other.y * fb;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) rs.acc[d][t] = rs.acc[d][t] * fa + xch[(d * RT + t) * 64] * fb;
                }
            }
        }
        if (tw == 0) {
            const Params p = reload();
            if (nf_step >= step0) rs.add_special(p, cur, rows.at(p, cur.seg.b), t0, t1, lane);
            store_piece<D, BF16, RT, NTT>(p, rs, cur, t0, t1, range, first, rw, tid, ls);
        }
        left -= t1 - t0 + kPieceTiles;
        if (left <= 0) break;
        cur.next_segment(rows);
        arrived();
        ++step;
    }
}

// Joins the pieces of the segments that more than one workgroup cut, and clears rows of segments without tokens. Bound by the
// pieces' bytes, 4 (D + 4) a query row and piece: 383 pieces of 256 rows of a chunk (52 MB) 12 us, 4.3 TB/s; a few pieces 4 us, of
// which a launch and two dependent loads are most.
// A workgroup of 256 threads has D / 4 lanes per query row (4 dims each) and shares a row's pieces among SP groups of
// lanes: RPG = 256 / (D / 4) / SP query rows at a time.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void tree_merge_kernel(Params p, int sp) {
    using E = Elt<BF16>;
    constexpr int LN = D / 4;
    constexpr int GR = 256 / LN;  // lane groups
    __shared__ float4v sacc[GR][LN];
    __shared__ float2 sml[GR];
    const int tid = threadIdx.x;
    const int grp = tid / LN, x = tid % LN;
    const int rows_per = GR / sp;
    const int blocks = (p.R + rows_per - 1) / rows_per;
    const int segid = blockIdx.x / blocks, rr = (blockIdx.x - segid * blocks) * rows_per + grp / sp, part = grp % sp;
    const int rt = segid % p.nrt, kvh = segid / p.nrt % p.Hkv, b = segid / p.nrt / p.Hkv;
    const int qrow = rt * p.R + rr, n = qrow / p.G, h = kvh * p.G + qrow - n * p.G;
    const int2 info = p.pieces[segid];  // nothing sensible where the segment has no tile
    const bool any = seg_tiles(p, row_of(p, b), rt) > 0;
    if (any && info.y == 1) return;  // written whole
    const int first = info.x >> 1, head = info.x & 1, pieces = any ? info.y : 0;
    float m = kLowest, l = 0.0f;
    float4v acc{0.0f, 0.0f, 0.0f, 0.0f};
    const bool live = rr < p.R && n < p.T;
    if (live) {
        constexpr int U = 4;  // pieces in flight
        for (int k0 = part; k0 < pieces; k0 += U * sp) {
            float4v o[U];
            float2 ml[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * sp < pieces ? k0 + u * sp : k0;
                const int slot = 2 * (first + k) + (k == 0 ? head : 0);
                const float* src = p.part + ((int64_t)slot * p.R + rr) * (D + 4);
                o[u] = *reinterpret_cast<const float4v*>(src + 4 * x);
                ml[u] = *reinterpret_cast<const float2*>(src + D);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // (a piece of which the row sees nothing counts for nothing)
                if (k0 + u * sp >= pieces || ml[u].y == 0.0f) continue;
                const float mx = fmaxf(m, ml[u].x);
                const float fa = __builtin_amdgcn_exp2f(m - mx), fb = __builtin_amdgcn_exp2f(ml[u].x - mx) * ml[u].y;
                acc = acc * fa + o[u] * fb;
                l = l * fa + fb;
                m = mx;
            }
        }
    }
    if (sp > 1) {
        sacc[grp][x] = acc;
        if (x == 0) sml[grp] = float2{m, l};
        __syncthreads();
        if (part == 0) {
            for (int i = 1; i < sp; ++i) {
                const float2 ml = sml[grp + i];
                if (ml.y == 0.0f) continue;
                const float mx = fmaxf(m, ml.x);
                const float fa = __builtin_amdgcn_exp2f(m - mx), fb = __builtin_amdgcn_exp2f(ml.x - mx);
                acc = acc * fa + sacc[grp + i][x] * fb;
                l = l * fa + ml.y * fb;
                m = mx;
            }
        }
    }
    if (!live || part) return;
    half4v o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = l == 0.0f ? (_Float16)0.0f : E::round(acc[i] / l);
    *reinterpret_cast<half4v*>(p.out + (int64_t)b * p.o_sb + (int64_t)n * p.o_st + (int64_t)h * p.o_sh + 4 * x) = o;
}

struct Plan {
    int rt, rw, tw;  // template arguments
    int R, nrt, workers;
};

// Query rows per workgroup: as few wasted rows as the tiles allow up to 256, so that K and V are read once. The next larger shape
// takes, on 32 rows of U[128, 4096] tokens, 54 us for 16 query rows (this one 50), 59 for 32 (55) and 66 for 64 (58), and 159
// for 100 query rows over 131,071 tokens (102); workgroups of 128 query rows for 256 of them, which read K and V twice, 79 on 8
// rows of U[4096, 8192] tokens (72), 88 on a chunk (76).
// Workgroups: what the CUs hold at once, two by the LDS or one of eight waves. Half as many take 71 and 125 us on the 32 rows with 16 nodes
// and on the long row (58, 102), twice as many 70 and 117, and 81 on the 8 rows with 64 nodes (69): more pieces to begin and to join.
static Plan plan_of(int64_t B, int64_t T, int64_t Hkv, int64_t G, int64_t max_tokens) {
    Plan p{};
    const int64_t rows = G * T;
    if (rows <= 16) p = {1, 1, 2};
    else if (rows <= 32) p = {2, 1, 2};
    else if (rows <= 64) p = {2, 2, 2};
    else if (rows <= 128) p = {2, 4, 1};
    else p = {2, 8, 1};
    p.R = 16 * p.rt * p.rw;
    p.nrt = (int)ceil_div(rows, p.R);
    const int64_t most = B * Hkv * p.nrt * (ceil_div(max_tokens, kTok) + kPieceTiles);
    const int64_t full = p.rw * p.tw == 8 ? kCus : 2 * kCus;
    p.workers = (int)ceil_div(most < full ? most : full, kXcds) * kXcds;
    return p;
}

static size_t part_bytes(const Plan& p, int D) { return (size_t)2 * p.workers * p.R * (D + 4) * sizeof(float); }

template <int D, bool BF16, bool STREAM>
static void launch(const Plan& pl, const Params& p, hipStream_t st) {
    const dim3 grid((unsigned)p.workers), block(64 * pl.rw * pl.tw);
    if (pl.rt == 1) hipLaunchKernelGGL((tree_attn_kernel<D, BF16, 1, 1, 2, STREAM>), grid, block, 0, st, p);
    else if (pl.rw == 1) hipLaunchKernelGGL((tree_attn_kernel<D, BF16, 2, 1, 2, STREAM>), grid, block, 0, st, p);
    else if (pl.rw == 2) hipLaunchKernelGGL((tree_attn_kernel<D, BF16, 2, 2, 2, STREAM>), grid, block, 0, st, p);
    else if (pl.rw == 4) hipLaunchKernelGGL((tree_attn_kernel<D, BF16, 2, 4, 1, STREAM>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((tree_attn_kernel<D, BF16, 2, 8, 1, STREAM>), grid, block, 0, st, p);
}

template <int D, bool BF16>
static void launch(const Plan& pl, const Params& p, bool stream, hipStream_t st) {
    if (stream) launch<D, BF16, true>(pl, p, st);
    else launch<D, BF16, false>(pl, p, st);
    const int64_t segs = (int64_t)p.B * p.Hkv * p.nrt;
    const int groups = 256 / (D / 4);
    // A row's pieces are shared among groups of lanes where there are more than four to a segment: 64 pieces take 9 us so, 19 one
    // after the other. With few the blocks that hold more rows each end as early (7 us either way at two pieces).
    int sp = 1;
    while (sp < groups && p.workers > 4 * sp * segs) sp *= 2;
    const int64_t blocks = segs * ceil_div(p.R, groups / sp);
    hipLaunchKernelGGL((tree_merge_kernel<D, BF16>), dim3((unsigned)blocks), dim3(256), 0, st, p, sp);
}

}  // namespace tree
}  // namespace mx

using namespace mx;

extern "C" size_t mx_tree_attn_workspace_bytes(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t D,
                                               int32_t max_blocks, int32_t block_size) {
    if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_blocks <= 0 || block_size <= 0 || Hq % Hkv != 0) return 0;
    const tree::Plan pl = tree::plan_of(B, T, Hkv, Hq / Hkv, (int64_t)max_blocks * block_size);
    return tree::part_bytes(pl, D) + (size_t)B * Hkv * pl.nrt * sizeof(int2);
}

extern "C" int mx_tree_attn(const uint16_t* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const uint16_t* k,
                            const uint16_t* v, int64_t kv_sblk, int64_t kv_shead, const int32_t* block_tables,
                            int64_t bt_sb, int32_t max_blocks, const int32_t* seq_lens, const uint8_t* mask,
                            int64_t mask_sb, int64_t mask_st, const int32_t* counts, int32_t B, int32_t T, int32_t Hq,
                            int32_t Hkv, int32_t D, int32_t block_size, int32_t num_blocks, float scale, uint16_t* out,
                            int64_t o_sb, int64_t o_st, int64_t o_sh, void* workspace, size_t workspace_bytes,
                            int32_t* err, uint32_t flags, void* stream) {
    clear_error();
    const char* what = "mx_tree_attn";
    if (B < 0 || T < 0) return fail(MX_ERR_INVALID, "%s: B and T must be >= 0", what);
    if (B == 0 || T == 0) return MX_OK;
    if (!q || !k || !v || !block_tables || !seq_lens || !out) return fail(MX_ERR_NULL, "%s: null pointer", what);
    if (Hkv < 1 || Hq < 1 || Hq % Hkv != 0)
        return fail(MX_ERR_INVALID, "%s: Hq (%d) must be a positive multiple of Hkv (%d)", what, Hq, Hkv);
    if (D != 64 && D != 128) return fail(MX_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, D);
    if (block_size != 4 && block_size != 8 && block_size != 16 && block_size != 32)
        return fail(MX_ERR_UNSUPPORTED, "%s: block_size %d (4, 8, 16 or 32)", what, block_size);
    if (max_blocks < 1 || num_blocks < 1) return fail(MX_ERR_INVALID, "%s: max_blocks and num_blocks must be >= 1", what);
    if (flags & ~(uint32_t)(MX_PA_BF16 | MX_PA_SHARED_BLOCKS))
        return fail(MX_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
    if (!(scale >= 1.17549435e-38f) || scale * 1.4426950408889634f > 3.4e38f)
        return fail(MX_ERR_UNSUPPORTED, "%s: scale must be positive and a normal fp32 number, also times log2(e)", what);
    const int64_t strides[] = {q_sb, q_sh, q_st, o_sb, o_st, o_sh, kv_sblk, kv_shead};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return fail(MX_ERR_ALIGNMENT, "%s: strides must be non-negative multiples of 8 elements", what);
    if (mask && (mask_sb < 0 || mask_st < 0)) return fail(MX_ERR_INVALID, "%s: mask strides must be >= 0", what);
    if (bt_sb < 0) return fail(MX_ERR_INVALID, "%s: block table stride must be >= 0", what);
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
        return fail(MX_ERR_ALIGNMENT, "%s: 16-byte alignment", what);
    const int64_t max_tokens = (int64_t)max_blocks * block_size, G = Hq / Hkv;
    // Tokens, query rows, segments, tiles and the merge's threads are 32-bit numbers.
    if (max_tokens > (1 << 30) || G * T > (1 << 24) || (int64_t)B * Hkv > (1 << 24))
        return fail(MX_ERR_UNSUPPORTED, "%s: more tokens or rows than 32-bit numbers hold", what);
    const tree::Plan pl = tree::plan_of(B, T, Hkv, G, max_tokens);
    if ((double)B * Hkv * pl.nrt * (ceil_div(max_tokens, tree::kTok) + tree::kPieceTiles) > (double)(1 << 30) ||
        (double)B * Hkv * pl.nrt * pl.R * (D / 4) > 4.0e9)
        return fail(MX_ERR_UNSUPPORTED, "%s: more tiles than 32-bit numbers hold", what);
    const size_t need = mx_tree_attn_workspace_bytes(B, T, Hq, Hkv, D, max_blocks, block_size);
    if (!workspace || workspace_bytes < need)
        return fail(MX_ERR_WORKSPACE, "%s: workspace needs %zu bytes, got %zu", what, need, workspace ? workspace_bytes : 0);
    if (!aligned(workspace, 16)) return fail(MX_ERR_ALIGNMENT, "%s: workspace alignment", what);
    tree::Params p{};
    p.q = reinterpret_cast<const _Float16*>(q), p.q_sb = q_sb, p.q_sh = q_sh, p.q_st = q_st;
    p.k = reinterpret_cast<const _Float16*>(k), p.v = reinterpret_cast<const _Float16*>(v);
    p.kv_sblk = kv_sblk, p.kv_shead = kv_shead;
    p.bt = block_tables, p.bt_sb = bt_sb, p.max_blocks = max_blocks;
    p.bs_shift = block_size == 4 ? 2 : block_size == 8 ? 3 : block_size == 16 ? 4 : 5;
    p.seq_lens = seq_lens;
    p.mask = mask, p.mask_sb = mask_sb, p.mask_st = mask_st;
    p.counts = counts;
    p.B = B, p.T = T, p.Hkv = Hkv, p.G = (int)G;
    p.num_blocks = num_blocks;
    p.scale_log2e = scale * 1.4426950408889634f;
    p.out = reinterpret_cast<_Float16*>(out), p.o_sb = o_sb, p.o_st = o_st, p.o_sh = o_sh;
    p.part = static_cast<float*>(workspace);
    p.pieces = reinterpret_cast<int2*>(static_cast<char*>(workspace) + tree::part_bytes(pl, D));
    p.err = err;
    p.workers = pl.workers, p.nrt = pl.nrt, p.R = pl.R;
    // Read once, K and V only push out of the caches what is read again, and each other: 32 rows of U[128, 4096] tokens 73 us a call
    // through the caches, 64 past them, one row of 131,071 tokens 119 and 110. Blocks that rows share are read again, and so are
    // those of several tiles of query rows.
    const bool past = pl.nrt == 1 && !(flags & MX_PA_SHARED_BLOCKS);
    hipStream_t st = as_stream(stream);
    const bool bf16 = flags & MX_PA_BF16;
    if (D == 64) {
        if (bf16) tree::launch<64, true>(pl, p, past, st);
        else tree::launch<64, false>(pl, p, past, st);
    } else {
        if (bf16) tree::launch<128, true>(pl, p, past, st);
        else tree::launch<128, false>(pl, p, past, st);
    }
    return check_launch(what);
}
