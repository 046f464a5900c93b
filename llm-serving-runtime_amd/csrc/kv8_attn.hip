// Decode attention over the 8-bit KV cache (kv8.h) on gfx950: out = softmax(scale q K^T) V per query
// head, K and V the values that the pages stand for. The 8-bit form of paged_attn.hip, which replaces
// paged_attention_decode_batched (runtime/phase2/paged_attention_triton.py:745-775).
//
// Work. A segment is one row and one group of at most 16 query heads of a kv-head (a larger GQA group is
// cut into equal ones; each reads the head's pages again). Its tokens are chunks of 16. Two forms, chosen
// from the table's width and the number of segments (by_segment):
//   * a workgroup per segment, whose waves take the steps in turn and join in LDS: one launch;
//   * the chunks of all segments, row after row, as one sequence cut into equal ranges, one per wave, so
//     that every wave streams the same bytes whatever the mix of lengths and a single row fills the chip; a
//     segment that several waves share is joined by a second, small launch from their (m, l, acc).
// All of them fp32.
//
// A wave takes 4 chunks a step, one per lane group g = lane / 16, so that what a lane scores is what it
// weighs, and no score crosses lanes:
//   * scores, 4 x D / 32 products v_mfma_f32_16x16x32: the A operand's row r of product j is token
//     4 j + r % 4 of chunk r / 4, so lane group g receives tokens 4 j + i of chunk g, for head lane % 16
//     (the B operand holds the query heads). K enters as its integers q, and the page's scale multiplies
//     the fp32 score. (As q + 1152 it would take no add, but fp32 would hold 1152 times the query's sum
//     beside the score, whole units of it lost for queries with a mean. Batch 32 with that bias and
//     without: fp16 the same, bf16 35.1 and 36.6 us by segments, 34.3 and 33.6 by ranges.) The head dim is
//     contracted in the order of the lane's 16-byte loads, the query's operand in the same order;
//   * online softmax in fp32 on the exp2 scale; the reference maximum moves only when a score exceeds it
//     by more than 2^8, so most steps neither rescale nor exchange maxima between lane groups;
//   * P.V, 2 x D / 16 products over 32 tokens: lane group g supplies tokens 8 u .. 8 u + 7 of chunk g,
//     which is what its scores gave (weights) and half of a 16-byte load of a dim's token row (V, times
//     the page's scale: exact in 16 bits, a permute and a fused multiply-add per pair).
// Weights are rounded to the 16-bit type before the product, as the 16-bit path's are; the denominator
// sums the rounded ones, by a product with ones. The smallest fp16
// weights are off by up to 2^-25 of a wave's largest, n tokens' by n 2^-25 together: half a step of the output
// where a wave has 2^14 tokens, a layer of 8 GB (two rows of 131,071 tokens and 8 heads: 2^10 tokens).
//
// Bound: HBM. One layer of batch 32, U[128, 4096] tokens, Llama-3-8B heads (139 MB): 33 us by segments, 31.5
// by ranges (tables of 8192 tokens), 27 at the rate of a large copy; two rows of 65,521 to 131,071 tokens
// (403 MB) 76 us in a graph: the ranges read at 6.1 TB/s, then 8 us of merge. By ranges the loads alone took
// 27 of the batch's first launch's 29 us. A CU streams at most about 55 GB/s of such pages, with 64 KiB or
// 128 KiB of loads in flight: two steps ahead instead of one measured 5 to 20 % slower. In bf16, where K and
// V cost a conversion per byte, the batch takes 36.6 us by segments and 33.6 by ranges.
#include <algorithm>

#include "common.h"
#include "elt.h"
#include "kv8.h"

namespace mx {
namespace kv8 {

// Waves per workgroup of the form by ranges. They share nothing; alone, few waves spread over more CUs: in
// wide tables (in a graph) one row of 100 tokens takes 10.0 us with one wave, 10.2 with two and 10.7 with
// four, 7 bf16 rows 10.1, 10.3 and 10.6; batch 32 and two rows of 100,000 tokens the same with any.
constexpr int kAttnWaves = 1;
constexpr int kChunk = 16;         // tokens per chunk
constexpr int kStep = 4;           // chunks per step of a wave
constexpr int kHeads = 16;         // query heads of a segment, at most
// Waves of a launch by ranges: 256 CUs x 8, two per SIMD. Per call with 1536, 2048 and 4096 (two rounds):
// batch 32 of U[128, 4096] tokens in tables of 8192 31.4, 31.5 and 36.1 us, one row of 32,768 27.6, 27.9 and
// 38.7, two of 65,521 to 131,071 73.5, 75.6 and 86.2. Three per SIMD spill: half as slow again.
constexpr int kWorkers = 2048;
constexpr int kSegmentWaves = 8;   // waves of a workgroup that has a segment of its own, at most
constexpr int kMaxTokens = 1 << 30;  // of a table row, so that token and chunk numbers are 32-bit
constexpr float kLazyLog2 = 8.0f;

struct AttnParams {
    const uint16_t* q;
    int64_t q_sb, q_sh;
    Pages pages;
    const int32_t* bt;
    int64_t bt_sb;
    int max_blocks;
    const int32_t* seq_lens;
    int B, G;      // rows; query heads per kv-head
    int NG, GS;    // segments per kv-head, query heads of one (the last may have fewer)
    int Hv;        // segments per row: Hkv * NG
    int workers;   // waves of the launch by ranges
    float scale_log2e;
    uint16_t* out;
    int64_t o_sb, o_sh;
    int32_t* err;
    float* part_ml;   // [2 workers][GS][2]: a piece's maximum and denominator
    float* part_acc;  // [2 workers][GS][D]: its unnormalised output
};

// A row's tokens within its table, and their chunks.
template <int BS>
__device__ __forceinline__ int row_tokens(const AttnParams& p, int b) {
    const int most = p.max_blocks * BS, s = p.seq_lens[b];  // at most kMaxTokens (checked on the host)
    return s < 0 ? 0 : (s < most ? s : most);
}
__device__ __forceinline__ int chunks_of(int tokens) { return (tokens + kChunk - 1) / kChunk; }

// Inclusive prefix sum over the lanes: within rows of 16, then the rows' totals.
__device__ __forceinline__ int incl_scan(int v, int lane) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8; 0 comes in
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31);
    const int r2 = __builtin_amdgcn_readlane(v, 47);
    return v + (lane >= 16 ? r0 : 0) + (lane >= 32 ? r1 : 0) + (lane >= 48 ? r2 : 0);
}

// Sums and maxima over the wave (every lane gets them): row rotations, then row exchanges.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<0x128>(v));  // row_ror:8, 4, 2, 1
    v = fmaxf(v, dpp<0x124>(v));
    v = fmaxf(v, dpp<0x122>(v));
    v = fmaxf(v, dpp<0x121>(v));
    return xor_max_16_32(v);
}
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<0x128>(v);
    v += dpp<0x124>(v);
    v += dpp<0x122>(v);
    v += dpp<0x121>(v);
    return xor_sum_16_32(v);
}
__device__ __forceinline__ int wave_sum(int v) {
    v += __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, false);
    v += __builtin_amdgcn_mov_dpp(v, 0x124, 0xf, 0xf, false);
    v += __builtin_amdgcn_mov_dpp(v, 0x122, 0xf, 0xf, false);
    v += __builtin_amdgcn_mov_dpp(v, 0x121, 0xf, 0xf, false);
    return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
           __builtin_amdgcn_readlane(v, 48);
}

// Chunks of rows [0, b) and of all rows.
template <int BS>
__device__ __forceinline__ void sum_rows(const AttnParams& p, int b, int lane, int& before, int& total) {
    int s0 = 0, s1 = 0;
    for (int i = lane; i < p.B; i += 64) {
        const int n = chunks_of(row_tokens<BS>(p, i));
        s1 += n;
        if (i < b) s0 += n;
    }
    before = wave_sum(s0);
    total = wave_sum(s1);
}

// The cut of T chunks into W ranges: the first `rem` have base + 1 chunks, the others base.
struct Cut {
    int W, base, rem;
    __device__ __forceinline__ Cut(int T, int workers) {
        const int steps = (T + kStep - 1) / kStep;  // no range shorter than a step
        W = steps < workers ? steps : workers;
        base = W > 0 ? T / W : 0;
        rem = T - base * W;
    }
    __device__ __forceinline__ int lo(int w) const { return w * base + (w < rem ? w : rem); }
    __device__ __forceinline__ int worker_of(int x) const {
        const int edge = rem * (base + 1);
        return x < edge ? x / (base + 1) : rem + (x - edge) / base;
    }
};

// The state of a piece: its heads' running maximum and denominator (in every lane of the head), the
// unnormalised output (acc[e][i]: dim 16 e + 4 g + i of head lane % 16).
template <int D>
struct Piece {
    float m, l;
    float4v acc[D / 16];
};

// Where every page stands in one row, K and V are read once and their loads carry the streaming policy:
// batch 32 34.9 -> 32.7 us per call by segments, 33.1 -> 31.5 by ranges, two rows of 100,000 tokens 85.6 ->
// 75.6 (three layers in turn). Pages that the caches hold still from the last call read faster without it:
// one row of 32,768 tokens 25.9 us against 27.9. Rows that share pages (MX_PA_SHARED_BLOCKS) read them with
// the default one.
typedef uint32_t u32x4n __attribute__((ext_vector_type(4)));
template <bool STREAM>
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
    if constexpr (STREAM)
        return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4n*>(p)));
    else
        return *reinterpret_cast<const uint4*>(p);
}

// One step's loads. NP pages stand in a chunk: 1, or 16 / BS.
template <int D, int BS>
struct Regs {
    static constexpr int NP = BS >= kChunk ? 1 : kChunk / BS;
    uint4 k[4][D / 64];
    uint32_t v[D / 16][4];
    uint32_t codes[NP];  // K code | V code << 8
};

template <int D, int BS, bool BF16, bool STREAM>
__device__ __forceinline__ void run_piece(const AttnParams& p, int b, int kvh, int h0, int nh, int c0, int c1,
                                          int stride, int tokens, int lane, Piece<D>& st) {
    constexpr int NP = Regs<D, BS>::NP, KA = D / 64;
    constexpr int PT = BS < kChunk ? BS : kChunk;  // tokens of a chunk in one page
    const int g = lane >> 4, r = lane & 15;
    const float kNegInf = -__builtin_huge_valf();
    const int32_t* bt = p.bt + (int64_t)b * p.bt_sb;
    const int nblk = (tokens + BS - 1) / BS;

    // Page ids of this lane's chunks in a step: of the chunk whose K row it loads (r / 4), and of the
    // chunk whose V and scores it holds (g). -1: past the piece or the row, or outside the pool.
    struct Ids {
        int k[NP], v[NP];
    };
    auto load_ids = [&](int c, Ids& id) {  // c: the step's first chunk
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int ck = c + (r >> 2), cv = c + g;
            const int pk = ck * kChunk / BS + n, pv = cv * kChunk / BS + n;
            id.k[n] = ck < c1 && pk < nblk ? bt[pk] : -1;
            id.v[n] = cv < c1 && pv < nblk ? bt[pv] : -1;
        }
    };
    auto in_pool = [&](int id) { return (unsigned)id < (unsigned)p.pages.num_blocks; };

    // The query operand, negated where the scale is negative (its magnitude multiplies the scores).
    half8v qf[2 * KA];
#pragma unroll
    for (int a = 0; a < 2 * KA; ++a) {
        uint4 w{0, 0, 0, 0};
        if (r < nh)
            w = *reinterpret_cast<const uint4*>(p.q + (int64_t)b * p.q_sb + (int64_t)(h0 + r) * p.q_sh + 16 * g +
                                                64 * (a / 2) + 8 * (a & 1));
        const uint32_t sign = p.scale_log2e < 0.0f ? 0x80008000u : 0u;
        w.x ^= sign, w.y ^= sign, w.z ^= sign, w.w ^= sign;
        qf[a] = __builtin_bit_cast(half8v, w);
    }
    const float scale = fabsf(p.scale_log2e);

    st.m = kNegInf;
    float4v l = {0.0f, 0.0f, 0.0f, 0.0f};  // the denominator, as a product of the weights with ones
    const half8v ones = __builtin_bit_cast(half8v, BF16 ? uint4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}
                                                        : uint4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u});
#pragma unroll
    for (int e = 0; e < D / 16; ++e) st.acc[e] = float4v{0.0f, 0.0f, 0.0f, 0.0f};

    auto load_k = [&](int c, const Ids& id, Regs<D, BS>& rg) {
        // Token 4 j + r % 4 of chunk r / 4, dims 64 a + 16 g + [0, 16).
        const int base = BS > kChunk ? (c + (r >> 2)) * kChunk % BS : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = 4 * j / PT, slot = base + (4 * j) % PT + (r & 3);
            const int id_ = id.k[n];
            if (in_pool(id_)) {
                const uint8_t* run = p.pages.data + run_offset<D, BS>(p.pages, id_, kvh, 0) + slot * 64 + 16 * g;
#pragma unroll
                for (int a = 0; a < KA; ++a) rg.k[j][a] = load16<STREAM>(run + a * (BS * 64));
            }
        }
    };
    auto load_v = [&](int c, const Ids& id, Regs<D, BS>& rg) {
        // Token row of dim 16 e + r, chunk g; zero scale where there is no page.
        const int base = BS > kChunk ? (c + g) * kChunk % BS : 0;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            rg.codes[n] = 0;
            if (in_pool(id.v[n])) {
                rg.codes[n] = *reinterpret_cast<const uint16_t*>(p.pages.codes + code_offset(p.pages, id.v[n], kvh, 0));
                const uint8_t* run = p.pages.data + run_offset<D, BS>(p.pages, id.v[n], kvh, 1) + r * BS + base;
#pragma unroll
                for (int e = 0; e < D / 16; ++e) {
                    const uint8_t* src = run + e * (16 * BS);
                    if constexpr (PT == 16) {
                        const uint4 w = load16<STREAM>(src);
                        rg.v[e][0] = w.x, rg.v[e][1] = w.y, rg.v[e][2] = w.z, rg.v[e][3] = w.w;
                    } else if constexpr (PT == 8) {
                        const uint2 w = *reinterpret_cast<const uint2*>(src);
                        rg.v[e][2 * n] = w.x, rg.v[e][2 * n + 1] = w.y;
                    } else {
                        rg.v[e][n] = *reinterpret_cast<const uint32_t*>(src);
                    }
                }
            }
        }
    };

    Regs<D, BS> rg{};  // lanes without a page keep what is there: any bytes, masked (K) or at scale 0 (V)
    Ids id, next;
    load_ids(c0, id);
    load_k(c0, id, rg);
    load_v(c0, id, rg);
    load_ids(c0 + stride, next);
    for (int c = c0; c < c1; c += stride) {
        // Scores of tokens 4 j + i of chunk g.
        float4v s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int a = 0; a < KA; ++a) {
                s[j] = Elt<BF16>::mma32(ints8<BF16>(rg.k[j][a].x, rg.k[j][a].y), qf[2 * a], s[j]);
                s[j] = Elt<BF16>::mma32(ints8<BF16>(rg.k[j][a].z, rg.k[j][a].w), qf[2 * a + 1], s[j]);
            }
        }
        if (c + stride < c1) load_k(c + stride, next, rg);
        bool live[NP], all = true;
        float ks[NP];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            live[n] = in_pool(id.v[n]);
            if (!live[n] && r == 0 && p.err && c + g < c1 && (c + g) * kChunk / BS + n < nblk) atomicOr(p.err, 4);
            all = all && live[n];
            ks[n] = scale_of((int)(rg.codes[n] & 0xffu)) * scale;
        }
        // A step whose 64 tokens all count, one page a chunk: the page's scale multiplies the maximum and
        // goes into the exponent's fused multiply-add. Else every score is scaled, or masked, by itself.
        const bool whole = NP == 1 && (c + kStep) * kChunk <= tokens && c + kStep <= c1 &&
                           __builtin_amdgcn_ballot_w64(all) == ~(uint64_t)0;
        float mx = kNegInf, mul = 1.0f;
        if (whole) {
#pragma unroll
            for (int j = 0; j < 4; ++j) mx = fmaxf(fmaxf(mx, fmaxf(s[j][0], s[j][1])), fmaxf(s[j][2], s[j][3]));
            mul = ks[0];
            mx *= mul;
        } else {
            const int t0 = (c + g) * kChunk;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = 4 * j / PT;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[j][i] = live[n] && t0 + 4 * j + i < tokens ? s[j][i] * ks[n] : kNegInf;
                    mx = fmaxf(mx, s[j][i]);
                }
            }
        }
        if (__builtin_amdgcn_ballot_w64(mx > st.m + kLazyLog2) != 0) {
            mx = xor_max_16_32(mx);  // all lane groups of a head move together
            const bool grow = mx > st.m + kLazyLog2;
            const float now = grow ? mx : st.m;
            const float alpha = grow ? __builtin_amdgcn_exp2f(st.m - now) : 1.0f;  // 0 from -inf
            l *= alpha;
#pragma unroll
            for (int e = 0; e < D / 16; ++e) st.acc[e] *= alpha;
            st.m = now;
        }
        const float ref = st.m == kNegInf ? 0.0f : st.m;
        half8v pv[2];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                pv[j / 2][4 * (j & 1) + i] =
                    Elt<BF16>::round(__builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], mul, -ref)));
        l = Elt<BF16>::mma32(ones, pv[0], l);
        l = Elt<BF16>::mma32(ones, pv[1], l);
        RawScale<BF16> vs[NP];
        bool large = false;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            vs[n] = RawScale<BF16>((int)(rg.codes[n] >> 8));
            large = large || vs[n].excess != 1.0f;
        }
        if (__builtin_amdgcn_ballot_w64(large) != 0) {  // V beyond 4064 (fp16): the rest of its scale goes to the weights
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 4 * (j & 1) + i;  // pin_f32: not computed ahead of the branch, on every step
                    pv[j / 2][e] = Elt<BF16>::round(pin_f32(Elt<BF16>::widen(pv[j / 2][e])) * vs[4 * j / PT].excess);
                }
        }
#pragma unroll
        for (int e = 0; e < D / 16; ++e)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const half8v a = scaled4x2<BF16>(rg.v[e][2 * u], rg.v[e][2 * u + 1], vs[8 * u / PT], vs[(8 * u + 4) / PT]);
                st.acc[e] = Elt<BF16>::mma32(a, pv[u], st.acc[e]);
            }
        if (c + stride < c1) load_v(c + stride, next, rg);
        id = next;
        load_ids(c + 2 * stride, next);
    }
    st.l = l[0];
}

// A finished segment's output.
template <int D, bool BF16>
__device__ __forceinline__ void write_out(const AttnParams& p, int b, int h0, int nh, int lane, const Piece<D>& st) {
    const int g = lane >> 4, r = lane & 15;
    if (r >= nh) return;
    const float inv = st.l == 0.0f ? 0.0f : 1.0f / st.l;
    uint16_t* o = p.out + (int64_t)b * p.o_sb + (int64_t)(h0 + r) * p.o_sh + 4 * g;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) {
        half4v v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = Elt<BF16>::round(st.acc[e][i] * inv);
        *reinterpret_cast<uint2*>(o + 16 * e) = __builtin_bit_cast(uint2, v);
    }
}

__device__ __forceinline__ void heads_of(const AttnParams& p, int vh, int& kvh, int& h0, int& nh) {
    kvh = vh / p.NG;
    const int first = (vh - kvh * p.NG) * p.GS;
    h0 = kvh * p.G + first;
    nh = p.G - first < p.GS ? p.G - first : p.GS;
}

// LDS floats of a workgroup's (m, l) pairs, whole 16 bytes of them.
__host__ __device__ constexpr int stats_floats(int waves, int GS) { return (2 * waves * GS + 3) / 4 * 4; }

// One workgroup per segment: its waves take the steps in turn and join their pieces in LDS.
template <int D, int BS, bool BF16, bool STREAM>
__global__ __launch_bounds__(kSegmentWaves * 64, 2) void kv8_attn_segment_kernel(AttnParams p) {
    extern __shared__ __align__(16) float lds[];  // [waves][GS][2] (m, l), [waves][GS][D] outputs
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6, b = blockIdx.y;
    int kvh, h0, nh;
    heads_of(p, blockIdx.x, kvh, h0, nh);
    const int tokens = __builtin_amdgcn_readfirstlane(row_tokens<BS>(p, b));
    Piece<D> st;
    run_piece<D, BS, BF16, STREAM>(p, b, kvh, h0, nh, wave * kStep, chunks_of(tokens), waves * kStep, tokens, lane, st);
    if (waves == 1) {
        write_out<D, BF16>(p, b, h0, nh, lane, st);
        return;
    }
    float* const acc = lds + stats_floats(waves, p.GS);
    const int g = lane >> 4, r = lane & 15;
    if (r < nh) {
        if (g == 0) *reinterpret_cast<float2*>(lds + (wave * p.GS + r) * 2) = float2{st.m, st.l};
        float* a = acc + (wave * p.GS + r) * D + 4 * g;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) *reinterpret_cast<float4v*>(a + 16 * e) = st.acc[e];
    }
    __syncthreads();
    // 4 dims of a head a thread.
    const float kNegInf = -__builtin_huge_valf();
    for (int i = threadIdx.x; i < nh * (D / 4); i += blockDim.x) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float m = kNegInf;
        for (int w = 0; w < waves; ++w) m = fmaxf(m, lds[(w * p.GS + h) * 2]);
        const float ref = m == kNegInf ? 0.0f : m;
        float l = 0.0f;
        float4v num = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < waves; ++w) {
            const float f = __builtin_amdgcn_exp2f(lds[(w * p.GS + h) * 2] - ref);
            l += f * lds[(w * p.GS + h) * 2 + 1];
            num += f * *reinterpret_cast<const float4v*>(acc + (w * p.GS + h) * D + d);
        }
        half4v v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = Elt<BF16>::round(l == 0.0f ? 0.0f : num[k] / l);
        *reinterpret_cast<uint2*>(p.out + (int64_t)b * p.o_sb + (int64_t)(h0 + h) * p.o_sh + d) =
            __builtin_bit_cast(uint2, v);
    }
}

template <int D, int BS, bool BF16, bool STREAM>
__global__ __launch_bounds__(kAttnWaves * 64, 2) void kv8_attn_kernel(AttnParams p) {
    const int lane = threadIdx.x & 63;
    const int w = blockIdx.x * kAttnWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Piece<D> st;
    int kvh, h0, nh;
    // Up to 64 rows: one read of the lengths, a row a lane. More: their sum first, then 64 at a time.
    const bool one_pass = p.B <= 64;
    int at = 0, before = 0, tok = 0, incl = 0, total;  // rows [at, at + 64) in the lanes; chunks before them
    if (!one_pass) sum_rows<BS>(p, 0, lane, before, total);
    auto load_rows = [&]() {
        tok = at + lane < p.B ? row_tokens<BS>(p, at + lane) : 0;
        incl = incl_scan(chunks_of(tok), lane);
    };
    load_rows();
    if (one_pass) total = __builtin_amdgcn_readlane(incl, 63);
    const Cut cut(total * p.Hv, p.workers);
    if (w >= cut.W) return;
    int x = cut.lo(w);
    const int x0 = x, hi = cut.lo(w + 1);
    while (x < hi) {
        while (!one_pass && (before + __builtin_amdgcn_readlane(incl, 63)) * p.Hv <= x && at + 64 < p.B) {
            before += __builtin_amdgcn_readlane(incl, 63);
            at += 64;
            load_rows();
        }
        // The last row that begins at or before chunk x: a row without tokens ends where it begins.
        const int first = before + incl - chunks_of(tok);
        const int i = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at + lane < p.B && first * p.Hv <= x)) - 1;
        const int tokens = __builtin_amdgcn_readlane(tok, i), n = chunks_of(tokens), b = at + i;
        const int rel = x - __builtin_amdgcn_readlane(first, i) * p.Hv;
        const int vh = n > 0 ? rel / n : p.Hv, c0 = rel - vh * n;
        const int nc = n - c0 < hi - x ? n - c0 : hi - x;
        if (nc <= 0 || vh >= p.Hv) break;  // cannot happen for lengths that stay as they are
        heads_of(p, vh, kvh, h0, nh);
        run_piece<D, BS, BF16, STREAM>(p, b, kvh, h0, nh, c0, c0 + nc, kStep, tokens, lane, st);
        if (nc == n) {
            write_out<D, BF16>(p, b, h0, nh, lane, st);
        } else {
            // A range holds at most two shared pieces: the one it begins with and the one it ends with.
            const int64_t slot = 2 * (int64_t)w + (x == x0 ? 0 : 1);
            const int g = lane >> 4, r = lane & 15;
            if (r < nh) {
                if (g == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * p.GS + r) * 2) = float2{st.m, st.l};
                float* a = p.part_acc + (slot * p.GS + r) * D + 4 * g;
#pragma unroll
                for (int e = 0; e < D / 16; ++e) *reinterpret_cast<float4v*>(a + 16 * e) = st.acc[e];
            }
        }
        x += nc;
    }
}

// Joins a segment's pieces and writes its heads; zeros for a row without tokens. One workgroup per query
// head and row. 4 dims a lane, so a wave's load holds 256 / D pieces and the workgroup's 1024 / D; the
// pieces' (m, l) stand in every wave, a piece a lane, and no load waits for a weight. What remains is a
// chain: lengths, cut, pieces, LDS. A loop with a lane's weights one after the other, one piece a wave and
// step, took 16.8 us for 128 pieces (two rows of 100,000 tokens) and 4.9 for 9.
constexpr int kMergeWaves = 4, kMergeLoads = 4;
template <int D, int BS, bool BF16>
__global__ __launch_bounds__(kMergeWaves * 64) void kv8_merge_kernel(AttnParams p) {
    constexpr int LP = D / 4, PW = 64 / LP, PB = kMergeWaves * PW;  // lanes per piece; pieces per wave, workgroup
    __shared__ float4v red[PB][LP];
    const int h = blockIdx.x, b = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = h / p.G, hg = h - kvh * p.G;
    const int vh = kvh * p.NG + hg / p.GS, r = hg % p.GS;
    int before, total;
    sum_rows<BS>(p, b, lane, before, total);
    const int n = chunks_of(row_tokens<BS>(p, b));
    uint16_t* o = p.out + (int64_t)b * p.o_sb + (int64_t)h * p.o_sh;
    if (n == 0) {
        if (threadIdx.x < D) o[threadIdx.x] = 0;
        return;
    }
    const Cut cut(total * p.Hv, p.workers);
    const int x = before * p.Hv + vh * n;
    const int w0 = cut.worker_of(x), np = cut.worker_of(x + n - 1) - w0 + 1;
    if (np == 1) return;  // one wave had the whole segment and wrote it
    const float kNegInf = -__builtin_huge_valf();
    const bool cut_first = cut.lo(w0) < x;  // the first piece is its range's last, not its first
    auto slot = [&](int k) { return (2 * (int64_t)(w0 + k) + (k == 0 && cut_first ? 1 : 0)) * p.GS + r; };
    float m = kNegInf, l = 0.0f;
    float4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < np; k0 += 64) {
        const int most = np - k0 < 64 ? np - k0 : 64;
        float2 ml = {kNegInf, 0.0f};
        if (lane < most) ml = *reinterpret_cast<const float2*>(p.part_ml + slot(k0 + lane) * 2);
        float scale = 0.0f, f = 0.0f;
        for (int k = 0; k < most; k += PB * kMergeLoads) {
            float4v a[kMergeLoads];
#pragma unroll
            for (int u = 0; u < kMergeLoads; ++u) {
                const int i = k + u * PB + wave * PW + lane / LP;
                a[u] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
                if (i < most) a[u] = *reinterpret_cast<const float4v*>(p.part_acc + slot(k0 + i) * D + lane % LP * 4);
            }
            if (k == 0) {  // the weights, while the first outputs are on their way
                const float now = fmaxf(m, wave_max(ml.x)), ref = now == kNegInf ? 0.0f : now;
                scale = __builtin_amdgcn_exp2f(m - ref);
                f = __builtin_amdgcn_exp2f(ml.x - ref);
                l = l * scale + f * ml.y;
                acc *= scale;
                m = now;
            }
#pragma unroll
            for (int u = 0; u < kMergeLoads; ++u) {
                const int i = k + u * PB + wave * PW + lane / LP;
                const float wgt = __shfl(f, i < most ? i : 0);
                if (i < most) acc += wgt * a[u];
            }
        }
    }
    l = wave_sum(l);
    red[wave * PW + lane / LP][lane % LP] = acc;
    __syncthreads();
    if (threadIdx.x >= LP) return;
    float4v num = red[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < PB; ++i) num += red[i][threadIdx.x];
    half4v v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = Elt<BF16>::round(l == 0.0f ? 0.0f : num[i] / l);
    *reinterpret_cast<uint2*>(o + threadIdx.x * 4) = __builtin_bit_cast(uint2, v);
}

// Whether every segment gets a workgroup of its own, from what both forms were measured to take (us):
// 4.7 and the longest row's bytes at 50 GB/s, which is all that one CU streams of such pages, against 9 and
// the bytes of half-full tables at 5.4 TB/s. Of tables up to 1 MiB per segment only: with wider ones a
// single long row among short ones would keep one CU at work for 20 us and more. Measured, one against the
// other: 8 segments of 100 tokens 4.5 and 10.0 us, 14 of up to 1501 (bf16, D = 64) 7.7 and 10.1, 128 of up
// to 2000 17.4 and 18.7; about even 256 of up to 4096 (the tables' whole width 34.1 and 36.0, U[128, 4096]
// 32.7 and 31.5); the other way 8 of 1024 10.6 and 8.2, 64 of up to 4096 26.9 and 18.9. The rule sees the
// tables' width, not the lengths: rows much shorter than their tables, or one long row among short ones,
// can take the slower form.
static bool by_segment(int64_t segments, int64_t max_tokens, int D) {
    const double bytes = (double)max_tokens * D * 2;
    return bytes <= 1 << 20 && 4.7 + bytes / 50e3 <= 9.0 + segments * bytes / 2 / 5.4e6;
}

static void head_groups(int G, int& NG, int& GS) {
    NG = (int)ceil_div(G, kHeads);
    GS = (int)ceil_div(G, NG);
    NG = (int)ceil_div(G, GS);
}

}  // namespace kv8
}  // namespace mx

using namespace mx;

extern "C" size_t mx_kv8_attn_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_blocks,
                                              int32_t block_size) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_blocks <= 0 || block_size <= 0 || Hq % Hkv != 0) return 0;
    int NG, GS;
    kv8::head_groups(Hq / Hkv, NG, GS);
    if (kv8::by_segment((int64_t)B * Hkv * NG, (int64_t)max_blocks * block_size, D)) return 0;
    return (size_t)2 * kv8::kWorkers * GS * (D + 2) * sizeof(float);
}

extern "C" int mx_kv8_attn_decode(const uint16_t* q, int64_t q_sb, int64_t q_sh, const uint8_t* data,
                                  const uint8_t* codes, const int32_t* block_tables, int64_t bt_sb, int32_t max_blocks,
                                  const int32_t* seq_lens, int32_t B, int32_t Hq, int32_t Hkv, int32_t D,
                                  int32_t block_size, int32_t num_blocks, float scale, uint16_t* out, int64_t o_sb,
                                  int64_t o_sh, void* workspace, size_t workspace_bytes, int32_t* err, uint32_t flags,
                                  void* stream) {
    const char* what = "mx_kv8_attn_decode";
    if (B < 0) return fail(MX_ERR_INVALID, "%s: B must be >= 0", what);
    if (B == 0) return MX_OK;
    if (!q || !block_tables || !seq_lens || !out) return fail(MX_ERR_NULL, "%s: null pointer", what);
    int rc = kv8::check_pages(what, data, codes, Hkv, D, block_size, num_blocks);
    if (rc != MX_OK) return rc;
    if (Hq < 1 || Hq % Hkv != 0)
        return fail(MX_ERR_INVALID, "%s: Hq (%d) must be a positive multiple of Hkv (%d)", what, Hq, Hkv);
    if (max_blocks < 1) return fail(MX_ERR_INVALID, "%s: max_blocks must be >= 1", what);
    if (B > 65535 || Hq > 65535) return fail(MX_ERR_UNSUPPORTED, "%s: B or Hq too large", what);
    if (flags & ~(uint32_t)(MX_PA_BF16 | MX_PA_SHARED_BLOCKS))
        return fail(MX_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
    const bool shared = flags & MX_PA_SHARED_BLOCKS;
    if (!aligned(q, 16) || q_sb % 8 || q_sh % 8 || !aligned(out, 16) || o_sb % 8 || o_sh % 8)
        return fail(MX_ERR_ALIGNMENT, "%s: q and out rows must be 16-byte aligned", what);
    if (!aligned(codes, 2)) return fail(MX_ERR_ALIGNMENT, "%s: codes must be 2-byte aligned", what);
    const int64_t max_tokens = (int64_t)max_blocks * block_size;
    kv8::AttnParams p{};
    p.q = q, p.q_sb = q_sb, p.q_sh = q_sh;
    p.pages = {const_cast<uint8_t*>(data), const_cast<uint8_t*>(codes), Hkv, num_blocks};
    p.bt = block_tables, p.bt_sb = bt_sb, p.max_blocks = max_blocks, p.seq_lens = seq_lens;
    p.B = B, p.G = Hq / Hkv;
    kv8::head_groups(p.G, p.NG, p.GS);
    p.Hv = Hkv * p.NG;
    if (max_tokens > kv8::kMaxTokens || (int64_t)B * p.Hv * ceil_div(max_tokens, kv8::kChunk) > (int64_t)1 << 30)
        return fail(MX_ERR_UNSUPPORTED, "%s: more tokens than 32-bit numbers hold", what);
    const bool segments = kv8::by_segment((int64_t)B * p.Hv, max_tokens, D);
    p.workers = kv8::kWorkers;
    p.scale_log2e = scale * 1.4426950408889634f;
    p.out = out, p.o_sb = o_sb, p.o_sh = o_sh, p.err = err;
    if (!segments) {
        const size_t need = mx_kv8_attn_workspace_bytes(B, Hq, Hkv, D, max_blocks, block_size);
        if (!workspace || workspace_bytes < need)
            return fail(MX_ERR_WORKSPACE, "%s: workspace needs %zu bytes, got %zu", what, need, workspace_bytes);
        if (!aligned(workspace, 256)) return fail(MX_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", what);
        p.part_acc = static_cast<float*>(workspace);
        p.part_ml = p.part_acc + (size_t)2 * p.workers * p.GS * D;
    }
    hipStream_t st = as_stream(stream);
    // Waves of a segment's workgroup: at most a step each at the table's width, within 64 KiB of LDS. A CU
    // holds 8 of them: where there are more segments than CUs, two workgroups of 4 beat one of 8 (1024
    // segments of up to 300 tokens 24.5 -> 18.2 us, of up to 2048 63.6 -> 59.6).
    const int64_t piece = (int64_t)p.GS * (D + 2) * sizeof(float);
    const int64_t most = (int64_t)B * p.Hv > 256 ? kv8::kSegmentWaves / 2 : kv8::kSegmentWaves;
    const int waves = (int)std::min<int64_t>({most, ceil_div(max_tokens, kv8::kStep * kv8::kChunk),
                                              65520 / piece});
    const size_t lds = waves > 1 ? (kv8::stats_floats(waves, p.GS) + (size_t)waves * p.GS * D) * sizeof(float) : 0;
#define LAUNCH(DD, BB, F, S)                                                                                           \
    if (segments) {                                                                                                    \
        hipLaunchKernelGGL((kv8::kv8_attn_segment_kernel<DD, BB, F, S>), dim3(p.Hv, B), dim3(waves * 64), lds, st, p); \
    } else {                                                                                                           \
        hipLaunchKernelGGL((kv8::kv8_attn_kernel<DD, BB, F, S>), dim3(kv8::kWorkers / kv8::kAttnWaves),                \
                           dim3(kv8::kAttnWaves * 64), 0, st, p);                                                      \
        hipLaunchKernelGGL((kv8::kv8_merge_kernel<DD, BB, F>), dim3(Hq, B), dim3(kv8::kMergeWaves * 64), 0, st, p);    \
    }
#define CALL(DD, BB)                                        \
    if (flags & MX_PA_BF16) {                               \
        if (shared) { LAUNCH(DD, BB, true, false) }         \
        else { LAUNCH(DD, BB, true, true) }                 \
    } else {                                                \
        if (shared) { LAUNCH(DD, BB, false, false) }        \
        else { LAUNCH(DD, BB, false, true) }                \
    }
    MX_KV8_DISPATCH(D, block_size, CALL)
#undef CALL
#undef LAUNCH
    return check_launch(what);
}
