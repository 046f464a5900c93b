// Writing and reading the 8-bit KV cache (kv8.h: its pages) on gfx950.
//
// kv8_write quantises new K/V states into a layer's pages, kv8_rope_append does so for a decode
// step's fused QKV rows after rotating them, kv8_gather reads whole rows back in 16 bits. They are
// the 8-bit forms of kv_append, qkv_rope_append and kv_gather (decode_glue.hip), which replace
// GpuKVBlockPool.write_tokens_batch and gather_layer (runtime/phase2/paged_kv_kernel.py:176-309).
//
// One wave owns one run, the K or the V of one page and head, and does everything for it: the
// largest magnitude of the new tokens, the run's new scale, the kept tokens at that scale, the new
// ones. No two waves of a launch touch the same run as long as no page stands in two rows' written
// ranges, so nothing is ordered between waves. K is handled by (token, 8 dims) pieces, as its 16-byte
// loads come; V by dims, each lane holding every token of its D / 64 dims, so that the token-minor
// rows are built in registers without a transpose.
#include <type_traits>

#include "common.h"
#include "glue_common.h"
#include "kv8.h"

namespace mx {
namespace kv8 {

constexpr int kWaves = 4;  // waves per workgroup

struct WriteParams {
    const uint16_t* k_new;
    const uint16_t* v_new;
    int64_t sb, sh, st;  // element strides of the new states [B, Hkv, T, D]
    int T;
    const int32_t* bt;
    int64_t bt_sb;
    int max_blocks;
    const int32_t* start;
    Pages pages;
    int32_t* err;
    uint8_t* used;  // optional [num_blocks] map: 1 where a token was written
    int pages_per_row;  // pages a row's write can touch: T tokens that begin inside a page
    int stream;         // the states are read with the streaming policy
    int64_t units;
};

// States larger than the L2s together are gone from them when the next reader comes, and read with the
// streaming policy they displace nothing: 134 MB of them 50 -> 37 us. Smaller ones, 8 MB that the L2s still
// hold, take 6.6 us that way and 5.9 with the default.
constexpr int64_t kStreamBytes = 32 << 20;
typedef uint32_t u32x4n __attribute__((ext_vector_type(4)));

// A run's codes: the one it had (0 when the write starts the page anew) and the one it gets.
struct Codes {
    int old, now;
};

// The K tokens below slot o at a larger scale.
template <int D, int BS>
__device__ __forceinline__ void regrow_k(uint8_t* run, int o, Codes c, int lane) {
    const float f = growth_factor(c.old, c.now);
    for (int i = lane; i < o * (D / 8); i += 64) {
        const int s = i / (D / 8), d = (i % (D / 8)) * 8;
        uint2* p = reinterpret_cast<uint2*>(run + (d / 64) * (BS * 64) + s * 64 + d % 64);
        const uint2 w = *p;
        *p = uint2{requant4(w.x, f), requant4(w.y, f)};
    }
}

// Bytes [lo, hi) of the 4-byte word that begins at byte `at`.
__device__ __forceinline__ uint32_t byte_mask(int lo, int hi, int at) {
    const int a = lo - at < 0 ? 0 : (lo - at > 4 ? 4 : lo - at), b = hi - at < 0 ? 0 : (hi - at > 4 ? 4 : hi - at);
    return (uint32_t)(((uint64_t)1 << (8 * b)) - ((uint64_t)1 << (8 * a)));  // 0 where a == b
}

// The whole V run: kept tokens below slot o, new ones in [o, e), zero from e on. x[s]: the lane's
// D / 64 dims of slot s (16-bit patterns, low half first).
template <int D, int BS, bool BF16>
__device__ __forceinline__ void store_v(uint8_t* run, int o, int e, Codes c, const uint32_t (&x)[BS],
                                        const uint32_t (&kept)[D / 64][BS / 4], int lane) {
    constexpr int DP = D / 64, W = BS / 4;
    const Quant quant(c.now);
    uint32_t row[DP * W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const uint32_t fresh = byte_mask(o, e, 4 * w), was = byte_mask(0, o, 4 * w);
#pragma unroll
        for (int j = 0; j < DP; ++j) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = widen<BF16>(j == 0 ? x[4 * w + i] & 0xffffu : x[4 * w + i] >> 16);
            row[j * W + w] = (quant.word(v[0], v[1], v[2], v[3]) & fresh) | (0x80808080u & ~(fresh | was));
        }
    }
    if (o > 0) {
        const float f = growth_factor(c.old, c.now);
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int j = 0; j < DP; ++j)
                row[j * W + w] |= (c.old == c.now ? kept[j][w] : requant4(kept[j][w], f)) & byte_mask(0, o, 4 * w);
    }
    uint8_t* dst = run + lane * (DP * BS);
    if constexpr (DP * W % 4 == 0) {
#pragma unroll
        for (int w = 0; w < DP * W; w += 4)
            *reinterpret_cast<uint4*>(dst + 4 * w) = uint4{row[w], row[w + 1], row[w + 2], row[w + 3]};
    } else if constexpr (DP * W == 2) {
        *reinterpret_cast<uint2*>(dst) = uint2{row[0], row[1]};
    } else {
        *reinterpret_cast<uint32_t*>(dst) = row[0];
    }
}

// The lane's rows of a V run as it was (read only where tokens are kept).
template <int D, int BS>
__device__ __forceinline__ void load_v(const uint8_t* run, int o, uint32_t (&kept)[D / 64][BS / 4], int lane) {
    constexpr int DP = D / 64, W = BS / 4;
#pragma unroll
    for (int j = 0; j < DP; ++j)
#pragma unroll
        for (int w = 0; w < W; ++w) kept[j][w] = 0;
    if (o == 0) return;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(run + lane * (DP * BS));
#pragma unroll
    for (int j = 0; j < DP; ++j)
#pragma unroll
        for (int w = 0; w < W; ++w) kept[j][w] = src[j * W + w];
}

// Grows a run's scale to hold `bits` (the new tokens' largest magnitude) and stores it. old: the scale it
// had where tokens are kept, else 0.
template <bool BF16>
__device__ __forceinline__ Codes grow(uint8_t* code, int old, uint32_t bits, int lane) {
    const int need = code_of<BF16>(bits);
    const int now = old > need ? old : need;
    if (lane == 0) *code = (uint8_t)now;
    return Codes{old, now};
}

template <int D, int BS, bool BF16>
__global__ __launch_bounds__(kWaves * 64) void kv8_write_kernel(WriteParams p) {
    constexpr int CH = D / 8;        // 8-dim pieces of a token
    constexpr int TPI = 64 / CH;     // tokens of one K load
    constexpr int NI = (BS + TPI - 1) / TPI, DP = D / 64;
    const int lane = threadIdx.x & 63;
    int64_t u = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= p.units) return;
    const int kind = (int)(u & 1);
    u >>= 1;
    const int h = (int)(u % p.pages.Hkv);
    u /= p.pages.Hkv;
    const int j = (int)(u % p.pages_per_row);
    const int b = (int)(u / p.pages_per_row);

    // The page's share [lo, hi) of the row's new positions; negative positions are skipped and flagged.
    const int64_t start = p.start[b], end = start + p.T;
    const int64_t first = start > 0 ? start : 0;
    const int64_t lb = first / BS + j;
    const int64_t lo = lb * BS > first ? lb * BS : first;
    const int64_t hi = (lb + 1) * BS < end ? (lb + 1) * BS : end;
    const bool flags = lane == 0 && kind == 0 && h == 0 && p.err;
    if (start < 0 && j == 0 && flags) atomicOr(p.err, 1);
    if (lo >= hi) return;
    const int o = (int)(lo - lb * BS), e = (int)(hi - lb * BS);
    // The new tokens, all loads at once and ahead of the page's: slots outside [o, e) load a neighbour's
    // token again, which a branch per slot would not be faster than.
    const int64_t src = (int64_t)b * p.sb + (int64_t)h * p.sh + (lo - start) * p.st;
    auto offset = [&](int s) { return (int64_t)((s < o ? o : (s < e ? s : e - 1)) - o) * p.st; };
    uint4 xk[NI];
    uint32_t xv[BS];
    if (kind == 0) {
        auto at = [&](int i) { return p.k_new + src + offset(i * TPI + lane / CH) + (lane % CH) * 8; };
        if (p.stream) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
                xk[i] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4n*>(at(i))));
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) xk[i] = glue::ld16(at(i));
        }
    } else {
        typedef typename std::conditional<DP == 2, uint32_t, uint16_t>::type Elem;
        auto at = [&](int s) { return reinterpret_cast<const Elem*>(p.v_new + src + offset(s) + lane * DP); };
        if (p.stream) {
#pragma unroll
            for (int s = 0; s < BS; ++s) xv[s] = __builtin_nontemporal_load(at(s));
        } else {
#pragma unroll
            for (int s = 0; s < BS; ++s) xv[s] = *at(s);
        }
    }
    const int phys = lb < p.max_blocks ? p.bt[(int64_t)b * p.bt_sb + lb] : -1;
    if ((unsigned)phys >= (unsigned)p.pages.num_blocks) {
        if (flags) atomicOr(p.err, 1);
        return;
    }
    uint8_t* run = p.pages.data + run_offset<D, BS>(p.pages, phys, h, kind);
    uint8_t* code = p.pages.codes + code_offset(p.pages, phys, h, kind);
    const int old = o > 0 ? *code : 0;
    uint32_t m = 0;
    if (kind == 0) {
        if (p.used && h == 0 && lane == 0) p.used[phys] = 1;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            m = max_u16x2(m, max_u16x2(xk[i].x & 0x7fff7fffu, xk[i].y & 0x7fff7fffu));
            m = max_u16x2(m, max_u16x2(xk[i].z & 0x7fff7fffu, xk[i].w & 0x7fff7fffu));
        }
        const Codes cd = grow<BF16>(code, old, wave_max_u16x2(m), lane);
        if (cd.now != cd.old && cd.now != kPoison) regrow_k<D, BS>(run, o, cd, lane);
        const Quant quant(cd.now);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int s = i * TPI + lane / CH, d = (lane % CH) * 8;
            const uint32_t w[4] = {xk[i].x, xk[i].y, xk[i].z, xk[i].w};
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = widen<BF16>(q & 1 ? w[q / 2] >> 16 : w[q / 2] & 0xffffu);
            if (s >= o && s < e)
                *reinterpret_cast<uint2*>(run + (d / 64) * (BS * 64) + s * 64 + d % 64) =
                    uint2{quant.word(v[0], v[1], v[2], v[3]), quant.word(v[4], v[5], v[6], v[7])};
        }
    } else {
        uint32_t kept[DP][BS / 4];
        load_v<D, BS>(run, o, kept, lane);
#pragma unroll
        for (int s = 0; s < BS; ++s) m = max_u16x2(m, xv[s] & 0x7fff7fffu);
        const Codes cd = grow<BF16>(code, old, wave_max_u16x2(m), lane);
        store_v<D, BS, BF16>(run, o, e, cd, xv, kept, lane);
    }
}

struct GatherParams {
    Pages pages;
    const int32_t* bt;
    int64_t bt_sb;
    int max_blocks;
    const int32_t* lens;  // NULL: every row has S tokens
    int S, pages_per_row;
    uint16_t* k_out;  // [B, Hkv, S, D]
    uint16_t* v_out;
    int32_t* err;
    int64_t units;
};

// Rows of the cache as 16-bit K and V: a wave reads one run and writes its tokens, zero past the
// row's length.
template <int D, int BS, bool BF16>
__global__ __launch_bounds__(kWaves * 64) void kv8_gather_kernel(GatherParams p) {
    constexpr int CH = D / 8, TPI = 64 / CH, NI = (BS + TPI - 1) / TPI, DP = D / 64;
    const int lane = threadIdx.x & 63;
    int64_t u = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= p.units) return;
    const int kind = (int)(u & 1);
    u >>= 1;
    const int j = (int)(u % p.pages_per_row);
    u /= p.pages_per_row;
    const int h = (int)(u % p.pages.Hkv);
    const int b = (int)(u / p.pages.Hkv);
    const int64_t base = (int64_t)j * BS;
    const int n = p.S - base < BS ? (int)(p.S - base) : BS;  // slots that the output holds
    int64_t left = (p.lens ? p.lens[b] : p.S) - base;         // ... and that hold tokens
    int live = left < 0 ? 0 : (left < n ? (int)left : n);
    int phys = 0;
    if (live > 0) {
        phys = j < p.max_blocks ? p.bt[(int64_t)b * p.bt_sb + j] : -1;
        if ((unsigned)phys >= (unsigned)p.pages.num_blocks) {
            if (lane == 0 && kind == 0 && h == 0 && p.err) atomicOr(p.err, 1);
            live = phys = 0;
        }
    }
    const uint8_t* run = p.pages.data + run_offset<D, BS>(p.pages, phys, h, kind);
    const float s = scale_of(p.pages.codes[code_offset(p.pages, phys, h, kind)]);
    uint16_t* out = (kind == 0 ? p.k_out : p.v_out) + (((int64_t)b * p.pages.Hkv + h) * p.S + base) * D;
    if (kind == 0) {
        const int c = lane % CH;
        uint2 x[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int t = i * TPI + lane / CH;
            x[i] = uint2{0, 0};
            if (t < live) x[i] = *reinterpret_cast<const uint2*>(run + (c * 8 / 64) * (BS * 64) + t * 64 + c * 8 % 64);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int t = i * TPI + lane / CH;
            if (t >= n) continue;
            half8v v = values8<BF16>(x[i].x, x[i].y, s);
            if (t >= live) v = half8v{};
            glue::st16(out + t * D + c * 8, glue::as_u4(v));
        }
    } else {
        uint32_t row[DP][BS / 4];
        load_v<D, BS>(run, live, row, lane);
#pragma unroll
        for (int t0 = 0; t0 < BS; t0 += 4) {
            half8v v;  // 4 tokens of the lane's dims
            if constexpr (DP == 2) v = values8<BF16>(row[0][t0 / 4], row[DP - 1][t0 / 4], s);
            else v = values8<BF16>(row[0][t0 / 4], row[0][t0 / 4], s);
            const uint4 w = glue::as_u4(v);
            const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + i;
                if (t >= n) continue;
                const uint32_t lo = (a[i / 2] >> (16 * (i & 1))) & 0xffffu;
                const uint32_t hi = (a[2 + i / 2] >> (16 * (i & 1))) & 0xffffu;
                if constexpr (DP == 2)
                    *reinterpret_cast<uint32_t*>(out + t * D + lane * 2) = t < live ? (lo | hi << 16) : 0u;
                else
                    out[t * D + lane] = t < live ? (uint16_t)lo : (uint16_t)0;
            }
        }
    }
}

struct TokenParams {
    const uint16_t* qkv;  // rows of (Hq + 2 Hkv) * D, or NULL with part != NULL
    int64_t qkv_stride;
    const float* part;    // split-K partials [splits][B][(Hq + 2 Hkv) * D] of the producing linear
    int splits;
    int64_t split_stride;
    const uint16_t* bias;  // added to the partial sums (NULL: none)
    int Hq;
    const float2* rope;  // [max_pos][D/2] (cos, sin)
    int max_pos;
    const int32_t* positions;
    uint16_t* q_out;
    int64_t q_stride;
    const int32_t* bt;
    int64_t bt_sb;
    int max_blocks;
    Pages pages;
    int32_t* err;
    int32_t* lens_out;  // optional: lens_out[b] = positions[b] + 1
    uint8_t* used;
    int64_t units;
};

template <bool BF16>
__device__ __forceinline__ uint32_t round16(float v) {
    if constexpr (BF16) return __builtin_bit_cast(uint16_t, (__bf16)pin_f32(v));
    return __builtin_bit_cast(uint16_t, (_Float16)pin_f32(v));
}

// One element of the QKV projection's output, as the linear would have written it (16-bit pattern).
template <bool BF16>
__device__ __forceinline__ uint32_t qkv_element(const TokenParams& p, int b, int width, int col) {
    if (!p.part) return p.qkv[(int64_t)b * p.qkv_stride + col];
    float acc = p.bias ? widen<BF16>(p.bias[col]) : 0.0f;
    const float* q = p.part + (int64_t)b * width + col;
    for (int s0 = 0; s0 < p.splits; s0 += 8) {  // 8 loads in flight, added in order
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = q[(s0 + u < p.splits ? s0 + u : p.splits - 1) * p.split_stride];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (s0 + u < p.splits) acc += v[u];
    }
    return round16<BF16>(acc);
}

// One wave per head of a row: a q head is rotated and written out, a k head rotated and written to
// the row's page, a v head written there.
template <int D, int BS, bool BF16>
__global__ __launch_bounds__(kWaves * 64) void kv8_token_kernel(TokenParams p) {
    constexpr int HALF = D / 2, DP = D / 64;
    const int lane = threadIdx.x & 63;
    int64_t u = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= p.units) return;
    const int heads = p.Hq + 2 * p.pages.Hkv, width = heads * D;
    const int hs = (int)(u % heads), b = (int)(u / heads);
    const int pos = p.positions[b];
    const bool pos_ok = pos >= 0 && pos < p.max_pos;
    if (hs == 0 && lane == 0) {
        if (p.lens_out) p.lens_out[b] = pos + 1;
        if (!pos_ok && p.err) atomicOr(p.err, 2);
    }
    const bool is_v = hs >= p.Hq + p.pages.Hkv;
    // q and k: dims lane and lane + 64 (D = 128) or dim lane (D = 64); their rotate-half partners are
    // the other of the two, or lane ^ 32's.
    uint32_t x[DP];
#pragma unroll
    for (int j = 0; j < DP; ++j)
        x[j] = qkv_element<BF16>(p, b, width, hs * D + (is_v ? lane * DP + j : lane + 64 * j));
    if (!is_v) {
        const float2 cs = pos_ok ? p.rope[(int64_t)pos * HALF + lane % HALF] : float2{0.0f, 0.0f};
        // Each output is one fma of a rounded product, rounded once more to 16 bits (rope_rotate).
        if constexpr (DP == 2) {
            const float a = widen<BF16>(x[0]), c = widen<BF16>(x[1]);
            x[0] = round16<BF16>(__builtin_fmaf(a, cs.x, -pin_f32(c * cs.y)));
            x[1] = round16<BF16>(__builtin_fmaf(c, cs.x, pin_f32(a * cs.y)));
        } else {
            const float a = widen<BF16>(x[0]), other = __shfl_xor(a, 32);
            const float prod = pin_f32(other * cs.y);
            x[0] = round16<BF16>(__builtin_fmaf(a, cs.x, lane < 32 ? -prod : prod));
        }
        if (hs < p.Hq) {
            uint16_t* q = p.q_out + (int64_t)b * p.q_stride + hs * D + lane;
#pragma unroll
            for (int j = 0; j < DP; ++j) q[64 * j] = pos_ok ? (uint16_t)x[j] : (uint16_t)0;
            return;
        }
    }
    if (!pos_ok) return;
    const int lb = pos / BS, o = pos % BS;
    const int phys = lb < p.max_blocks ? p.bt[(int64_t)b * p.bt_sb + lb] : -1;
    const int kvh = is_v ? hs - p.Hq - p.pages.Hkv : hs - p.Hq;
    if ((unsigned)phys >= (unsigned)p.pages.num_blocks) {
        if (p.err && lane == 0 && hs == p.Hq) atomicOr(p.err, 1);
        return;
    }
    uint8_t* run = p.pages.data + run_offset<D, BS>(p.pages, phys, kvh, is_v);
    uint8_t* code = p.pages.codes + code_offset(p.pages, phys, kvh, is_v);
    const int old = o > 0 ? *code : 0;
    uint32_t m = x[0];
    if constexpr (DP == 2) m |= x[1] << 16;
    if (!is_v) {
        if (p.used && kvh == 0 && lane == 0) p.used[phys] = 1;
        const Codes cd = grow<BF16>(code, old, wave_max_u16x2(m & 0x7fff7fffu), lane);
        if (cd.now != cd.old && cd.now != kPoison) regrow_k<D, BS>(run, o, cd, lane);
        const Quant quant(cd.now);
#pragma unroll
        for (int j = 0; j < DP; ++j) run[j * (BS * 64) + o * 64 + lane] = (uint8_t)quant.byte(widen<BF16>(x[j]));
    } else {
        uint32_t kept[DP][BS / 4], xs[BS];
        load_v<D, BS>(run, o, kept, lane);
        const Codes cd = grow<BF16>(code, old, wave_max_u16x2(m & 0x7fff7fffu), lane);
#pragma unroll
        for (int s = 0; s < BS; ++s) xs[s] = m;
        store_v<D, BS, BF16>(run, o, o + 1, cd, xs, kept, lane);
    }
}

// Workgroups of a launch over `units` waves, or -1 where one launch does not hold them.
static int64_t groups_for(int64_t units) {
    const int64_t n = ceil_div(units, kWaves);
    return n * kWaves * 64 < ((int64_t)1 << 32) ? n : -1;
}

}  // namespace kv8
}  // namespace mx

using namespace mx;

extern "C" int mx_kv8_write(const uint16_t* k_new, const uint16_t* v_new, int64_t new_sb, int64_t new_sh,
                            int64_t new_st, int32_t B, int32_t T, int32_t Hkv, int32_t D, const int32_t* block_tables,
                            int64_t bt_sb, int32_t max_blocks, const int32_t* start_pos, uint8_t* data, uint8_t* codes,
                            int32_t block_size, int32_t num_blocks, int32_t* err, uint8_t* used, uint32_t flags,
                            void* stream) {
    const char* what = "mx_kv8_write";
    if (B < 0 || T < 0) return fail(MX_ERR_INVALID, "%s: B and T must be >= 0", what);
    if (B == 0 || T == 0) return MX_OK;
    if (!k_new || !v_new || !block_tables || !start_pos) return fail(MX_ERR_NULL, "%s: null pointer", what);
    int rc = kv8::check_pages(what, data, codes, Hkv, D, block_size, num_blocks);
    if (rc != MX_OK) return rc;
    if (max_blocks < 1) return fail(MX_ERR_INVALID, "%s: max_blocks must be >= 1", what);
    if (flags & ~(uint32_t)MX_PA_BF16) return fail(MX_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
    if (!aligned(k_new, 16) || !aligned(v_new, 16) || new_sb % 8 || new_sh % 8 || new_st % 8)
        return fail(MX_ERR_ALIGNMENT, "%s: states must be 16-byte aligned rows", what);
    kv8::WriteParams p{k_new, v_new, new_sb, new_sh, new_st, T, block_tables, bt_sb, max_blocks, start_pos,
                       {data, codes, Hkv, num_blocks}, err, used, 0, 0, 0};
    // Pages that T tokens beginning at any slot can touch.
    p.pages_per_row = (int)(((int64_t)T + block_size - 2) / block_size + 1);
    if ((double)B * p.pages_per_row * Hkv * 2 > 1e11) return fail(MX_ERR_UNSUPPORTED, "%s: too many tokens", what);
    p.units = (int64_t)B * p.pages_per_row * Hkv * 2;
    const int64_t groups = kv8::groups_for(p.units);
    if (groups < 0) return fail(MX_ERR_UNSUPPORTED, "%s: more tokens than one launch holds", what);
    p.stream = (int64_t)B * T * Hkv * D * 4 > kv8::kStreamBytes;
    hipStream_t st = as_stream(stream);
#define CALL(DD, BB)                                                                                                   \
    if (flags & MX_PA_BF16)                                                                                            \
        hipLaunchKernelGGL((kv8::kv8_write_kernel<DD, BB, true>), dim3(groups), dim3(kv8::kWaves * 64), 0, st, p);      \
    else                                                                                                               \
        hipLaunchKernelGGL((kv8::kv8_write_kernel<DD, BB, false>), dim3(groups), dim3(kv8::kWaves * 64), 0, st, p)
    MX_KV8_DISPATCH(D, block_size, CALL)
#undef CALL
    return check_launch(what);
}

extern "C" int mx_kv8_gather(const uint8_t* data, const uint8_t* codes, const int32_t* block_tables, int64_t bt_sb,
                             int32_t max_blocks, const int32_t* seq_lens, int32_t B, int32_t S, int32_t Hkv, int32_t D,
                             int32_t block_size, int32_t num_blocks, uint16_t* k_out, uint16_t* v_out, int32_t* err,
                             uint32_t flags, void* stream) {
    const char* what = "mx_kv8_gather";
    if (B < 0 || S < 0) return fail(MX_ERR_INVALID, "%s: B and S must be >= 0", what);
    if (B == 0 || S == 0) return MX_OK;
    if (!block_tables || !k_out || !v_out) return fail(MX_ERR_NULL, "%s: null pointer", what);
    int rc = kv8::check_pages(what, data, codes, Hkv, D, block_size, num_blocks);
    if (rc != MX_OK) return rc;
    if (max_blocks < 1) return fail(MX_ERR_INVALID, "%s: max_blocks must be >= 1", what);
    if (flags & ~(uint32_t)MX_PA_BF16) return fail(MX_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return fail(MX_ERR_ALIGNMENT, "%s: outputs must be 16-byte aligned", what);
    kv8::GatherParams p{{const_cast<uint8_t*>(data), const_cast<uint8_t*>(codes), Hkv, num_blocks},
                        block_tables, bt_sb, max_blocks, seq_lens, S, (int)ceil_div(S, block_size), k_out, v_out, err, 0};
    if ((double)B * p.pages_per_row * Hkv * 2 > 1e11) return fail(MX_ERR_UNSUPPORTED, "%s: too many tokens", what);
    p.units = (int64_t)B * p.pages_per_row * Hkv * 2;
    const int64_t groups = kv8::groups_for(p.units);
    if (groups < 0) return fail(MX_ERR_UNSUPPORTED, "%s: more tokens than one launch holds", what);
    hipStream_t st = as_stream(stream);
#define CALL(DD, BB)                                                                                                   \
    if (flags & MX_PA_BF16)                                                                                            \
        hipLaunchKernelGGL((kv8::kv8_gather_kernel<DD, BB, true>), dim3(groups), dim3(kv8::kWaves * 64), 0, st, p);     \
    else                                                                                                               \
        hipLaunchKernelGGL((kv8::kv8_gather_kernel<DD, BB, false>), dim3(groups), dim3(kv8::kWaves * 64), 0, st, p)
    MX_KV8_DISPATCH(D, block_size, CALL)
#undef CALL
    return check_launch(what);
}

extern "C" int mx_kv8_rope_append(const uint16_t* qkv, int64_t qkv_stride, const float* partials, int32_t splits,
                                  const uint16_t* bias, int32_t B, int32_t Hq, int32_t Hkv, int32_t D,
                                  const float* rope, int32_t max_pos, const int32_t* positions, uint16_t* q_out,
                                  int64_t q_stride, const int32_t* block_tables, int64_t bt_sb, int32_t max_blocks,
                                  uint8_t* data, uint8_t* codes, int32_t block_size, int32_t num_blocks, int32_t* err,
                                  int32_t* lens_out, uint8_t* used, uint32_t flags, void* stream) {
    const char* what = "mx_kv8_rope_append";
    if (B < 0) return fail(MX_ERR_INVALID, "%s: B must be >= 0", what);
    if (B == 0) return MX_OK;
    if (!rope || !positions || !q_out || !block_tables) return fail(MX_ERR_NULL, "%s: null pointer", what);
    if (!qkv == !partials) return fail(MX_ERR_INVALID, "%s: give exactly one of qkv and partials", what);
    int rc = kv8::check_pages(what, data, codes, Hkv, D, block_size, num_blocks);
    if (rc != MX_OK) return rc;
    if (Hq < 1 || max_blocks < 1 || max_pos < 1)
        return fail(MX_ERR_INVALID, "%s: Hq, max_blocks and max_pos must be >= 1", what);
    if (partials && splits < 1) return fail(MX_ERR_INVALID, "%s: splits must be >= 1", what);
    if ((int64_t)Hq + 2 * (int64_t)Hkv > (1 << 20)) return fail(MX_ERR_UNSUPPORTED, "%s: too many heads", what);
    if (flags & ~(uint32_t)MX_PA_BF16) return fail(MX_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
    if (!aligned(rope, 8)) return fail(MX_ERR_ALIGNMENT, "%s: the rope table must be 8-byte aligned", what);
    const int64_t width = ((int64_t)Hq + 2 * Hkv) * D;
    kv8::TokenParams p{qkv, qkv_stride, partials, splits, (int64_t)B * width, bias, Hq,
                       reinterpret_cast<const float2*>(rope), max_pos, positions, q_out, q_stride, block_tables, bt_sb,
                       max_blocks, {data, codes, Hkv, num_blocks}, err, lens_out, used, (int64_t)B * (Hq + 2 * Hkv)};
    const int64_t groups = kv8::groups_for(p.units);
    if (groups < 0) return fail(MX_ERR_UNSUPPORTED, "%s: more rows than one launch holds", what);
    hipStream_t st = as_stream(stream);
#define CALL(DD, BB)                                                                                                   \
    if (flags & MX_PA_BF16)                                                                                            \
        hipLaunchKernelGGL((kv8::kv8_token_kernel<DD, BB, true>), dim3(groups), dim3(kv8::kWaves * 64), 0, st, p);      \
    else                                                                                                               \
        hipLaunchKernelGGL((kv8::kv8_token_kernel<DD, BB, false>), dim3(groups), dim3(kv8::kWaves * 64), 0, st, p)
    MX_KV8_DISPATCH(D, block_size, CALL)
#undef CALL
    return check_launch(what);
}
