// Verification of drafted tokens for gfx950: the path of a tree of drafted tokens that the target model's
// distributions accept, from given uniform numbers, and the token that follows it. (The reference verifies greedily, one
// token after the other: runtime/phase2/worker_server.py:1010-1075.)
//
// The walk stands at a node whose target distribution is r = softmax(logits / temperature) and tries the node's
// children in the order of their indices. A child with token x is taken where u q(x) < r(x), q the distribution that it was
// drafted from (a point at x where none is given). A child that is not taken leaves r = max(r - q, 0), scaled to a
// sum of 1. Where no child is taken the following token is drawn from r. That gives tokens of the target's own
// distribution whatever the draft was.
//
// All of it in 64 bits (sums that workgroups exchange keep 44 of their 52): an answer is a whole number, and a sum over 10^5 terms in
// 32 bits would put a border of the running sum on the other side of a uniform number in one draw of some hundred. A pass over
// a vocabulary takes 27 vector instructions per logit with everything, 18 of them for the exponential and its sum: 2 to 5 us of
// its 10 over a slice. The rest is the exchange and the decision behind it (32 rows of 16 nodes: the walk's waves wait in 72 % of
// their cycles), so only the nodes that a path visits are read.
//
// A row of the batch is walked by S workgroups together, each of which owns a slice of the vocabulary. A pass over a
// node's logits ends in one partial per slice (a sum and what it is relative to); every workgroup reads all partials
// of its row and then decides for itself, so all take the same way and nothing else is passed on. The first nodes of every tree
// (node 0 at least) are passed over by a launch of their own, which needs no exchange; the second launch walks.
//
// Partials are exchanged through 8-byte words that carry the number of the pass in their low bits, written and read
// past the L2s (relaxed atomics of agent scope), so that a word says by itself whether it is the one waited for: no
// fence, no counter, one round trip. Words of odd and even passes stand apart, since a workgroup is at most one pass
// ahead of another of its row, and so do those of passes over a node and of refusals, each numbered by itself: what a word
// held before is then always two passes older, and a number taken modulo 255 tells the two apart. Every wait ends: workgroups
// take their row and slice from a counter as they start, so all rows but the last one started have all their workgroups
// running, finish, and make room for what the last one lacks.
#include "common.h"

namespace mx {
namespace verify {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kVec = 8;                    // neighbouring logits per thread
constexpr int kBlock = kThreads * kVec;    // logits per step of a workgroup
constexpr int kWords = 5;                  // exchanged per slice: four of a pass over a node, one of a refusal
constexpr int kMaxSlices = 64;             // one lane of a wave each
constexpr int kMaxNodes = 1024;
// Workgroups, two a CU: 256 take 66 us for 32 rows of 16 nodes (128,256 logits), 1024 take 73, these 57; one row of 5 nodes
// (151,936) takes 19 us with 64 slices, 21 with 32.
constexpr int kFill = 512;
constexpr int kMaxVocab = 1 << 22;
constexpr int kMaxPolls = 1 << 23;         // seconds: a wait that long means a broken launch; the row then ends with -1
                                           // (MX_VERIFY_NO_WAIT: after one look, which shows that end)

// What a pass over a slice gives: sums of 2^((l - ref) c), c = log2(e) / temperature, of the logits and the draft's.
// Greedy rows: the largest logit in ref[0] and its first index in at. ref NaN: no distribution.
struct Part {
    double sum[2];
    float ref[2];
    int at, pad;
};

struct Params {
    const void* logits;
    int64_t l_sb, l_st;
    const void* draft;  // nullable
    int64_t d_sb, d_st;
    const int64_t* tokens;
    int64_t t_sb;
    const int32_t* parents;
    int64_t p_sb;
    const int32_t* counts;  // nullable: T
    const float* uniforms;
    int64_t u_sb;
    const float* temps;
    int64_t temp_sb;
    int B, T, V;
    int slices, len;  // of a row's vocabulary, logits per slice
    int first;        // nodes passed over by the first launch
    int max_polls;    // of a wait
    Part* parts;      // [B][first][slices]
    uint64_t* words;  // [B][2][slices][kWords]
    int* ticket;
    int64_t* tokens_out;
    int32_t* counts_out;
    int32_t* path_out;
};

// Elements of the logits: 0 fp16, 1 bf16, 2 fp32.
template <int KIND>
__device__ __forceinline__ float logit(const void* row, int64_t i) {
    if constexpr (KIND == 0) return (float)static_cast<const _Float16*>(row)[i];
    else if constexpr (KIND == 1) return __builtin_bit_cast(float, (uint32_t)static_cast<const uint16_t*>(row)[i] << 16);
    else return static_cast<const float*>(row)[i];
}
template <int KIND>
__device__ __forceinline__ const void* row_at(const void* base, int64_t off) {
    return static_cast<const char*>(base) + off * (KIND == 2 ? 4 : 2);
}
// A vector of a slice [lo, end) on the way: logits v + [0, 8). The load is unconditional, so that it can stand ahead of the
// work on the one before it: one that would pass the end is moved back, and take() drops what another thread has.
// (Rows begin at any element: the loads may be unaligned.)
template <int KIND, bool SMALL>
struct Ahead {
    typedef uint32_t raw __attribute__((ext_vector_type(KIND == 2 ? 8 : 4)));
    raw x;
    __device__ __forceinline__ static int at(int v, int end) {
        const int last = SMALL ? 0 : end - kVec;
        return v < last ? v : last;
    }
    __device__ __forceinline__ void load(const void* row, int v, int end) {
        constexpr int S = KIND == 2 ? 4 : 2;
        if constexpr (!SMALL) {
            __builtin_memcpy(&x, static_cast<const char*>(row) + (int64_t)at(v, end) * S, kVec * S);
        } else {  // a vocabulary of less than a vector
            x = raw{};
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (e < end) {
                    if constexpr (KIND == 2) x[e] = static_cast<const uint32_t*>(row)[e];
                    else x[e / 2] |= (uint32_t)static_cast<const uint16_t*>(row)[e] << 16 * (e % 2);
                }
        }
    }
    // The logits as numbers, -inf where the slice has ended or another thread has the logit; returns the first's index.
    __device__ __forceinline__ int take(int v, int end, float (&out)[kVec]) const {
        const int from = at(v, end);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const uint32_t word = x[KIND == 2 ? e : e / 2];  // (bit_cast of a vector's element itself takes the first one)
            if constexpr (KIND == 2) out[e] = __builtin_bit_cast(float, word);
            else if constexpr (KIND == 1) out[e] = __builtin_bit_cast(float, e % 2 ? word & 0xffff0000u : word << 16);
            else out[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(word >> 16 * (e % 2)));
        }
        if (__builtin_amdgcn_ballot_w64(v + kVec > end))
#pragma unroll
            for (int e = 0; e < kVec; ++e) out[e] = from + e >= v && from + e < end ? out[e] : -__builtin_huge_valf();
        return from;
    }
};

__device__ __forceinline__ int count_of(const Params& p, int b) {
    const int c = p.counts ? p.counts[b] : p.T;
    return c < 0 ? 0 : c < p.T ? c : p.T;
}
// log2(e) / temperature; 0 for a greedy row.
__device__ __forceinline__ double rate_of(const Params& p, int b) {
    const float t = p.temps[b * p.temp_sb];
    return t > 0.0f ? 1.4426950408889634074 / (double)t : 0.0;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// 2^t: t = n + f, |f| <= 1/2, the Taylor series of e^(f ln 2) to the 12th power (the next term is below 2e-16). t below -2000
// counts as -2000 (the result is 0 either way), and so does NaN, which a logit of -inf gives at an infinite temperature.
__device__ __forceinline__ double exp2_64(double t) {
    t = fmax(t, -2000.0);
    const double n = rint(t), f = t - n;
    double y = 2.56784359934882051e-11;          // ln(2)^12 / 12!
    y = __builtin_fma(y, f, 4.44553827187081178e-10);
    y = __builtin_fma(y, f, 7.05491162080112333e-9);
    y = __builtin_fma(y, f, 1.01780860092396999e-7);
    y = __builtin_fma(y, f, 1.32154867901443095e-6);
    y = __builtin_fma(y, f, 1.52527338040598403e-5);
    y = __builtin_fma(y, f, 1.54035303933816099e-4);
    y = __builtin_fma(y, f, 1.33335581464284434e-3);
    y = __builtin_fma(y, f, 9.61812910762847716e-3);
    y = __builtin_fma(y, f, 5.55041086648215800e-2);
    y = __builtin_fma(y, f, 2.40226506959100712e-1);
    y = __builtin_fma(y, f, 6.93147180559945309e-1);
    y = __builtin_fma(y, f, 1.0);
    return ldexp(y, (int)n);
}
__device__ __forceinline__ double weight(float l, float ref, double c) {
    return l == -__builtin_huge_valf() ? 0.0 : exp2_64(((double)l - (double)ref) * c);
}

// The same for whole slices, from a table of 2^(k / 128) in LDS: 2^t = 2^(n / 128) 2^(f / 128), |f| <= 1/2, four terms of the
// series (the next one is below 2e-15). All instructions cost alike here, fp64 or not: 18 a logit with the sum.
constexpr int kTable = 128;  // 2^7
struct Exp {
    const double* table;
    __device__ __forceinline__ static void fill(double* table) {
        if (threadIdx.x < kTable) table[threadIdx.x] = exp2_64((double)threadIdx.x / kTable);
    }
    // of (l - ref) c, given c * kTable
    __device__ __forceinline__ double operator()(float l, float ref, double ct) const {
        const double t = fmax(((double)l - (double)ref) * ct, -2000.0 * kTable);  // (l -inf: 2^-2000, which is 0)
        const double big = t + 6755399441055744.0;          // 1.5 * 2^52: its low bits are rint(t)
        const double f = t - (big - 6755399441055744.0);
        const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, big);
        double y = 3.583032305400251e-11;               // (ln(2) / 128)^4 / 4!
        y = __builtin_fma(y, f, 2.6466421444330967e-08);
        y = __builtin_fma(y, f, 1.4662262387640423e-05);
        y = __builtin_fma(y, f, 0.0054152123481245725);
        y = __builtin_fma(y, f, 1.0);
        return ldexp(y * table[n & (kTable - 1)], n >> 7);
    }
};

// A thread's running sum of 2^((l - ref) c). ref is the largest logit of the first it met; 64 bits hold the sum until
// a logit lies 2^900 above it.
struct Sum {
    double sum = 0.0;
    float ref = -__builtin_huge_valf();
    bool bad = false;  // a NaN (an infinity shows in ref, or below)
    __device__ __forceinline__ void add(const float (&x)[kVec], double c, const Exp& ex) {
        float top = fmaxf(x[0], x[1]);
#pragma unroll
        for (int i = 2; i < kVec; ++i) top = fmaxf(top, x[i]);
        bad |= top == __builtin_huge_valf();
#pragma unroll
        for (int i = 0; i < kVec; i += 2) bad |= __builtin_isunordered(x[i], x[i + 1]);
        if (top > ref && !(((double)top - (double)ref) * c <= 900.0)) {  // (ref -inf: the difference is inf, or NaN at rate 0)
            sum *= ref == -__builtin_huge_valf() ? 0.0 : exp2_64(((double)ref - (double)top) * c);
            ref = top;
        }
        const double ct = c * kTable;
        double part = 0.0;
#pragma unroll
        for (int i = 0; i < kVec; ++i) part += ex(x[i], ref, ct);
        sum += part;
    }
};

struct Shared {
    double table[kTable];
    double red[2][kWaves];
    float redf[2][kWaves];
    int redi[kWaves];
};

// A workgroup's Sums joined: every thread gets the result.
__device__ __forceinline__ void join(Shared& sh, int which, const Sum& s, double c, double& sum, float& ref) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float top = wave_max(s.ref);
    const bool bad = __builtin_amdgcn_ballot_w64(s.bad) != 0;
    __syncthreads();
    if (lane == 0) sh.redf[which][wave] = bad ? __builtin_nanf("") : top;
    __syncthreads();
    top = sh.redf[which][0];
    bool nan = top != top;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
        nan |= sh.redf[which][i] != sh.redf[which][i];
        top = fmaxf(top, sh.redf[which][i]);
    }
    double part = s.ref == -__builtin_huge_valf() ? 0.0 : s.sum * exp2_64(((double)s.ref - (double)top) * c);
    part = wave_sum(part);
    if (lane == 0) sh.red[which][wave] = part;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) sum += sh.red[which][i];
    ref = nan ? __builtin_nanf("") : top;
}

__device__ __forceinline__ double block_sum(Shared& sh, double v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[0][threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += sh.red[0][i];
    return s;
}

// A node's children that a draft without logits has drafted: their tokens stay out of the slices' sums, so that what
// remains once some are refused is a sum and never a difference.
struct Children {
    int n;
    const int* token;  // -1: outside the vocabulary
};

// One pass over slice s of a node: the softmax's sums, or a greedy row's largest logit.
template <int KIND, bool SMALL>
__device__ __forceinline__ Part pass(const Params& p, Shared& sh, const void* lrow, const void* drow, int s, double c,
                                     bool greedy, const Children& ch) {
    const int tid = threadIdx.x, lo = s * p.len, end = lo + p.len < p.V ? lo + p.len : p.V;
    Part out{};
    if (greedy) {
        float top = -__builtin_huge_valf();
        int at = 0x7fffffff;
        bool bad = false;
        Ahead<KIND, SMALL> a;
        a.load(lrow, lo + tid * kVec, end);
#pragma unroll 1
        for (int v = lo + tid * kVec; v < end; v += kBlock) {
            float x[kVec];
            const int from = a.take(v, end, x);
            a.load(lrow, v + kBlock, end);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                bad |= x[i] != x[i];
                if (x[i] > top) top = x[i], at = from + i;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const float t = __shfl_xor(top, o);
            const int a = __shfl_xor(at, o);
            if (t > top || (t == top && a < at)) top = t, at = a;
        }
        bad = __builtin_amdgcn_ballot_w64(bad) != 0;
        __syncthreads();
        if ((tid & 63) == 0) sh.redf[0][tid >> 6] = bad ? __builtin_nanf("") : top, sh.redi[tid >> 6] = at;
        __syncthreads();
        top = sh.redf[0][0], at = sh.redi[0];
        bad = top != top;
        for (int i = 1; i < kWaves; ++i) {
            const float t = sh.redf[0][i];
            bad |= t != t;
            if (t > top || (t == top && sh.redi[i] < at)) top = t, at = sh.redi[i];
        }
        out.ref[0] = bad ? __builtin_nanf("") : top;
        out.at = at;
        return out;
    }
    const Exp ex{sh.table};
    Sum a, d;
    Ahead<KIND, SMALL> al, ad;
    al.load(lrow, lo + tid * kVec, end);
    if (drow) ad.load(drow, lo + tid * kVec, end);
#pragma unroll 1
    for (int v = lo + tid * kVec; v < end; v += kBlock) {
        float x[kVec];
        const int from = al.take(v, end, x);
        al.load(lrow, v + kBlock, end);
        for (int j = 0; j < ch.n; ++j) {
            const int t = ch.token[j] - from;
            if ((unsigned)t < (unsigned)kVec)
#pragma unroll
                for (int i = 0; i < kVec; ++i) x[i] = i == t ? -__builtin_huge_valf() : x[i];
        }
        a.add(x, c, ex);
        if (drow) {
            ad.take(v, end, x);
            ad.load(drow, v + kBlock, end);
            d.add(x, c, ex);
        }
    }
    join(sh, 0, a, c, out.sum[0], out.ref[0]);
    if (drow) join(sh, 1, d, c, out.sum[1], out.ref[1]);
    return out;
}

// The children of `node` in order, their tokens (-1 outside the vocabulary): by one wave, from the tree in LDS or memory.
template <typename P, typename T>
__device__ __forceinline__ int children_of(P parent, T token, int node, int count, int* index, int* tok) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int i0 = node + 1; i0 < count; i0 += 64) {
        const int i = i0 + lane;
        const bool mine = i < count && parent(i) == node;
        const uint64_t who = __builtin_amdgcn_ballot_w64(mine);
        if (mine) {
            const int at = n + __builtin_popcountll(who & ((1ull << lane) - 1));
            if (index) index[at] = i;
            tok[at] = token(i);
        }
        n += __builtin_popcountll(who);
    }
    return n;
}
__device__ __forceinline__ int token_in(int64_t x, int V) { return x >= 0 && x < V ? (int)x : -1; }

// The nodes below `first` of every row, a workgroup per slice; clears what the walk's exchange begins with.
template <int KIND, bool SMALL>
__global__ __launch_bounds__(kThreads) void first_kernel(Params p) {
    __shared__ Shared sh;
    __shared__ int tok[kMaxNodes];
    __shared__ int nch;
    const int s = blockIdx.x % p.slices, rest = blockIdx.x / p.slices;
    const int node = rest % p.first, b = rest / p.first;
    if (node == 0 && threadIdx.x < 2 * kWords)
        p.words[(((int64_t)b * 2 + threadIdx.x / kWords) * p.slices + s) * kWords + threadIdx.x % kWords] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
    Exp::fill(sh.table);
    __syncthreads();
    const int count = count_of(p, b);
    if (node >= count) return;
    const double c = rate_of(p, b);
    const bool greedy = !(p.temps[b * p.temp_sb] > 0.0f);
    if (!p.draft && !greedy) {
        if (threadIdx.x < 64) {
            const int32_t* parents = p.parents + b * p.p_sb;
            const int64_t* tokens = p.tokens + b * p.t_sb;
            const int n = children_of([&](int i) { return parents[i]; }, [&](int i) { return token_in(tokens[i], p.V); },
                                      node, count, nullptr, tok);
            if (threadIdx.x == 0) nch = n;
        }
        __syncthreads();
    }
    const Children ch{!p.draft && !greedy ? nch : 0, tok};
    const Part out = pass<KIND, SMALL>(p, sh, row_at<KIND>(p.logits, b * p.l_sb + node * p.l_st),
                                p.draft && !greedy ? row_at<KIND>(p.draft, b * p.d_sb + node * p.d_st) : nullptr, s, c,
                                greedy, ch);
    if (threadIdx.x == 0) p.parts[((int64_t)b * p.first + node) * p.slices + s] = out;
}

template <int KIND, bool SMALL>
__global__ __launch_bounds__(kThreads) void walk_kernel(Params p, int per_row) {
    __shared__ Shared sh;
    __shared__ int parent[kMaxNodes], token[kMaxNodes];
    __shared__ float uniform[kMaxNodes];
    __shared__ int cidx[kMaxNodes], ctok[kMaxNodes], cfirst[kMaxNodes];  // children; the first with the same token
    __shared__ double cw[kMaxNodes];     // without draft logits: weight, 0 once refused; with: scales of the refusals
    __shared__ double part[kMaxSlices];  // r's weight in each slice
    __shared__ double whole[2], per_whole[2];
    __shared__ float refs[2];
    __shared__ int sbest, snch, sid, stail[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float inf = __builtin_huge_valf();
    if (tid == 0) sid = per_row > 1 ? atomicAdd(p.ticket, 1) : (int)blockIdx.x;
    Exp::fill(sh.table);
    __syncthreads();
    const int b = sid / per_row, s = sid % per_row;
    const int count = count_of(p, b);
    int64_t* tout = p.tokens_out + (int64_t)b * p.T;
    int32_t* pout = p.path_out + (int64_t)b * p.T;
    const float temp = p.temps[b * p.temp_sb];
    const bool greedy = !(temp > 0.0f);
    const double c = rate_of(p, b);
    const bool drafted = p.draft && !greedy;
    for (int i = tid; i < p.T; i += kThreads) {  // (not `count`: no need to wait for it)
        const int up = p.parents[b * p.p_sb + i];
        parent[i] = up < i ? up : -1;
        token[i] = token_in(p.tokens[b * p.t_sb + i], p.V);
        uniform[i] = p.uniforms[b * p.u_sb + i];
    }
    __syncthreads();

    int node_passes = 0, refusal_passes = 0;  // cooperative passes so far
    // Every slice's words of pass number `pass` of its kind, n of them from `first` on; a lane of the first wave each.
    auto exchange = [&](int pass, int first, const uint64_t (&mine)[4], int n, uint64_t (&all)[4]) -> bool {
        const uint64_t tag = pass % 255 + 1;
        uint64_t* base = p.words + ((int64_t)b * 2 + (pass & 1)) * p.slices * kWords + first;
        if (tid == 0)
            for (int i = 0; i < n; ++i)
                __hip_atomic_store(base + s * kWords + i, (mine[i] & ~0xffull) | tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        bool ok = true;
        if (wave == 0) {
            const int from = lane < p.slices ? lane : 0;
            for (int polls = 0;; ++polls) {
                bool there = true;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < n) {
                        all[i] = __hip_atomic_load(base + from * kWords + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        there &= (all[i] & 0xff) == tag;
                    }
                if (__builtin_amdgcn_ballot_w64(!there) == 0) break;
                if (polls >= p.max_polls) {
                    ok = false;
                    break;
                }
                __builtin_amdgcn_s_sleep(1);
            }
        }
        return ok;
    };
    auto word_of = [](double x) { return __builtin_bit_cast(uint64_t, x); };
    // (a sum loses its low 8 bits to the tag: 2^-44 of it, and all workgroups use the same one)
    auto sum_of = [](uint64_t w) { return __builtin_bit_cast(double, w & ~0xffull); };
    auto ref_word = [](float x) { return (uint64_t)__builtin_bit_cast(uint32_t, x) << 32; };
    auto ref_of = [](uint64_t w) { return __builtin_bit_cast(float, (uint32_t)(w >> 32)); };

    int node = 0, n = 0;
    int refused = 0;  // with draft logits: refusals that r carries
    bool have = false;
    const void *lrow = nullptr, *drow = nullptr;

    // Stand at `node`: its distribution's parts and its children.
    auto enter = [&]() {
        lrow = row_at<KIND>(p.logits, b * p.l_sb + node * p.l_st);
        drow = drafted ? row_at<KIND>(p.draft, b * p.d_sb + node * p.d_st) : nullptr;
        refused = 0;
        __syncthreads();
        if (wave == 0) {
            const int k = children_of([&](int i) { return parent[i]; }, [&](int i) { return token[i]; }, node, count, cidx, ctok);
            if (lane == 0) snch = k;
        }
        __syncthreads();
        const int k = snch;
        float cl = -inf;  // logits of this thread's child, loaded ahead of the pass
        if (!drafted && !greedy && tid < k && ctok[tid] >= 0) cl = logit<KIND>(lrow, ctok[tid]);
        Part mine{};
        bool ok = true;
        if (node < p.first) {
            if (wave == 0 && lane < p.slices) mine = p.parts[((int64_t)b * p.first + node) * p.slices + lane];
        } else {
            const Children ch{!drafted && !greedy ? k : 0, ctok};
            mine = pass<KIND, SMALL>(p, sh, lrow, drow, s, c, greedy, ch);
            uint64_t w[4] = {greedy ? (uint64_t)(uint32_t)mine.at << 8 : word_of(mine.sum[0]), ref_word(mine.ref[0]),
                             word_of(mine.sum[1]), ref_word(mine.ref[1])}, all[4];
            ok = exchange(++node_passes, 0, w, drafted ? 4 : 2, all);
            if (wave == 0) {
                mine.at = greedy ? (int)(all[0] >> 8) : 0;
                mine.sum[0] = sum_of(all[0]);
                mine.ref[0] = ref_of(all[1]);
                if (drafted) mine.sum[1] = sum_of(all[2]), mine.ref[1] = ref_of(all[3]);
            }
        }
        // Children's weights count with the slices' for the largest logit. (The first 256 are at hand.)
        // (One that is NaN counts as infinite: either way there is no distribution.)
        float ctop = cl == cl ? cl : inf;
        if (!drafted && !greedy)
            for (int j = tid + kThreads; j < k; j += kThreads)
                if (ctok[j] >= 0) {
                    const float l = logit<KIND>(lrow, ctok[j]);
                    ctop = fmaxf(ctop, l == l ? l : inf);
                }
        ctop = wave_max(ctop);
        __syncthreads();
        if (lane == 0) sh.redf[1][wave] = ctop;
        __syncthreads();
        if (wave == 0) {
            const bool live = lane < p.slices;
            for (int i = 0; i < kWaves; ++i) ctop = fmaxf(ctop, sh.redf[1][i]);
            for (int which = 0; which < (drafted ? 2 : 1); ++which) {
                float ref = live ? mine.ref[which] : -inf;
                bool bad = __builtin_amdgcn_ballot_w64(ref != ref || !ok) != 0;
                float top = wave_max(ref);
                if (which == 0) top = fmaxf(top, ctop);
                bad |= top == -inf || (!greedy && top == inf);
                int at = live && ref == top ? mine.at : 0x7fffffff;
                if (greedy) {
#pragma unroll
                    for (int o = 32; o > 0; o >>= 1) {
                        const int t = __shfl_xor(at, o);
                        at = t < at ? t : at;
                    }
                }
                double z = 0.0;
                if (live && !bad && !greedy && ref != -inf) z = mine.sum[which] * exp2_64(((double)ref - (double)top) * c);
                if (which == 0 && live) part[lane] = z;
                z = wave_sum(z);
                if (lane == 0) {
                    refs[which] = bad ? __builtin_nanf("") : top;
                    whole[which] = z;
                    per_whole[which] = 1.0 / z;
                    if (which == 0) sbest = at;
                }
            }
        }
        __syncthreads();
        have = refs[0] == refs[0];
        if (!drafted && !greedy && have) {
            for (int j = tid; j < k; j += kThreads) {
                const int x = ctok[j];
                int first = j;
                for (int i = 0; i < j; ++i)
                    if (ctok[i] == x) {
                        first = i;
                        break;
                    }
                cfirst[j] = first;
                cw[j] = x < 0 || first != j ? 0.0 : weight(j == tid ? cl : logit<KIND>(lrow, x), refs[0], c);
            }
            __syncthreads();
        }
    };
    // r of token v. Without draft logits up to a factor, and so with them until a child is refused.
    const Exp ex{sh.table};
    auto rest = [&](auto& l, auto& d, auto& r) {
        constexpr int N = sizeof(r) / sizeof(r[0]);
#pragma unroll
        for (int e = 0; e < N; ++e) r[e] = ex(l[e], refs[0], c * kTable);
        if (refused == 0) return;
        double q[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            r[e] *= per_whole[0];
            q[e] = ex(d[e], refs[1], c * kTable) * per_whole[1];
        }
#pragma unroll 1
        for (int i = 0; i < refused; ++i) {
            const double f = cw[i];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                r[e] -= q[e];
                r[e] = (r[e] > 0.0 ? r[e] : 0.0) * f;
            }
        }
    };
    // Children's weights (without draft logits): all that r still has, `but` one of them.
    auto child_mass = [&](int k, int but) {
        double m = 0.0;
        for (int j = lane; j < k; j += 64) m += j == but ? 0.0 : cw[j];
        return wave_sum(m);
    };

    if (count > 0) {
        if (s == 0 && tid == 0) pout[0] = 0;
        n = 1;
        for (bool moved = true; moved;) {
            moved = false;
            enter();
            const int k = snch;
            if (!have) break;
            double all = drafted || greedy ? 0.0 : whole[0] + child_mass(k, -1);
            const bool qhave = drafted && refs[1] == refs[1];
            for (int j = 0; j < k; ++j) {
                const int x = ctok[j], i = cidx[j];
                if (x < 0 || (drafted && !qhave)) continue;
                bool take;
                if (greedy) take = x == sbest;
                else if (!drafted) take = (double)uniform[i] * all < cw[cfirst[j]];
                else {
                    const float l[1] = {logit<KIND>(lrow, x)}, d[1] = {logit<KIND>(drow, x)};
                    double r[1];
                    rest(l, d, r);
                    if (!refused) r[0] *= per_whole[0];
                    take = (double)uniform[i] * (ex(d[0], refs[1], c * kTable) * per_whole[1]) < r[0];
                }
                if (take) {
                    if (s == 0 && tid == 0) {
                        pout[n] = i;
                        tout[n - 1] = x;
                    }
                    ++n;
                    node = i;
                    moved = true;
                    break;
                }
                if (greedy) continue;
                if (!drafted) {
                    const int f = cfirst[j];
                    const double left = whole[0] + child_mass(k, f);
                    if (cw[f] > 0.0 && left > 0.0) {  // (where nothing remains r stays)
                        all = left;
                        __syncthreads();
                        if (tid == 0) cw[f] = 0.0;
                        __syncthreads();
                    }
                } else {
                    // A pass for the mass that remains.
                    __syncthreads();
                    if (tid == 0) cw[refused] = 1.0;
                    ++refused;
                    __syncthreads();
                    const int lo = s * p.len, end = lo + p.len < p.V ? lo + p.len : p.V;
                    double m = 0.0;
                    Ahead<KIND, SMALL> al, ad;
                    al.load(lrow, lo + tid * kVec, end);
                    ad.load(drow, lo + tid * kVec, end);
#pragma unroll 1
                    for (int v = lo + tid * kVec; v < end; v += kBlock) {
                        float xl[kVec], xd[kVec];
                        double r[kVec];
                        al.take(v, end, xl);
                        ad.take(v, end, xd);
                        al.load(lrow, v + kBlock, end);
                        ad.load(drow, v + kBlock, end);
                        rest(xl, xd, r);
#pragma unroll
                        for (int e = 0; e < kVec; ++e) m += r[e];
                    }
                    const uint64_t w[4] = {word_of(block_sum(sh, m)), 0, 0, 0};
                    uint64_t got[4];
                    const bool ok = exchange(++refusal_passes, 4, w, 1, got);
                    if (wave == 0) {
                        const double z = ok && lane < p.slices ? sum_of(got[0]) : 0.0;
                        const double sum = wave_sum(z);
                        if (sum > 0.0 && lane < p.slices) part[lane] = z * (1.0 / sum);  // of r, whose sum is 1
                        if (lane == 0) cw[refused - 1] = !ok ? __builtin_nan("") : sum > 0.0 ? 1.0 / sum : 0.0;
                    }
                    __syncthreads();
                    const double f = cw[refused - 1];
                    if (f != f) {  // the wait gave up
                        have = false;
                        break;
                    }
                    if (!(f > 0.0)) --refused;  // nothing remains: r stays
                }
            }
        }
        if (s != 0) return;
        int64_t next = -1;
        if (have && greedy) next = sbest;
        else if (have) {
            const int k = snch;
            double all;
            int hit_at, tail_at;
            __syncthreads();
            if (!drafted) {  // the children that were not refused, in their slices
                for (int j = 0; j < k; ++j)
                    if (tid == 0 && ctok[j] >= 0) part[ctok[j] / p.len] += cw[j];
                __syncthreads();
            }
            // Every wave finds the slice, a lane for each: the first whose running sum exceeds the goal.
            const double mine_part = lane < p.slices ? part[lane] : 0.0;
            double upto = mine_part;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double t = __shfl_up(upto, o);
                if (lane >= o) upto += t;
            }
            all = __shfl(upto, 63);
            const double goal = (double)uniform[0] * all;
            const uint64_t above = __builtin_amdgcn_ballot_w64(upto > goal && mine_part > 0.0);
            const uint64_t some = __builtin_amdgcn_ballot_w64(mine_part > 0.0);
            const bool beyond = above == 0;  // a uniform number that is not below 1: the last token there is
            const int slice = beyond ? (some ? 63 - __builtin_clzll(some) : 0) : __builtin_ctzll(above);
            double before = __shfl(upto - mine_part, slice);
            hit_at = tail_at = -1;
            const int lo = slice * p.len, end = lo + p.len < p.V ? lo + p.len : p.V;
            Ahead<KIND, SMALL> al, ad;
            al.load(lrow, lo + tid * kVec, end);
            if (refused) ad.load(drow, lo + tid * kVec, end);
#pragma unroll 1
            for (int v0 = lo; v0 < end; v0 += kBlock) {
                float xl[kVec], xd[kVec] = {};
                const int v = al.take(v0 + tid * kVec, end, xl);
                if (refused) ad.take(v0 + tid * kVec, end, xd);
                if (v0 + kBlock < end) {
                    al.load(lrow, v0 + kBlock + tid * kVec, end);
                    if (refused) ad.load(drow, v0 + kBlock + tid * kVec, end);
                }
                double w[kVec], mine = 0.0;
                rest(xl, xd, w);
                if (!drafted)
                    for (int j = 0; j < k; ++j) {
                        const int t = ctok[j] - v;
                        if ((unsigned)t < (unsigned)kVec)
#pragma unroll
                            for (int e = 0; e < kVec; ++e) w[e] = e == t ? cw[cfirst[j]] : w[e];
                    }
#pragma unroll
                for (int e = 0; e < kVec; ++e) mine += w[e];
                double run = mine;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const double t = __shfl_up(run, o);
                    if (lane >= o) run += t;
                }
                __syncthreads();
                if (lane == 63) sh.red[0][wave] = run;
                __syncthreads();
                double block = 0.0;
                for (int i = 0; i < kWaves; ++i) {
                    if (i < wave) run += sh.red[0][i];
                    block += sh.red[0][i];
                }
                run = before + run - mine;
                int mhit = -1, mtail = -1;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    run += w[e];
                    if (w[e] > 0.0) {
                        mtail = v + e;
                        if (!beyond && run > goal && mhit < 0) mhit = v + e;
                    }
                }
                // Threads are in the tokens' order: the first one with a hit, the last one with any weight.
                const uint64_t hits = __builtin_amdgcn_ballot_w64(mhit >= 0), tails = __builtin_amdgcn_ballot_w64(mtail >= 0);
                const int whit = hits ? __builtin_amdgcn_readlane(mhit, __builtin_ctzll(hits)) : -1;
                const int wtail = tails ? __builtin_amdgcn_readlane(mtail, 63 - __builtin_clzll(tails)) : -1;
                if (lane == 0) sh.redi[wave] = whit, stail[wave] = wtail;
                before += block;
                __syncthreads();
#pragma unroll
                for (int i = kWaves - 1; i >= 0; --i) {
                    if (sh.redi[i] >= 0) hit_at = sh.redi[i];
                }
#pragma unroll
                for (int i = 0; i < kWaves; ++i)
                    if (stail[i] >= 0) tail_at = stail[i];
                if (hit_at >= 0) break;
            }
            next = hit_at >= 0 ? hit_at : tail_at;
        }
        if (tid == 0) tout[n - 1] = next;
    }
    if (s != 0) return;
    for (int i = n + tid; i < p.T; i += kThreads) {
        tout[i] = -1;
        pout[i] = -1;
    }
    if (tid == 0) p.counts_out[b] = n;
}

struct Plan {
    int slices, len, first;
    size_t words_at, ticket_at, bytes;  // in the workspace
};

// Slices: enough workgroups to fill the chip, each with at least a step of logits. The first launch takes node 0, and as many more
// as cost it about what the walk's passes over those that its path visits would (a pass and its exchange 10 us, twice that with
// draft logits): 4 million logits, 12 with draft logits. Both launches together: one row of 5 nodes 27 us with node 0 alone, 19
// with all; 32 rows of 16 nodes 57, 55, 59, 58, 65 us with 4, 8, 12, 16, 24 million, 8 rows of 16 nodes 41, 46, 49, -, 52; 8
// chains of 7 with draft logits 60 us with node 0 alone, 58, 50, 41, 41, 41 with those numbers, 4 chains of 24 87, 73, 59, -, 77.
static Plan plan_of(int64_t B, int64_t T, int64_t V, bool draft) {
    Plan p{};
    int64_t s = kFill / B;
    const int64_t most = ceil_div(V, kBlock);
    s = s < 1 ? 1 : s > kMaxSlices ? kMaxSlices : s;
    s = s < most ? s : most;
    p.len = (int)(ceil_div(ceil_div(V, s), kVec) * kVec);
    p.slices = (int)ceil_div(V, p.len);
    const int64_t f = draft ? (12 << 20) / (B * V * 2) : (4 << 20) / (B * V);
    p.first = (int)(f < 1 ? 1 : f < T ? f : T);
    p.words_at = (size_t)B * p.first * p.slices * sizeof(Part);
    p.ticket_at = p.words_at + (size_t)B * 2 * p.slices * kWords * sizeof(uint64_t);
    p.bytes = p.ticket_at + 16;
    return p;
}

template <int KIND, bool SMALL>
static void launch(const Params& p, hipStream_t st) {
    hipLaunchKernelGGL((first_kernel<KIND, SMALL>), dim3((unsigned)(p.B * p.first * p.slices)), dim3(kThreads), 0, st, p);
    // Without an exchange to come one workgroup a row walks.
    const int per_row = p.draft || p.first < p.T ? p.slices : 1;
    hipLaunchKernelGGL((walk_kernel<KIND, SMALL>), dim3((unsigned)(p.B * per_row)), dim3(kThreads), 0, st, p, per_row);
}
template <int KIND>
static void launch_any(const Params& p, hipStream_t st) {
    if (p.V < kVec) launch<KIND, true>(p, st);
    else launch<KIND, false>(p, st);
}

}  // namespace verify
}  // namespace mx

using namespace mx;

extern "C" size_t mx_verify_draft_workspace_bytes(int32_t B, int32_t T, int32_t V, int32_t draft) {
    if (B <= 0 || T <= 0 || V <= 0) return 0;
    return verify::plan_of(B, T, V, draft != 0).bytes;
}

extern "C" int mx_verify_draft(const void* logits, int64_t l_sb, int64_t l_st, const void* draft_logits, int64_t d_sb,
                               int64_t d_st, const int64_t* tokens, int64_t t_sb, const int32_t* parents, int64_t p_sb,
                               const int32_t* counts, const float* uniforms, int64_t u_sb, const float* temperatures,
                               int64_t temp_sb, int32_t B, int32_t T, int32_t V, int64_t* tokens_out,
                               int32_t* counts_out, int32_t* path_out, void* workspace, size_t workspace_bytes,
                               uint32_t flags, void* stream) {
    clear_error();
    const char* what = "mx_verify_draft";
    if (B < 0 || T < 0 || V < 1) return fail(MX_ERR_INVALID, "%s: need B >= 0, T >= 0 and V >= 1", what);
    if (B == 0 || T == 0) return MX_OK;
    if (!logits || !tokens || !parents || !uniforms || !temperatures || !tokens_out || !counts_out || !path_out)
        return fail(MX_ERR_NULL, "%s: null pointer", what);
    if (flags & ~(uint32_t)(MX_PA_BF16 | MX_LOGITS_FP32 | MX_VERIFY_NO_WAIT) ||
        (flags & (MX_PA_BF16 | MX_LOGITS_FP32)) == (MX_PA_BF16 | MX_LOGITS_FP32))
        return fail(MX_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
    if (l_sb < 0 || l_st < 0 || d_sb < 0 || d_st < 0 || t_sb < 0 || p_sb < 0 || u_sb < 0 || temp_sb < 0)
        return fail(MX_ERR_INVALID, "%s: strides must be >= 0", what);
    if (T > verify::kMaxNodes) return fail(MX_ERR_UNSUPPORTED, "%s: more than %d nodes", what, verify::kMaxNodes);
    if (V > verify::kMaxVocab) return fail(MX_ERR_UNSUPPORTED, "%s: more than %d logits", what, verify::kMaxVocab);
    if (B > (1 << 20)) return fail(MX_ERR_UNSUPPORTED, "%s: more than %d rows", what, 1 << 20);
    const size_t need = mx_verify_draft_workspace_bytes(B, T, V, draft_logits != nullptr);
    if (!workspace || workspace_bytes < need)
        return fail(MX_ERR_WORKSPACE, "%s: workspace needs %zu bytes, got %zu", what, need, workspace ? workspace_bytes : 0);
    if (!aligned(workspace, 16)) return fail(MX_ERR_ALIGNMENT, "%s: workspace alignment", what);
    verify::Params p{};
    p.logits = logits, p.l_sb = l_sb, p.l_st = l_st;
    p.draft = draft_logits, p.d_sb = d_sb, p.d_st = d_st;
    p.tokens = tokens, p.t_sb = t_sb, p.parents = parents, p.p_sb = p_sb, p.counts = counts;
    p.uniforms = uniforms, p.u_sb = u_sb, p.temps = temperatures, p.temp_sb = temp_sb;
    p.B = B, p.T = T, p.V = V;
    const verify::Plan pl = verify::plan_of(B, T, V, draft_logits != nullptr);
    p.slices = pl.slices, p.len = pl.len, p.first = pl.first;
    p.max_polls = flags & MX_VERIFY_NO_WAIT ? 0 : verify::kMaxPolls;
    char* ws = static_cast<char*>(workspace);
    p.parts = reinterpret_cast<verify::Part*>(ws);
    p.words = reinterpret_cast<uint64_t*>(ws + pl.words_at);
    p.ticket = reinterpret_cast<int*>(ws + pl.ticket_at);
    p.tokens_out = tokens_out, p.counts_out = counts_out, p.path_out = path_out;
    hipStream_t st = as_stream(stream);
    if (flags & MX_LOGITS_FP32) verify::launch_any<2>(p, st);
    else if (flags & MX_PA_BF16) verify::launch_any<1>(p, st);
    else verify::launch_any<0>(p, st);
    return check_launch(what);
}
