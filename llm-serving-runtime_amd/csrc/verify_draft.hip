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
// All of it in 64 bits: an answer is a whole number, and a sum over 10^5 terms in 32 bits would put a border of the
// running sum on the other side of a uniform number in one draw of some hundred.
#include "common.h"

namespace mx {
namespace verify {

constexpr int kThreads = 256;
constexpr int kPer = 16;                    // logits of a chunk per thread
constexpr int kChunk = kThreads * kPer;     // logits per chunk
constexpr int kMaxChunks = 1024;
constexpr int kMaxNodes = 1024;

struct Stat {
    double sum;  // of exp((l - top) / temperature)
    float top;   // largest logit; NaN: the chunk holds a NaN
    int at;      // its first index
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
    int B, T, V, chunks;
    Stat* stats;  // [2 or 1][B][T][chunks]
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

__device__ __forceinline__ int count_of(const Params& p, int b) {
    const int c = p.counts ? p.counts[b] : p.T;
    return c < 0 ? 0 : c < p.T ? c : p.T;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// exp((l - top) / temperature), 0 at -inf.
__device__ __forceinline__ double weight(float l, float top, double inv) {
    return l == -__builtin_huge_valf() ? 0.0 : exp(((double)l - (double)top) * inv);
}

// One workgroup per chunk of a node's logits.
template <int KIND>
__global__ __launch_bounds__(kThreads) void stats_kernel(Params p) {
    __shared__ float stop[kThreads / 64];
    __shared__ int sat[kThreads / 64];
    __shared__ double ssum[kThreads / 64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int chunk = blockIdx.x % p.chunks;
    const int64_t rowid = blockIdx.x / p.chunks;
    const bool is_draft = rowid >= (int64_t)p.B * p.T;
    const int64_t at = rowid - (is_draft ? (int64_t)p.B * p.T : 0);
    const int b = (int)(at / p.T), n = (int)(at - (int64_t)b * p.T);
    if (n >= count_of(p, b)) return;
    const void* row = is_draft ? row_at<KIND>(p.draft, b * p.d_sb + n * p.d_st) : row_at<KIND>(p.logits, b * p.l_sb + n * p.l_st);
    const float temp = p.temps[b * p.temp_sb];
    float x[kPer];
    float top = -__builtin_huge_valf();
    int first = 0x7fffffff;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int v = chunk * kChunk + i * kThreads + tid;
        x[i] = v < p.V ? logit<KIND>(row, v) : -__builtin_huge_valf();
        nan |= x[i] != x[i];
        if (x[i] > top) top = x[i], first = v;
    }
    for (int o = 32; o > 0; o >>= 1) {
        const float t = __shfl_xor(top, o);
        const int f = __shfl_xor(first, o);
        if (t > top || (t == top && f < first)) top = t, first = f;
    }
    nan = __builtin_amdgcn_ballot_w64(nan) != 0;
    if (lane == 0) stop[wave] = nan ? __builtin_nanf("") : top, sat[wave] = first;
    __syncthreads();
    top = stop[0], first = sat[0];
    for (int i = 1; i < kThreads / 64; ++i) {
        const float t = stop[i];
        if (t != t) top = t;
        else if (t > top || (t == top && sat[i] < first)) top = t, first = sat[i];
    }
    double sum = 0.0;
    if (temp > 0.0f && top == top && __builtin_fabsf(top) != __builtin_huge_valf()) {
        const double inv = 1.0 / (double)temp;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += weight(x[i], top, inv);
    }
    sum = wave_sum(sum);
    if (lane == 0) ssum[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
        for (int i = 0; i < kThreads / 64; ++i) sum += ssum[i];
        p.stats[rowid * p.chunks + chunk] = Stat{sum, top, first};
    }
}

// One workgroup per row of the batch.
template <int KIND>
__global__ __launch_bounds__(kThreads) void walk_kernel(Params p) {
    __shared__ double part[kMaxChunks];   // r's weight in each chunk
    __shared__ double scale[kMaxNodes];   // with draft logits: 1 / the mass that each child not taken left
    __shared__ int out_of[kMaxNodes];     // without: tokens taken out of r
    __shared__ double red[kThreads / 64];
    __shared__ float ftop[2];
    __shared__ int fat[2];
    __shared__ double fz[2];
    __shared__ int found;
    const int b = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int count = count_of(p, b);
    const int32_t* parents = p.parents + b * p.p_sb;
    const int64_t* tokens = p.tokens + b * p.t_sb;
    const float* uniforms = p.uniforms + b * p.u_sb;
    const float temp = p.temps[b * p.temp_sb];
    const bool greedy = !(temp > 0.0f);
    const double inv = greedy ? 0.0 : 1.0 / (double)temp;
    int64_t* tout = p.tokens_out + (int64_t)b * p.T;
    int32_t* pout = p.path_out + (int64_t)b * p.T;
    const float inf = __builtin_huge_valf();

    auto block_sum = [&](double v) {
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) red[wave] = v;
        __syncthreads();
        double s = 0.0;
        for (int i = 0; i < kThreads / 64; ++i) s += red[i];
        return s;
    };
    // The whole of a node's distribution from its chunks: largest logit, its first index, sum of weights (0: no distribution).
    auto gather = [&](int which, int n) {
        const Stat* st = p.stats + (((int64_t)which * p.B + b) * p.T + n) * p.chunks;
        __syncthreads();
        if (wave == 0) {
            float top = -inf;
            int first = 0x7fffffff;
            bool nan = false;
            for (int c = lane; c < p.chunks; c += 64) {
                const Stat s = st[c];
                nan |= s.top != s.top;
                if (s.top > top || (s.top == top && s.at < first)) top = s.top, first = s.at;
            }
            for (int o = 32; o > 0; o >>= 1) {
                const float t = __shfl_xor(top, o);
                const int f = __shfl_xor(first, o);
                if (t > top || (t == top && f < first)) top = t, first = f;
            }
            nan = __builtin_amdgcn_ballot_w64(nan) != 0 || top == -inf || (!greedy && top == inf);
            double z = 0.0;
            for (int c = lane; c < p.chunks; c += 64) {
                const Stat s = st[c];
                const double w = nan || greedy || s.top == -inf ? 0.0 : s.sum * exp(((double)s.top - (double)top) * inv);
                if (which == 0) part[c] = w;
                z += w;
            }
            z = wave_sum(z);
            if (lane == 0) ftop[which] = top, fat[which] = first, fz[which] = nan ? 0.0 : greedy ? 1.0 : z;
        }
        __syncthreads();
    };

    int node = 0, n = 0;
    if (count > 0) {
        if (tid == 0) pout[0] = 0;
        n = 1;
        int rejected = 0;
        double mass = 0.0;  // sum of part
        const void *lrow = nullptr, *drow = nullptr;
        auto enter = [&]() {
            gather(0, node);
            lrow = row_at<KIND>(p.logits, b * p.l_sb + node * p.l_st);
            if (p.draft && !greedy) {
                gather(1, node);
                drow = row_at<KIND>(p.draft, b * p.d_sb + node * p.d_st);
            }
            mass = fz[0];
            rejected = 0;
        };
        // r's weight of token v (times `mass`, but with draft logits, once a child was refused: of sum 1)
        auto rest = [&](int v) -> double {
            const double w = weight(logit<KIND>(lrow, v), ftop[0], inv);
            if (!p.draft) {
                for (int i = 0; i < rejected; ++i)
                    if (out_of[i] == v) return 0.0;
                return w;
            }
            if (rejected == 0) return w;
            const double q = weight(logit<KIND>(drow, v), ftop[1], inv) / fz[1];
            double r = w / fz[0];
            for (int i = 0; i < rejected; ++i) {
                r -= q;
                r = (r > 0.0 ? r : 0.0) * scale[i];
            }
            return r;
        };
        enter();
        for (int i = 1; i < count; ++i) {
            if (parents[i] != node || i <= node) continue;
            const int64_t x64 = tokens[i];
            if (x64 < 0 || x64 >= p.V || fz[0] == 0.0) continue;
            const int x = (int)x64;
            bool take;
            if (greedy) {
                take = x == fat[0];
            } else if (!p.draft) {
                take = (double)uniforms[i] * mass < rest(x);
            } else {
                if (fz[1] == 0.0) continue;
                const double q = weight(logit<KIND>(drow, x), ftop[1], inv) / fz[1];
                const double r = rejected ? rest(x) : weight(logit<KIND>(lrow, x), ftop[0], inv) / fz[0];
                take = (double)uniforms[i] * q < r;
            }
            if (take) {
                if (tid == 0) {
                    pout[n] = i;
                    tout[n - 1] = x;
                }
                ++n;
                node = i;
                enter();
                continue;
            }
            if (greedy) continue;
            if (!p.draft) {
                const double keep_mass = mass;
                __syncthreads();
                if (tid == 0) out_of[rejected] = x;
                ++rejected;
                __syncthreads();
                double s = 0.0;
                const int c = x / kChunk;
                for (int j = 0; j < kPer; ++j) {
                    const int v = c * kChunk + j * kThreads + tid;
                    if (v < p.V) s += rest(v);
                }
                s = block_sum(s);
                double all = 0.0;
                for (int j = lane; j < p.chunks; j += 64) all += j == c ? s : part[j];
                all = wave_sum(all);
                if (all > 0.0) {
                    __syncthreads();
                    if (tid == 0) part[c] = s;
                    mass = all;
                    __syncthreads();
                } else {
                    --rejected;  // nothing would remain: r stays
                    mass = keep_mass;
                }
            } else {
                __syncthreads();
                if (tid == 0) scale[rejected] = 1.0;
                ++rejected;
                __syncthreads();
                double all = 0.0;
                for (int v = tid; v < p.V; v += kThreads) all += rest(v);
                all = block_sum(all);
                if (all > 0.0) {
                    if (tid == 0) scale[rejected - 1] = 1.0 / all;
                    __syncthreads();
                } else {
                    --rejected;
                }
            }
        }
        // The token that follows.
        int64_t next = -1;
        if (fz[0] != 0.0) {
            if (greedy) {
                next = fat[0];
            } else {
                if (p.draft && rejected) {
                    for (int c = 0; c < p.chunks; ++c) {
                        double s = 0.0;
                        for (int j = 0; j < kPer; ++j) {
                            const int v = c * kChunk + j * kThreads + tid;
                            if (v < p.V) s += rest(v);
                        }
                        s = block_sum(s);
                        if (tid == 0) part[c] = s;
                    }
                }
                __syncthreads();
                double all = 0.0;
                for (int c = 0; c < p.chunks; ++c) all += part[c];
                const double goal = (double)uniforms[0] * all;
                double before = 0.0;
                int chunk = -1, last = -1;
                for (int c = 0; c < p.chunks; ++c) {
                    if (part[c] > 0.0) last = c;
                    if (before + part[c] > goal) {
                        chunk = c;
                        break;
                    }
                    before += part[c];
                }
                const bool beyond = chunk < 0;  // a uniform number of 1 or more, or none: the last token there is
                if (beyond) chunk = last;
                // a thread has kPer neighbouring tokens of the chunk
                double w[kPer], mine = 0.0;
                for (int j = 0; j < kPer; ++j) {
                    const int v = chunk * kChunk + tid * kPer + j;
                    w[j] = v < p.V ? rest(v) : 0.0;
                    mine += w[j];
                }
                double run = mine;
                for (int o = 1; o < 64; o <<= 1) {
                    const double t = __shfl_up(run, o);
                    if (lane >= o) run += t;
                }
                __syncthreads();
                if (lane == 63) red[wave] = run;
                if (tid == 0) found = 0x7fffffff, fat[1] = -1;
                __syncthreads();
                for (int i = 0; i < wave; ++i) run += red[i];
                run = before + run - mine;
                int hit = 0x7fffffff, tail = -1;
                for (int j = 0; j < kPer; ++j) {
                    run += w[j];
                    if (w[j] > 0.0) {
                        tail = chunk * kChunk + tid * kPer + j;
                        if (!beyond && run > goal && hit == 0x7fffffff) hit = tail;
                    }
                }
                atomicMin(&found, hit);
                atomicMax(&fat[1], tail);
                __syncthreads();
                next = found == 0x7fffffff ? fat[1] : found;
            }
        }
        if (tid == 0) tout[n - 1] = next;
    }
    for (int i = n + tid; i < p.T; i += kThreads) {
        tout[i] = -1;
        pout[i] = -1;
    }
    if (tid == 0) p.counts_out[b] = n;
}

template <int KIND>
static void launch(const Params& p, hipStream_t st) {
    const int64_t rows = (int64_t)p.B * p.T * (p.draft ? 2 : 1);
    hipLaunchKernelGGL(stats_kernel<KIND>, dim3((unsigned)(rows * p.chunks)), dim3(kThreads), 0, st, p);
    hipLaunchKernelGGL(walk_kernel<KIND>, dim3(p.B), dim3(kThreads), 0, st, p);
}

}  // namespace verify
}  // namespace mx

using namespace mx;

extern "C" size_t mx_verify_draft_workspace_bytes(int32_t B, int32_t T, int32_t V, int32_t draft) {
    if (B <= 0 || T <= 0 || V <= 0) return 0;
    return (size_t)B * T * (draft ? 2 : 1) * ceil_div(V, verify::kChunk) * sizeof(verify::Stat);
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
    if (flags & ~(uint32_t)(MX_PA_BF16 | MX_LOGITS_FP32) || flags == (MX_PA_BF16 | MX_LOGITS_FP32))
        return fail(MX_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
    if (l_sb < 0 || l_st < 0 || d_sb < 0 || d_st < 0 || t_sb < 0 || p_sb < 0 || u_sb < 0 || temp_sb < 0)
        return fail(MX_ERR_INVALID, "%s: strides must be >= 0", what);
    if (T > verify::kMaxNodes) return fail(MX_ERR_UNSUPPORTED, "%s: more than %d nodes", what, verify::kMaxNodes);
    if (V > verify::kMaxChunks * verify::kChunk)
        return fail(MX_ERR_UNSUPPORTED, "%s: more than %d logits", what, verify::kMaxChunks * verify::kChunk);
    const int chunks = (int)ceil_div(V, verify::kChunk);
    if ((double)B * T * 2 * chunks * verify::kThreads > 4.0e9)
        return fail(MX_ERR_UNSUPPORTED, "%s: more logits than one launch holds", what);
    const size_t need = mx_verify_draft_workspace_bytes(B, T, V, draft_logits != nullptr);
    if (!workspace || workspace_bytes < need)
        return fail(MX_ERR_WORKSPACE, "%s: workspace needs %zu bytes, got %zu", what, need, workspace ? workspace_bytes : 0);
    if (!aligned(workspace, 16)) return fail(MX_ERR_ALIGNMENT, "%s: workspace alignment", what);
    verify::Params p{};
    p.logits = logits, p.l_sb = l_sb, p.l_st = l_st;
    p.draft = draft_logits, p.d_sb = d_sb, p.d_st = d_st;
    p.tokens = tokens, p.t_sb = t_sb, p.parents = parents, p.p_sb = p_sb, p.counts = counts;
    p.uniforms = uniforms, p.u_sb = u_sb, p.temps = temperatures, p.temp_sb = temp_sb;
    p.B = B, p.T = T, p.V = V, p.chunks = chunks;
    p.stats = static_cast<verify::Stat*>(workspace);
    p.tokens_out = tokens_out, p.counts_out = counts_out, p.path_out = path_out;
    hipStream_t st = as_stream(stream);
    if (flags & MX_LOGITS_FP32) verify::launch<2>(p, st);
    else if (flags & MX_PA_BF16) verify::launch<1>(p, st);
    else verify::launch<0>(p, st);
    return check_launch(what);
}
