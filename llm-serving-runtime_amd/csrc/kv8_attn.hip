// Decode attention over the 8-bit KV cache (kv8.h) on gfx950: out = softmax(scale q K^T) V per query
// head, K and V the values that the pages stand for. The 8-bit form of paged_attn.hip, which replaces
// paged_attention_decode_batched (runtime/phase2/paged_attention_triton.py:745-775).
#include "common.h"
#include "elt.h"
#include "kv8.h"

namespace mx {
namespace kv8 {

constexpr int kAttnWaves = 4;

struct AttnParams {
    const uint16_t* q;
    int64_t q_sb, q_sh;
    Pages pages;
    const int32_t* bt;
    int64_t bt_sb;
    int max_blocks;
    const int32_t* seq_lens;
    int Hq, G;
    float scale_log2e;
    uint16_t* out;
    int64_t o_sb, o_sh;
    int32_t* err;
};

// One workgroup per (row, query head); its waves take the row's 64-token stretches in turn, a lane
// scoring one token, then D / 64 output dims.
template <int D, int BS, bool BF16>
__global__ __launch_bounds__(kAttnWaves * 64) void kv8_attn_kernel(AttnParams p) {
    constexpr int DP = D / 64;
    __shared__ float qs[D];
    __shared__ float ps[kAttnWaves][64];
    __shared__ int pg[kAttnWaves][64];
    __shared__ float red[kAttnWaves][D + 2];
    const int h = blockIdx.x, b = blockIdx.y, kvh = h / p.G;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint16_t* q = p.q + (int64_t)b * p.q_sb + (int64_t)h * p.q_sh;
    if (threadIdx.x < D) qs[threadIdx.x] = widen<BF16>(q[threadIdx.x]) * p.scale_log2e;
    __syncthreads();
    int64_t len = p.seq_lens[b];
    const int64_t most = (int64_t)p.max_blocks * BS;
    len = len < 0 ? 0 : (len < most ? len : most);
    const float kNegInf = -__builtin_huge_valf();
    float m = kNegInf, l = 0.0f, acc[DP];
    for (int j = 0; j < DP; ++j) acc[j] = 0.0f;
    for (int64_t t0 = wave * 64; t0 < len; t0 += kAttnWaves * 64) {
        const int64_t t = t0 + lane;
        int phys = -1;
        float s = kNegInf;
        if (t < len) {
            phys = p.bt[(int64_t)b * p.bt_sb + t / BS];
            if ((unsigned)phys >= (unsigned)p.pages.num_blocks) {
                if (p.err) atomicOr(p.err, 4);
                phys = -1;
            }
        }
        if (phys >= 0) {
            const uint8_t* run = p.pages.data + run_offset<D, BS>(p.pages, phys, kvh, 0) + (t % BS) * 64;
            s = 0.0f;
            for (int d = 0; d < D; ++d) s += qs[d] * ((float)run[(d / 64) * (BS * 64) + d % 64] - 128.0f);
            s *= scale_of(p.pages.codes[code_offset(p.pages, phys, kvh, 0)]);
        }
        float mx = s;
        for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        const float mn = fmaxf(m, mx), ref = mn == kNegInf ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        const float pr = phys >= 0 ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
        m = mn;
        l = l * alpha + pr;
        ps[wave][lane] = pr;
        pg[wave][lane] = phys;
        __builtin_amdgcn_wave_barrier();
        for (int j = 0; j < DP; ++j) acc[j] *= alpha;
        for (int i = 0; i < 64; ++i) {
            const int ph = pg[wave][i];
            if (ph < 0) continue;
            const uint8_t* run = p.pages.data + run_offset<D, BS>(p.pages, ph, kvh, 1) + (t0 + i) % BS;
            const float w = ps[wave][i] * scale_of(p.pages.codes[code_offset(p.pages, ph, kvh, 1)]);
            for (int j = 0; j < DP; ++j) acc[j] += w * ((float)run[(lane * DP + j) * BS] - 128.0f);
        }
        __builtin_amdgcn_wave_barrier();
    }
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    for (int j = 0; j < DP; ++j) red[wave][lane * DP + j] = acc[j];
    if (lane == 0) {
        red[wave][D] = m;
        red[wave][D + 1] = l;
    }
    __syncthreads();
    if (threadIdx.x < D) {
        float mx = kNegInf;
        for (int w = 0; w < kAttnWaves; ++w) mx = fmaxf(mx, red[w][D]);
        const float ref = mx == kNegInf ? 0.0f : mx;
        float num = 0.0f, den = 0.0f;
        for (int w = 0; w < kAttnWaves; ++w) {
            const float a = __builtin_amdgcn_exp2f(red[w][D] - ref);
            num += a * red[w][threadIdx.x];
            den += a * red[w][D + 1];
        }
        const float o = den == 0.0f ? 0.0f : num / den;
        uint16_t* dst = p.out + (int64_t)b * p.o_sb + (int64_t)h * p.o_sh + threadIdx.x;
        *dst = __builtin_bit_cast(uint16_t, Elt<BF16>::round(o));
    }
}

}  // namespace kv8
}  // namespace mx

using namespace mx;

extern "C" size_t mx_kv8_attn_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_blocks,
                                              int32_t block_size) {
    return 0;
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
    if (flags & ~(uint32_t)MX_PA_BF16) return fail(MX_ERR_INVALID, "%s: unknown flags 0x%x", what, flags);
    if (!aligned(q, 16) || q_sb % 8 || q_sh % 8 || !aligned(out, 16) || o_sb % 8 || o_sh % 8)
        return fail(MX_ERR_ALIGNMENT, "%s: q and out rows must be 16-byte aligned", what);
    kv8::AttnParams p{q, q_sb, q_sh, {const_cast<uint8_t*>(data), const_cast<uint8_t*>(codes), Hkv, num_blocks},
                      block_tables, bt_sb, max_blocks, seq_lens, Hq, Hq / Hkv, scale * 1.4426950408889634f, out, o_sb,
                      o_sh, err};
    hipStream_t st = as_stream(stream);
#define CALL(DD, BB)                                                                                                   \
    if (flags & MX_PA_BF16)                                                                                            \
        hipLaunchKernelGGL((kv8::kv8_attn_kernel<DD, BB, true>), dim3(Hq, B), dim3(kv8::kAttnWaves * 64), 0, st, p);    \
    else                                                                                                               \
        hipLaunchKernelGGL((kv8::kv8_attn_kernel<DD, BB, false>), dim3(Hq, B), dim3(kv8::kAttnWaves * 64), 0, st, p)
    MX_KV8_DISPATCH(D, block_size, CALL)
#undef CALL
    return check_launch(what);
}
