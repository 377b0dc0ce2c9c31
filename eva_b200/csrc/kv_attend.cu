// Attention over the paged 8-bit cache.
//
// One warp per token row and query head, one pass over the tokens with the running maximum and sum of the softmax in
// 32 bits: 32 tokens at a time, a lane scores one of them, then the lanes share the value dimensions.
#include "kv.cuh"

#include <cuda_fp8.h>

namespace eva {

constexpr int ATT_WARPS = 4;

struct AttendArgs {
    EvaKvCache c;
    EvaKvBatch b;
    const void* q;
    void* out;
    int64_t qt, qh;
    int heads, group, window, bf16;
    float scale;   // times log2(e)
};

__device__ __forceinline__ float e4m3_up(uint32_t byte)
{
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

template <int DK, int DV>
__global__ void __launch_bounds__(ATT_WARPS * 32) kv_attend_kernel(const AttendArgs p)
{
    __shared__ float qs[ATT_WARPS][DK];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * ATT_WARPS + warp;
    const int64_t bi = w / p.heads;
    const int head = static_cast<int>(w - bi * p.heads), kvh = head / p.group;
    const int b = static_cast<int>(bi / p.b.max_q), i = static_cast<int>(bi - static_cast<int64_t>(b) * p.b.max_q);
    if (b >= p.b.seqs) return;
    const KvSeq s = kv_seq(p.b, b, p.c.status);
    if (i >= s.n) return;
    const int64_t row = s.row0 + i;
    for (int d = lane; d < DK; d += 32) {
        const int64_t at = row * p.qt + head * p.qh + d;
        qs[warp][d] = p.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[at])
                             : __half2float(static_cast<const __half*>(p.q)[at]);
    }
    __syncwarp();
    const int pos = s.ctx + i, end = pos + 1, begin = p.window > 0 ? max(0, end - p.window) : 0;
    float m = -INFINITY, l = 0.0f, o[DV / 32] = {};
    for (int t0 = begin & ~31; t0 < end; t0 += 32) {
        const int page = kv_page(p.c, p.b, b, t0 / KV_PAGE, p.c.status);
        if (page < 0) continue;
        const int64_t ph = static_cast<int64_t>(page) * p.c.kv_heads + kvh;
        const int t = t0 + lane, in = t0 % KV_PAGE;
        const uint8_t* kr = static_cast<const uint8_t*>(p.c.k) + (ph * KV_PAGE + in + lane) * DK;
        const uint8_t* ksc = static_cast<const uint8_t*>(p.c.k_scale) + ph * KV_PAGE_BLOCKS + in / KV_BLOCK;
        const uint8_t* vsc = static_cast<const uint8_t*>(p.c.v_scale) + ph * KV_PAGE_BLOCKS + in / KV_BLOCK;
        float x = 0.0f;
        for (int d = 0; d < DK; ++d) x = fmaf(qs[warp][d], e4m3_up(kr[d]), x);
        x *= kv_scale(ksc[lane / KV_BLOCK]) * p.scale;
        const bool seen = t >= begin && t < end;
        x = seen ? x : -INFINITY;
        float mx = x;
#pragma unroll
        for (int sft = 16; sft > 0; sft >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sft));
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.0f : mn, down = exp2f(m - ref);
        const float e = seen ? exp2f(x - ref) : 0.0f;
        m = mn;
        l = l * down + e;
        const float ev = e * kv_scale(vsc[lane / KV_BLOCK]);
        const uint8_t* vr = static_cast<const uint8_t*>(p.c.v) + ph * KV_PAGE * DV + in;
#pragma unroll
        for (int j = 0; j < DV / 32; ++j) o[j] *= down;
        for (int u = 0; u < 32; ++u) {
            const float pu = __shfl_sync(0xffffffffu, ev, u);
            if (t0 + u < begin || t0 + u >= end) continue;
#pragma unroll
            for (int j = 0; j < DV / 32; ++j) o[j] = fmaf(pu, e4m3_up(vr[(lane + 32 * j) * KV_PAGE + u]), o[j]);
        }
    }
#pragma unroll
    for (int sft = 16; sft > 0; sft >>= 1) l += __shfl_xor_sync(0xffffffffu, l, sft);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < DV / 32; ++j) {
        const int64_t at = (row * p.heads + head) * DV + lane + 32 * j;
        if (p.bf16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(o[j] * inv);
        else static_cast<__half*>(p.out)[at] = __float2half_rn(o[j] * inv);
    }
}

}  // namespace eva

using namespace eva;

static bool attend_ok(const EvaKvCache* cache, const EvaKvBatch* batch, int32_t heads)
{
    return kv_cache_ok(cache) && kv_batch_ok(batch) && heads >= 1 && heads % cache->kv_heads == 0;
}

extern "C" size_t eva_kv_attend_workspace(const EvaKvCache* cache, const EvaKvBatch* batch, int32_t heads)
{
    return attend_ok(cache, batch, heads) ? 16 : 0;
}

extern "C" int eva_kv_attend(const EvaKvCache* cache, const EvaKvBatch* batch, const void* q, int32_t dtype, int32_t heads,
                             int64_t q_token_stride, int64_t q_head_stride, float scale, int32_t window, void* workspace,
                             size_t workspace_bytes, void* out, void* stream)
{
    if (!attend_ok(cache, batch, heads) || (dtype != EVA_DTYPE_F16 && dtype != EVA_DTYPE_BF16) || window < 0 ||
        !(scale >= 0.0f) || scale > 3.0e38f)
        return EVA_ERR_INVALID;
    if (batch->seqs == 0 || batch->tokens == 0 || batch->max_q == 0) return EVA_OK;
    if (!q || !out || !workspace ||
        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
        q_token_stride % 8 || q_head_stride % 8)
        return EVA_ERR_INVALID;
    if (workspace_bytes < eva_kv_attend_workspace(cache, batch, heads)) return EVA_ERR_WORKSPACE;
    AttendArgs p{};
    p.c = *cache;
    p.b = *batch;
    p.q = q;
    p.out = out;
    p.qt = q_token_stride;
    p.qh = q_head_stride;
    p.heads = heads;
    p.group = heads / cache->kv_heads;
    p.window = window;
    p.bf16 = dtype == EVA_DTYPE_BF16;
    p.scale = scale * 1.4426950408889634f;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t warps = static_cast<int64_t>(batch->seqs) * batch->max_q * heads;
    const int64_t grid = (warps + ATT_WARPS - 1) / ATT_WARPS;
    if (grid > 0x7fffffff) return EVA_ERR_INVALID;
    const unsigned g = static_cast<unsigned>(grid);
    if (cache->key_dim == 64) kv_attend_kernel<64, 64><<<g, ATT_WARPS * 32, 0, st>>>(p);
    else if (cache->key_dim == 128) kv_attend_kernel<128, 128><<<g, ATT_WARPS * 32, 0, st>>>(p);
    else kv_attend_kernel<192, 128><<<g, ATT_WARPS * 32, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? EVA_OK : EVA_ERR_CUDA;
}
