// Append to the paged 8-bit cache: rotation of the new keys, one power-of-two scale per 16 tokens and head, e4m3
// codes, in one pass.
//
// A warp owns one block (16 tokens of one sequence) and head: its rows stay in registers between the maximum and
// the rounding, so k and v are read once and the codes written once. The scale 2^e, e = ceil(log2(amax / 448)),
// comes from the exponent and mantissa bits of amax, and dividing by it is exact, so the only roundings are the
// rotation's (32 bits) and the one to e4m3. A block that already holds tokens keeps max(old e, new e); when
// that raises it, the older codes are multiplied by 2^(old - new), exact until they reach e4m3's subnormals.
// Cosines and sines come from the fast functions at a reduced angle (5e-7, against e4m3's half step of 2^-5).
#include "kv.cuh"

#include <cuda_fp8.h>

namespace eva {

constexpr int APPEND_WARPS = 4;   // the blocks of one page, so that its value rows' sectors meet in L2

struct AppendArgs {
    EvaKvCache c;
    EvaKvBatch b;
    EvaRotary r;
    const void* k;
    const void* v;
    int64_t kt, kh, vt, vh;
    int blocks;   // blocks one sequence's max_q rows can touch
    int64_t warps;
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// e4m3 code(s) times m, rounded to e4m3
__device__ __forceinline__ uint32_t e4m3_scaled(uint32_t two, float m)
{
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    return e4m3x2(f.x * m, f.y * m);
}

// Smallest biased exponent whose scale brings amax into e4m3's range (448 = 1.75 * 2^8), 1 .. 254.
__device__ __forceinline__ int scale_byte(uint32_t amax_bits)
{
    const int e = static_cast<int>(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, 1), 254);
}

// Up to 2^126 from byte 1: the product of amax's bound with it stays finite.
__device__ __forceinline__ float inv_scale(int byte) { return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23); }

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

template <typename T> __device__ __forceinline__ float up(T v);
template <> __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float up(__half v) { return __half2float(v); }

template <typename T, int DK, int DV>
__global__ void __launch_bounds__(APPEND_WARPS * 32) kv_append_kernel(const AppendArgs p)
{
    constexpr int KS = DK / 64, VS = DV / 32;   // key pairs and value dimensions of a lane
    const int lane = threadIdx.x & 31;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * APPEND_WARPS + (threadIdx.x >> 5);
    if (w >= p.warps) return;
    const int64_t bh = w / p.blocks;
    const int h = static_cast<int>(bh % p.c.kv_heads), b = static_cast<int>(bh / p.c.kv_heads);
    const KvSeq s = kv_seq(p.b, b, p.c.status);
    const int first = max(s.ctx, 0);
    const int base = (first / KV_BLOCK + static_cast<int>(w - bh * p.blocks)) * KV_BLOCK;
    if (base >= s.len) return;
    const int page = kv_page(p.c, p.b, b, base / KV_PAGE, p.c.status);
    if (page < 0) return;
    const int lo = max(first - base, 0), hi = min(s.len - base, KV_BLOCK), at = base % KV_PAGE;
    const int64_t ph = static_cast<int64_t>(page) * p.c.kv_heads + h;
    const int64_t tok0 = static_cast<int64_t>(s.row0) + base - s.ctx;   // token row of the block's slot 0
    const T* kp = static_cast<const T*>(p.k) + h * p.kh + tok0 * p.kt;
    const T* vp = static_cast<const T*>(p.v) + h * p.vh + tok0 * p.vt;

    // values: dimension lane + 32 m, the block's tokens in registers
    float v[VS][KV_BLOCK];
    uint32_t bad = 0, vmax = 0;
#pragma unroll
    for (int r = 0; r < KV_BLOCK; ++r)
#pragma unroll
        for (int m = 0; m < VS; ++m) v[m][r] = r >= lo && r < hi ? up(vp[r * p.vt + lane + 32 * m]) : 0.0f;
    // keys: pair lane + 32 m of the rotated pairs, then of the others (neighbours)
    float ka[KS][KV_BLOCK], kb[KS][KV_BLOCK];
    int da[KS], db[KS];
    const int half = p.r.dim / 2;
#pragma unroll
    for (int m = 0; m < KS; ++m) {
        const int i = lane + 32 * m;
        if (i < half) {
            da[m] = p.r.offset + (p.r.interleaved ? 2 * i : i);
            db[m] = da[m] + (p.r.interleaved ? 1 : half);
        } else {
            const int d = 2 * (i - half);
            da[m] = d < p.r.offset ? d : d + p.r.dim;
            db[m] = da[m] + 1;
        }
    }
#pragma unroll
    for (int m = 0; m < KS; ++m)
#pragma unroll
        for (int r = 0; r < KV_BLOCK; ++r) {
            const bool in = r >= lo && r < hi;
            ka[m][r] = in ? up(kp[r * p.kt + da[m]]) : 0.0f;
            kb[m][r] = in ? up(kp[r * p.kt + db[m]]) : 0.0f;
        }
#pragma unroll
    for (int m = 0; m < VS; ++m)
#pragma unroll
        for (int r = 0; r < KV_BLOCK; ++r) {
            if (!finite(v[m][r])) {
                bad |= 1u << r;
                v[m][r] = 0.0f;
            }
            vmax = max(vmax, __float_as_uint(fabsf(v[m][r])));
        }
    uint32_t kmax = 0;
#pragma unroll
    for (int m = 0; m < KS; ++m) {
        const int i = lane + 32 * m;
        if (i < half) {
            const uint64_t turns = p.r.turns[i];
#pragma unroll
            for (int r = 0; r < KV_BLOCK; ++r) {
                float sn, cs;
                __sincosf(kv_half_turns(base + r, turns) * 3.14159265358979f, &sn, &cs);
                sn *= p.r.mscale;
                cs *= p.r.mscale;
                const float x = ka[m][r], y = kb[m][r];
                ka[m][r] = x * cs - y * sn;
                kb[m][r] = y * cs + x * sn;
            }
        }
#pragma unroll
        for (int r = 0; r < KV_BLOCK; ++r) {
            if (!finite(ka[m][r]) || !finite(kb[m][r])) bad |= 1u << r;
            if (finite(ka[m][r])) kmax = max(kmax, __float_as_uint(fabsf(ka[m][r])));
            if (finite(kb[m][r])) kmax = max(kmax, __float_as_uint(fabsf(kb[m][r])));
        }
    }
    bad = __reduce_or_sync(0xffffffffu, bad);
    // a token with a non-finite element has no key of its own: it does not count for the scale either
    if (bad) {
        kmax = 0;
#pragma unroll
        for (int m = 0; m < KS; ++m)
#pragma unroll
            for (int r = 0; r < KV_BLOCK; ++r) {
                if (bad >> r & 1) ka[m][r] = kb[m][r] = __uint_as_float(0x7fc00000u);
                else kmax = max(kmax, max(__float_as_uint(fabsf(ka[m][r])), __float_as_uint(fabsf(kb[m][r]))));
            }
    }
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    vmax = __reduce_max_sync(0xffffffffu, vmax);

    uint8_t* ks = static_cast<uint8_t*>(p.c.k_scale) + ph * KV_PAGE_BLOCKS + at / KV_BLOCK;
    uint8_t* vs = static_cast<uint8_t*>(p.c.v_scale) + ph * KV_PAGE_BLOCKS + at / KV_BLOCK;
    uint8_t* kc = static_cast<uint8_t*>(p.c.k) + (ph * KV_PAGE + at) * DK;
    uint8_t* vc = static_cast<uint8_t*>(p.c.v) + ph * KV_PAGE * DV + at;
    int ke = scale_byte(kmax), ve = scale_byte(vmax);
    if (lo > 0) {
        const int ko = max(static_cast<int>(*ks), 1), vo = max(static_cast<int>(*vs), 1);
        ke = max(ke, ko);
        ve = max(ve, vo);
        if (ke > ko) {   // the older keys: lo rows of DK bytes, contiguous
            const float m = inv_scale(ke) * kv_scale(ko);
            for (int i = lane; i < lo * DK / 2; i += 32) {
                uint16_t* q = reinterpret_cast<uint16_t*>(kc) + i;
                *q = static_cast<uint16_t>(e4m3_scaled(*q, m));
            }
        }
        const float m = inv_scale(ve) * kv_scale(vo);
#pragma unroll
        for (int j = 0; j < VS; ++j) {
            uint8_t* q = vc + static_cast<int64_t>(lane + 32 * j) * KV_PAGE;
            const uint4 o = *reinterpret_cast<const uint4*>(q);
            uint32_t in[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int t = 0; t < 8; ++t) {   // tokens 2 t, 2 t + 1
                const uint32_t was = in[t / 2] >> (t % 2 * 16) & 0xffffu;
                const uint32_t moved = ve > vo ? e4m3_scaled(was, m) : was;
                const uint32_t fresh = e4m3x2(v[j][2 * t] * inv_scale(ve), v[j][2 * t + 1] * inv_scale(ve));
                const uint32_t a = 2 * t < lo ? moved : 2 * t < hi ? fresh : was;
                const uint32_t c = 2 * t + 1 < lo ? moved : 2 * t + 1 < hi ? fresh : was;
                const uint32_t two = (a & 0xffu) | (c & 0xff00u);
                in[t / 2] = t % 2 ? (in[t / 2] & 0xffffu) | two << 16 : (in[t / 2] & 0xffff0000u) | two;
            }
            *reinterpret_cast<uint4*>(q) = make_uint4(in[0], in[1], in[2], in[3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VS; ++j) {
            uint8_t* q = vc + static_cast<int64_t>(lane + 32 * j) * KV_PAGE;
            uint32_t in[4] = {0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < 8; ++t)
                in[t / 2] |= e4m3x2(v[j][2 * t] * inv_scale(ve), v[j][2 * t + 1] * inv_scale(ve)) << (t % 2 * 16);
            if (hi == KV_BLOCK) {
                *reinterpret_cast<uint4*>(q) = make_uint4(in[0], in[1], in[2], in[3]);
            } else {
                for (int t = 0; t < KV_BLOCK; ++t)
                    if (t < hi) q[t] = static_cast<uint8_t>(in[t / 4] >> (t % 4 * 8));
            }
        }
    }
    const float inv = inv_scale(ke);
#pragma unroll
    for (int m = 0; m < KS; ++m)
#pragma unroll
        for (int r = 0; r < KV_BLOCK; ++r)
            if (r >= lo && r < hi) {
                const uint32_t two = e4m3x2(ka[m][r] * inv, kb[m][r] * inv);
                kc[r * DK + da[m]] = static_cast<uint8_t>(two);
                kc[r * DK + db[m]] = static_cast<uint8_t>(two >> 8);
            }
    __syncwarp();   // every lane has read the old scales
    if (lane == 0) {
        *ks = static_cast<uint8_t>(ke);
        *vs = static_cast<uint8_t>(ve);
    }
}

template <typename T> static cudaError_t append_typed(const AppendArgs& p, cudaStream_t st)
{
    const int64_t grid = (p.warps + APPEND_WARPS - 1) / APPEND_WARPS;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    const unsigned g = static_cast<unsigned>(grid);
    if (p.c.key_dim == 64) kv_append_kernel<T, 64, 64><<<g, APPEND_WARPS * 32, 0, st>>>(p);
    else if (p.c.key_dim == 128) kv_append_kernel<T, 128, 128><<<g, APPEND_WARPS * 32, 0, st>>>(p);
    else kv_append_kernel<T, 192, 128><<<g, APPEND_WARPS * 32, 0, st>>>(p);
    return cudaGetLastError();
}

bool kv_cache_ok(const EvaKvCache* c)
{
    if (!c || c->pages < 1 || c->kv_heads < 1 || c->kv_heads > 65535 || !c->k || !c->v || !c->k_scale || !c->v_scale ||
        !c->status)
        return false;
    const bool dims = (c->key_dim == 64 && c->value_dim == 64) || (c->key_dim == 128 && c->value_dim == 128) ||
                      (c->key_dim == 192 && c->value_dim == 128);
    return dims && ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) == 0 &&
           ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) |
             reinterpret_cast<uintptr_t>(c->status)) & 3) == 0;
}

bool kv_batch_ok(const EvaKvBatch* b)
{
    if (!b || b->seqs < 0 || b->tokens < 0 || b->max_q < 0 || b->max_pages < 0 || b->max_pages > (1 << 24) ||
        b->table_stride < 0 || b->seqs > (1 << 24) || b->max_q > (1 << 28))
        return false;
    if (b->seqs == 0 || b->tokens == 0) return true;
    return b->q_start && b->seq_lens && b->table && b->max_pages > 0 &&
           ((reinterpret_cast<uintptr_t>(b->q_start) | reinterpret_cast<uintptr_t>(b->seq_lens) |
             reinterpret_cast<uintptr_t>(b->table)) & 3) == 0;
}

}  // namespace eva

using namespace eva;

extern "C" int eva_kv_append(const EvaKvCache* cache, const EvaKvBatch* batch, const EvaRotary* rotary, const void* k,
                             int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                             int64_t v_head_stride, int32_t dtype, void* stream)
{
    if (!kv_cache_ok(cache) || !kv_batch_ok(batch) || (dtype != EVA_DTYPE_F16 && dtype != EVA_DTYPE_BF16))
        return EVA_ERR_INVALID;
    if (rotary && (!rotary_ok(rotary, cache->key_dim) || rotary->inverse)) return EVA_ERR_INVALID;
    if (batch->seqs == 0 || batch->tokens == 0 || batch->max_q == 0) return EVA_OK;
    if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 1)) return EVA_ERR_INVALID;
    AppendArgs p{};
    p.c = *cache;
    p.b = *batch;
    if (rotary) p.r = *rotary;
    p.k = k;
    p.v = v;
    p.kt = k_token_stride;
    p.kh = k_head_stride;
    p.vt = v_token_stride;
    p.vh = v_head_stride;
    p.blocks = (batch->max_q + KV_BLOCK - 2) / KV_BLOCK + 1;
    p.warps = static_cast<int64_t>(batch->seqs) * cache->kv_heads * p.blocks;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == EVA_DTYPE_BF16 ? append_typed<__nv_bfloat16>(p, st) : append_typed<__half>(p, st);
    return e == cudaSuccess ? EVA_OK : EVA_ERR_CUDA;
}
