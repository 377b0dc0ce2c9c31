// Shared by the attention kernels over the paged cache.
#pragma once

#include <atomic>

#include "kv.cuh"

namespace eva {

constexpr int COMBINE_THREADS = 512;

struct AttendArgs {
    EvaKvCache c;
    EvaKvBatch b;
    const void* q;
    void* out;
    int64_t qt, qh;        // strides of q, elements
    int heads, group, window;
    float scale;           // times log2(e): the softmax's exponentials are powers of two
    int part_rows;         // rows of a partial sum
    int4* heads_of;        // [pieces]: item that begins in a piece and goes on {sequence, head, last piece}, -1: none
    float* part;           // [pieces][2] partial sums
};

template <typename T> __device__ __forceinline__ float2 two_floats(uint32_t bits);
template <> __device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t bits)
{
    return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 two_floats<__half>(uint32_t bits)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&bits));
}

template <typename T> __device__ __forceinline__ uint32_t two_bits(float lo, float hi);
template <> __device__ __forceinline__ uint32_t two_bits<__nv_bfloat16>(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t two_bits<__half>(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T> __device__ __forceinline__ T one_of(float v);
template <> __device__ __forceinline__ __nv_bfloat16 one_of(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half one_of(float v) { return __float2half_rn(v); }

// four e4m3 codes as four halves, exact
__device__ __forceinline__ void e4m3_halves(uint32_t four, uint32_t& lo, uint32_t& hi)
{
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One row's output from its partial sums, by a warp: maximum at part(k)[im], sum at part(k)[is], output from part(k) + io.
template <int DV, typename T, typename P>
__device__ __forceinline__ void join_parts(const P& part, int parts, int im, int is, int64_t io, T* out, int lane)
{
    float m = -INFINITY;
    for (int k = lane; k < parts; k += 32) m = fmaxf(m, part(k)[im]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ref = m == -INFINITY ? 0.0f : m;
    const int d = (lane * 4) % DV;
    float o[4] = {}, l = 0.0f;
    for (int k0 = 0; k0 < parts; k0 += 32) {
        float w = 0.0f;
        if (k0 + lane < parts) {
            w = ex2(part(k0 + lane)[im] - ref);
            l = fmaf(part(k0 + lane)[is], w, l);
        }
        const int n = min(32, parts - k0);
#pragma unroll 8
        for (int k = 0; k < n; ++k) {
            const float wk = __shfl_sync(0xffffffffu, w, k);
            const float2 v = *reinterpret_cast<const float2*>(part(k0 + k) + io + d), u = *reinterpret_cast<const float2*>(part(k0 + k) + io + d + 2);
            o[0] = fmaf(v.x, wk, o[0]);
            o[1] = fmaf(v.y, wk, o[1]);
            o[2] = fmaf(u.x, wk, o[2]);
            o[3] = fmaf(u.y, wk, o[3]);
        }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (lane * 4 < DV)
        *reinterpret_cast<uint2*>(out + d) = make_uint2(two_bits<T>(o[0] * inv, o[1] * inv), two_bits<T>(o[2] * inv, o[3] * inv));
}

// Shared memory of a kernel above the default, set once per device (`done`: a bit each).
inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done)
{
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t{1} << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Many rows (kv_prompt.cu): workspace bytes for a value dimension, and the launch.
size_t prompt_workspace(int dv);
cudaError_t launch_prompt(AttendArgs p, void* workspace, bool bf16, cudaStream_t st);

}  // namespace eva
