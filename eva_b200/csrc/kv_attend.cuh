// Shared by the attention kernels over the paged cache.
#pragma once

#include <atomic>

#include "kv.cuh"

namespace eva {

constexpr int COMBINE_THREADS = 512;

// A block's value scale 2^e joins its tokens' exponents as max(e, VALUE_EXP_MIN); what is left of it, 1 but for blocks whose values are
// all below 448 x 2^VALUE_EXP_MIN = 2^-39, is a factor of the rounded weights alone. So tokens with values of zero (e = -126) count in
// the sum: with e itself their 2^-e passes 32 bits, or their weights vanish beside those of larger values. The sum holds
// the tokens down to 2^-40 of the largest as long as no block has e above 35, values up to 2^43.
constexpr int VALUE_EXP_MIN = -48;

struct ValueScale {
    float e, inv, less;   // exponent, 2^-e, factor of the weights
};

__device__ __forceinline__ ValueScale value_scale(uint32_t byte)
{
    const int own = static_cast<int>(min(max(byte, 1u), 253u)) - 127, e = max(own, VALUE_EXP_MIN);
    return {static_cast<float>(e), __uint_as_float(static_cast<uint32_t>(127 - e) << 23),
            __uint_as_float(static_cast<uint32_t>(127 + own - e) << 23)};
}

struct AttendArgs {
    EvaKvCache c;
    EvaKvBatch b;
    const void* q;
    void* out;
    int64_t qt, qh;        // strides of q, elements
    int heads, group, window;
    float scale;           // times log2(e): the softmax's exponentials are powers of two
    int part_rows;         // rows of a partial sum (few rows: all that share a key)
    int4* heads_of;        // [pieces]: what a piece leaves unfinished (each kernel's own record)
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

// Bounded wait for bulk copies that have not arrived yet; sets EVA_STATUS_TIMEOUT where it gives up. The status word is the cache's and
// outlives the launch: a bit that is there already does not end the wait as in mbar_wait, but makes the limit 20 ms, a
// thousand times what a copy takes, so that a launch of many waves does not spend the whole limit in each.
static __device__ __noinline__ bool copies_late(uint64_t* bar, uint32_t parity, int* status)
{
    const uint64_t t0 = globaltimer();
    uint64_t limit = 0;
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 31) != 0) continue;
        if (limit == 0) limit = ld_volatile(status) & ST_TIMEOUT ? WAIT_LIMIT_NS / 100 : WAIT_LIMIT_NS;
        if (globaltimer() - t0 > limit) {
            atomicOr(status, ST_TIMEOUT);
            return false;
        }
    }
}

// Whether a warp's copies arrived (the whole warp asks and gets one answer). If not, the caller stores nothing that comes from them, waits
// once more for what it has in flight, and leaves.
__device__ __forceinline__ bool copies_arrived(uint64_t* bar, uint32_t parity, int* status)
{
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) ok = copies_late(bar, parity, status);
    return __all_sync(0xffffffffu, ok);
}

// Joins a row's partial sums, by a warp, eight at a time (their loads do not wait for one another): maximum at part(k)[im], sum at
// part(k)[is], output from part(k) + io; every lane gets the joint maximum and sum, and of the output dimensions
// 4 lane .. 4 lane + 3 (modulo DV).
template <int DV, typename P>
__device__ __forceinline__ void join_parts(const P& part, int parts, int im, int is, int64_t io, int lane, float& m, float& l, float (&o)[4])
{
    const int d = (lane * 4) % DV;
    m = -INFINITY;
    o[0] = o[1] = o[2] = o[3] = l = 0.0f;
    for (int k0 = 0; k0 < parts; k0 += 8) {
        float mk[8], lk[8];
        float2 x[8], y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in = k0 + k < parts;
            const float* q = part(in ? k0 + k : k0);
            mk[k] = in ? q[im] : -INFINITY;
            lk[k] = in ? q[is] : 0.0f;
            x[k] = in ? *reinterpret_cast<const float2*>(q + io + d) : make_float2(0.0f, 0.0f);
            y[k] = in ? *reinterpret_cast<const float2*>(q + io + d + 2) : make_float2(0.0f, 0.0f);
        }
        float now = m;
#pragma unroll
        for (int k = 0; k < 8; ++k) now = fmaxf(now, mk[k]);
        const float ref = now == -INFINITY ? 0.0f : now, fall = m == -INFINITY ? 1.0f : ex2(m - ref);   // (0, or NaN, so far)
        l *= fall;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] *= fall;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float w = mk[k] == -INFINITY ? 1.0f : ex2(mk[k] - ref);   // (nothing, or NaN)
            l = fmaf(lk[k], w, l);
            o[0] = fmaf(x[k].x, w, o[0]);
            o[1] = fmaf(x[k].y, w, o[1]);
            o[2] = fmaf(y[k].x, w, o[2]);
            o[3] = fmaf(y[k].y, w, o[3]);
        }
        m = now;
    }
}

// The row's output from what join_parts gives.
template <int DV, typename T> __device__ __forceinline__ void put_row(T* out, float l, const float (&o)[4], int lane)
{
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (lane * 4 < DV)
        *reinterpret_cast<uint2*>(out + lane * 4) = make_uint2(two_bits<T>(o[0] * inv, o[1] * inv), two_bits<T>(o[2] * inv, o[3] * inv));
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
