// Rotary positions: y = mscale * (a cos t - b sin t, b cos t + a sin t) over pairs of a head's dimensions.
//
// No tables of cosines: a frequency is held as a 64-bit fraction of a turn, and position x fraction modulo
// 2^64 (one integer product) is the exact angle modulo a turn at any position, so only the last 32 bits'
// conversion rounds (1e-7 of a radian). A thread takes one 16-byte unit of a head (for pairs (i, i + dim / 2)
// the two units that hold both halves), computes its pairs' cosines and sines once and applies them to
// `hc` heads. The traffic is one read and one write of x; the copied dimensions outside the rotated part
// go through the same threads, and are left out when x is rotated in place. 8192 x 32 heads of 192 bf16, 64 rotated: interleaved 42
// us, 201 MB at 4.8 TB/s of a copy's 6.5; half layout 59, each thread's angles serving four heads; bounded by loads, angles and stores in turn with 20 warps an SM (their registers hold
// eight units). One token: 9 us, the host's.
#include <algorithm>

#include "kv.cuh"

namespace eva {

constexpr int ROT_THREADS = 64;   // 256: 48.6 us for the case below, 128: 42; a block's loads, angles and stores follow one another

template <bool INTER> constexpr int ROT_HEADS = INTER ? 8 : 4;   // heads of a thread at most: eight units in flight

struct RotArgs {
    const void* x;
    void* out;
    const void* pos;
    const uint64_t* turns;
    int64_t xt, xh, ot, oh;
    int pos64, tokens, heads, head_dim, dim, offset, hc, nhc, units, copy, narrow;
    float mscale, sgn;
};

template <typename T> __device__ __forceinline__ float rot_up(T v);
template <> __device__ __forceinline__ float rot_up(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float rot_up(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float rot_up(float v) { return v; }
template <typename T> __device__ __forceinline__ T rot_down(float v);
template <> __device__ __forceinline__ __nv_bfloat16 rot_down(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half rot_down(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float rot_down(float v) { return v; }

template <typename T, int V> struct alignas(sizeof(T) * V) RotVec {
    T v[V];
};

// Units of a head, V elements each (half layout: a rotated unit is V elements of each half):
// [0, offset / V) copied, then the rotated ones, then the copied rest. V divides every part.
// Blocks an SM, 8192 x 32 heads of 192 bf16, the last 64 rotated: pairs of halves 59 us with ten, 63 with the registers that they would take;
// interleaved pairs 42 with those, 38.5 with ten. (All of 128 dimensions: 33 either way, 28.3 and 26.3.)
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(ROT_THREADS, INTER ? 1 : 10) rotary_kernel(RotArgs p)
{
    using Vec = RotVec<T, V>;
    constexpr int NP = INTER ? V / 2 : V, B = ROT_HEADS<INTER>;
    after_previous();
    // (token, group of heads, unit) of the thread; 32-bit divisions where they do
    const int64_t i = static_cast<int64_t>(blockIdx.x) * ROT_THREADS + threadIdx.x;
    int64_t row, tok;
    if (p.narrow) {
        row = static_cast<uint32_t>(i) / static_cast<uint32_t>(p.units);
        tok = static_cast<uint32_t>(row) / static_cast<uint32_t>(p.nhc);
    } else {
        row = i / p.units;
        tok = row / p.nhc;
    }
    if (tok >= p.tokens) return;
    const int u = static_cast<int>(i - row * p.units), h0 = static_cast<int>(row - tok * p.nhc) * p.hc, h1 = min(p.heads, h0 + p.hc);
    const T* x = static_cast<const T*>(p.x) + tok * p.xt;
    T* o = static_cast<T*>(p.out) + tok * p.ot;
    const int pre = p.copy ? p.offset / V : 0, nrot = (INTER ? p.dim : p.dim / 2) / V;
    const bool turns = u >= pre && u < pre + nrot;
    const int d = u < pre ? u * V : turns ? p.offset + (u - pre) * V : p.offset + p.dim + (u - pre - nrot) * V;
    const int half = p.dim / 2;
    // All of the thread's loads first, then its angles: a load is 1 us away, and so is the position. Copied and rotated units of a
    // warp take one path, so that their loads are under way together, and a thread with all B heads has no branch between them
    // (with a check of each head such a call took 76 us, not 45).
    Vec a[B], b[INTER ? 1 : B];
    const bool full = h1 - h0 == B;
    auto load = [&](int k) {
        a[k] = *reinterpret_cast<const Vec*>(x + (h0 + k) * p.xh + d);
        if constexpr (!INTER)
            if (turns) b[k] = *reinterpret_cast<const Vec*>(x + (h0 + k) * p.xh + d + half);
    };
    if (full) {
#pragma unroll
        for (int k = 0; k < B; ++k) load(k);
    } else {
#pragma unroll
        for (int k = 0; k < B; ++k)
            if (h0 + k < h1) load(k);
    }
    float c[NP], s[NP];
    if (turns) {
        const int64_t pos = p.pos64 ? static_cast<const int64_t*>(p.pos)[tok] : static_cast<const int32_t*>(p.pos)[tok];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            sincospif(kv_half_turns(pos, p.turns[(u - pre) * NP + j]), &s[j], &c[j]);
            c[j] *= p.mscale;
            s[j] *= p.sgn;
        }
    }
    auto store = [&](int k) {
        if (turns) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                T& lo = INTER ? a[k].v[2 * j] : a[k].v[j];
                T& hi = INTER ? a[k].v[2 * j + 1] : b[INTER ? 0 : k].v[j];
                const float e = rot_up(lo), f = rot_up(hi);
                lo = rot_down<T>(e * c[j] - f * s[j]);
                hi = rot_down<T>(f * c[j] + e * s[j]);
            }
            if constexpr (!INTER) *reinterpret_cast<Vec*>(o + (h0 + k) * p.oh + d + half) = b[k];
        }
        *reinterpret_cast<Vec*>(o + (h0 + k) * p.oh + d) = a[k];
    };
    if (full) {
#pragma unroll
        for (int k = 0; k < B; ++k) store(k);
    } else {
#pragma unroll
        for (int k = 0; k < B; ++k)
            if (h0 + k < h1) store(k);
    }
}

template <typename T, int V, bool INTER> static cudaError_t rotary_launch(RotArgs p, cudaStream_t st)
{
    const int nrot = (INTER ? p.dim : p.dim / 2) / V;
    p.units = nrot + (p.copy ? (p.head_dim - p.dim) / V : 0);
    if (p.units == 0) return cudaSuccess;
    // Heads of one thread (they share its cosines): as many as leave 16 warps for each SM.
    const int64_t all = static_cast<int64_t>(p.tokens) * p.heads * p.units, most = std::min(ROT_HEADS<INTER>, p.heads);
    p.hc = static_cast<int>(std::max<int64_t>(1, std::min(most, all / (num_sms() * 512))));
    p.nhc = (p.heads + p.hc - 1) / p.hc;
    const int64_t threads = static_cast<int64_t>(p.tokens) * p.nhc * p.units;
    const int64_t grid = (threads + ROT_THREADS - 1) / ROT_THREADS;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    p.narrow = grid * ROT_THREADS < int64_t{1} << 32;
    return launch_after(rotary_kernel<T, V, INTER>, dim3(static_cast<unsigned>(grid)), dim3(ROT_THREADS), 0, st, p);
}

template <typename T> static cudaError_t rotary_typed(const RotArgs& p, bool inter, cudaStream_t st)
{
    // Widest unit that divides every part, stride and address.
    uint64_t bits = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out);
    bits |= static_cast<uint64_t>(p.offset | (inter ? p.dim : p.dim / 2)) * sizeof(T);
    bits |= static_cast<uint64_t>(p.xt | p.xh | p.ot | p.oh) * sizeof(T);
    if (p.copy) bits |= static_cast<uint64_t>(p.head_dim) * sizeof(T);
    constexpr int W = 16 / sizeof(T);
    if (bits % 16 == 0) return inter ? rotary_launch<T, W, true>(p, st) : rotary_launch<T, W, false>(p, st);
    if (inter) {
        if (bits % (2 * sizeof(T)) == 0) return rotary_launch<T, 2, true>(p, st);
        return cudaErrorInvalidValue;   // pairs that are not aligned to their size
    }
    if (sizeof(T) == 2 && bits % 4 == 0) return rotary_launch<T, 2, false>(p, st);
    return rotary_launch<T, 1, false>(p, st);
}

bool rotary_ok(const EvaRotary* r, int head_dim)
{
    return r && r->dim >= 0 && r->dim % 2 == 0 && r->offset >= 0 && r->offset % 2 == 0 &&
           static_cast<int64_t>(r->offset) + r->dim <= head_dim && (r->dim == 0 || r->turns) &&
           (reinterpret_cast<uintptr_t>(r->turns) & 7) == 0;
}

}  // namespace eva

using namespace eva;

extern "C" int eva_rotary(const EvaRotary* rotary, const void* x, int32_t dtype, int32_t tokens, int32_t heads,
                          int32_t head_dim, int64_t x_token_stride, int64_t x_head_stride, const void* positions,
                          int32_t positions_i64, void* out, int64_t out_token_stride, int64_t out_head_stride,
                          void* stream)
{
    if (tokens < 0 || heads < 1 || head_dim < 1 || dtype < EVA_DTYPE_F16 || dtype > EVA_DTYPE_F32) return EVA_ERR_INVALID;
    if (!rotary_ok(rotary, head_dim)) return EVA_ERR_INVALID;
    if (tokens == 0) return EVA_OK;
    const uintptr_t es = dtype == EVA_DTYPE_F32 ? 4 : 2;
    if (!x || !out || !positions || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % es) ||
        (reinterpret_cast<uintptr_t>(positions) % (positions_i64 ? 8 : 4)))
        return EVA_ERR_INVALID;
    if (x == out && (x_token_stride != out_token_stride || x_head_stride != out_head_stride)) return EVA_ERR_INVALID;
    // interleaved pairs are moved as one: their addresses must be multiples of a pair
    if (rotary->interleaved && rotary->dim &&
        ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % (2 * es) ||
         (x_token_stride | x_head_stride | out_token_stride | out_head_stride) % 2 || (x != out && head_dim % 2)))
        return EVA_ERR_INVALID;
    RotArgs p{};
    p.x = x;
    p.out = out;
    p.pos = positions;
    p.turns = rotary->turns;
    p.xt = x_token_stride;
    p.xh = x_head_stride;
    p.ot = out_token_stride;
    p.oh = out_head_stride;
    p.pos64 = positions_i64 ? 1 : 0;
    p.tokens = tokens;
    p.heads = heads;
    p.head_dim = head_dim;
    p.dim = rotary->dim;
    p.offset = rotary->offset;
    p.copy = x != out;
    p.mscale = rotary->mscale;
    p.sgn = rotary->inverse ? -rotary->mscale : rotary->mscale;
    const bool inter = rotary->interleaved && rotary->dim;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == EVA_DTYPE_F32    ? rotary_typed<float>(p, inter, st)
                          : dtype == EVA_DTYPE_BF16 ? rotary_typed<__nv_bfloat16>(p, inter, st)
                                                    : rotary_typed<__half>(p, inter, st);
    return e == cudaSuccess ? EVA_OK : EVA_ERR_CUDA;
}
