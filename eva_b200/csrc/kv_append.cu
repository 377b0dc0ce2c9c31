// Append to the paged 8-bit cache: rotation of the new keys, one power-of-two scale per 16 tokens and head, e4m3
// codes, in one kernel.
//
// A CTA owns one block (16 tokens of one sequence) and a warp one head at a time. It goes over the head's rows twice, for the
// maximum and for the codes. The rows come through shared memory, a bulk copy each (10 KB of 192 + 128 dimensions), so that all 16
// are in flight at once and cost no registers; the next head's keys follow while this head's values are packed. The
// cosines and sines of the block's tokens are computed once for all heads and kept in shared memory. The scale 2^e,
// e = ceil(log2(amax / 448)), comes from the exponent and mantissa bits of amax, and dividing by it is exact, so the only
// roundings are the rotation's (32 bits) and the one to e4m3. A block that already holds tokens keeps max(old e, new e); when that
// raises it, the older codes are multiplied by 2^(old - new), exact until they reach e4m3's subnormals.
//
// 18037 tokens of 7 prompts, 16 heads of 192 (64 rotated) + 128 fp16: 73 us, 278 MB at 3.8 TB/s, against 43 us of bytes alone.
// What bounds it is latency with few warps (16 an SM hold 160 KB of rows; issue is active half of the time): rotation, conversion and packing
// take some 100 instructions for each row of 320 elements. The grid is sequences x blocks of the longest one: 8192 tokens beside 255 single
// ones take 169 us in one call, 17 and 11 in two. Steps there: rows read twice from global memory, the second time from L1, 118 us;
// staged with 16-byte asynchronous copies 94; bulk copies, and loops of fixed length for whole blocks and without the rotation
// for the warp's units that have none, 79; the next head's copies ahead 73. (4 warps a CTA 72, 5 86, 16 slower; rows held in
// registers 10 to 20 % slower than 118.)
#include <type_traits>

#include "kv.cuh"
#include "kv_attend.cuh"

#include <cuda_fp8.h>

namespace eva {

constexpr int APPEND_WARPS = 8;

// How a lane's four key dimensions (two pairs) lie: side by side, as two neighbours in either half, or anywhere.
constexpr int KEYS_QUADS = 0, KEYS_HALVES = 1, KEYS_SINGLE = 2;

struct AppendArgs {
    EvaKvCache c;
    EvaKvBatch b;
    EvaRotary r;
    const void* k;
    const void* v;
    int64_t kt, kh, vt, vh;
    int blocks;   // blocks that one sequence's rows can touch
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

// exponent bits of an element that is not finite
template <typename T> constexpr uint32_t INF_BITS = 0;
template <> constexpr uint32_t INF_BITS<__nv_bfloat16> = 0x7f80u;
template <> constexpr uint32_t INF_BITS<__half> = 0x7c00u;

// Dimensions of pair i of a key: the rotated ones as the layout pairs them, the others as neighbours.
__device__ __forceinline__ int2 key_pair(const EvaRotary& r, int i)
{
    if (r.interleaved || r.dim == 0) return make_int2(2 * i, 2 * i + 1);
    if (i < r.dim / 2) return make_int2(r.offset + i, r.offset + i + r.dim / 2);
    const int d = 2 * (i - r.dim / 2), e = d < r.offset ? d : d + r.dim;
    return make_int2(e, e + 1);
}

// STAGED: a warp's 16 rows of keys and of values come through shared memory; rows of other alignments are read where they are
// used, 118 us for the prompts above.
template <typename T, int DK, int DV, int KEYS, bool STAGED>
__global__ void __launch_bounds__(APPEND_WARPS * 32, STAGED ? (DK == 64 ? 4 : DK == 128 ? 3 : 2) : 4) kv_append_kernel(AppendArgs p)
{
    extern __shared__ uint4 stage_raw[];
    constexpr int UNITS = DK / 4, KU = (UNITS + 31) / 32;   // four dimensions each; of a lane
    __shared__ alignas(8) uint64_t bars[APPEND_WARPS];
    __shared__ float4 turn[KV_BLOCK][UNITS];                // of a token and unit: cosines of both pairs, sines of both
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    if constexpr (STAGED) {
        if (lane == 0) {
            mbar_init(&bars[warp], 1);
            fence_barrier_init();
        }
        __syncwarp();
    }
    after_previous();
    const int b = blockIdx.x / p.blocks;
    const KvSeq s = kv_seq(p.b, b, p.c.status);
    const int first = max(s.ctx, 0);
    const int base = (first / KV_BLOCK + static_cast<int>(blockIdx.x - b * p.blocks)) * KV_BLOCK;
    if (s.n == 0 || base >= s.len) return;   // (a sequence without new rows may share its last page with one that appends)
    const int page = kv_page(p.c, p.b, b, base / KV_PAGE, p.c.status);
    if (page < 0) return;
    const int lo = max(first - base, 0), hi = min(s.len - base, KV_BLOCK), at = base % KV_PAGE;
    const int64_t tok0 = static_cast<int64_t>(s.row0) + base - s.ctx;   // token row of the block's slot 0
    // A head's rows on their way to shared memory, a bulk copy each, in flight while the angles, or the head before, are worked on
    T* const staged_k = reinterpret_cast<T*>(stage_raw + warp * (KV_BLOCK * (DK + DV) / 8));
    T* const staged_v = staged_k + KV_BLOCK * DK;
    auto stage_keys = [&](int h) {   // and announces the values
        __syncwarp();                // every lane is done with the keys before
        if (lane == 0) mbar_arrive_expect_tx(&bars[warp], (hi - lo) * (DK + DV) * sizeof(T));
        __syncwarp();
        if (lane >= lo && lane < hi)
            bulk_g2s(staged_k + lane * DK, static_cast<const T*>(p.k) + h * p.kh + (tok0 + lane) * p.kt, DK * sizeof(T), &bars[warp]);
    };
    auto stage_values = [&](int h) {
        __syncwarp();
        if (lane >= lo && lane < hi)
            bulk_g2s(staged_v + lane * DV, static_cast<const T*>(p.v) + h * p.vh + (tok0 + lane) * p.vt, DV * sizeof(T), &bars[warp]);
    };
    if constexpr (STAGED) {
        stage_keys(warp);
        stage_values(warp);
    }
    const bool rotates = p.r.dim > 0;
    if (rotates) {
        for (int i = threadIdx.x; i < (hi - lo) * UNITS; i += blockDim.x) {
            const int r = lo + i / UNITS, u = i % UNITS;
            float c[2], sn[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int pair = 2 * u + k, f = p.r.interleaved ? pair - p.r.offset / 2 : pair;   // its frequency
                c[k] = 1.0f;
                sn[k] = 0.0f;
                if (f >= 0 && f < p.r.dim / 2) {
                    sincospif(kv_half_turns(base + r, p.r.turns[f]), &sn[k], &c[k]);
                    c[k] *= p.r.mscale;
                    sn[k] *= p.r.mscale;
                }
            }
            turn[r][u] = make_float4(c[0], c[1], sn[0], sn[1]);
        }
        __syncthreads();
    }
    // The lane's units; lanes with none repeat the last one, which changes no maximum and spares the loads a branch, and do not store.
    int unit[KU], da[KU][2], db[KU][2];   // KEYS_SINGLE: the unit's dimensions; else da[.][0], db[.][0] begin its two neighbours
    bool has[KU], spins[KU];              // a unit of the warp is rotated
#pragma unroll
    for (int m = 0; m < KU; ++m) {
        has[m] = lane + 32 * m < UNITS;
        unit[m] = min(lane + 32 * m, UNITS - 1);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int2 d = key_pair(p.r, 2 * unit[m] + k);
            da[m][k] = d.x;
            db[m][k] = d.y;
        }
        const int f = 2 * unit[m] - (p.r.interleaved ? p.r.offset / 2 : 0);   // frequency of its first pair
        spins[m] = __any_sync(0xffffffffu, f + 1 >= 0 && f < p.r.dim / 2);
    }
    const bool vlane = 4 * lane < DV;
    const int slot0 = lo, slot1 = hi;
    uint32_t phase = 0;
    // WHOLE: the call fills the block, all loops are of 16
    auto one_head = [&](auto whole, const int h) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int lo = WHOLE ? 0 : slot0, hi = WHOLE ? KV_BLOCK : slot1;
        const int64_t ph = static_cast<int64_t>(page) * p.c.kv_heads + h;
        uint8_t* ks = static_cast<uint8_t*>(p.c.k_scale) + ph * KV_PAGE_BLOCKS + at / KV_BLOCK;
        uint8_t* vs = static_cast<uint8_t*>(p.c.v_scale) + ph * KV_PAGE_BLOCKS + at / KV_BLOCK;
        uint8_t* kc = static_cast<uint8_t*>(p.c.k) + (ph * KV_PAGE + at) * DK;
        uint8_t* vc = static_cast<uint8_t*>(p.c.v) + ph * KV_PAGE * DV + at;
        int kbyte = 0, vbyte = 0;   // the scales of the tokens that the block holds already
        if (lo > 0) {
            kbyte = min(max(static_cast<int>(*ks), 1), 253);
            vbyte = min(max(static_cast<int>(*vs), 1), 253);
        }
        const T* kp = static_cast<const T*>(p.k) + h * p.kh + tok0 * p.kt;
        const T* vp = static_cast<const T*>(p.v) + h * p.vh + tok0 * p.vt;
        if constexpr (STAGED) {
            if (!copies_arrived(&bars[warp], phase, p.c.status)) {   // the block's older tokens stay as they were
                copies_late(&bars[warp], phase, p.c.status);
                return false;
            }
            phase ^= 1;
            kp = staged_k;
            vp = staged_v;
        }
        if (vlane) vp += 4 * lane;
        const int64_t kt = STAGED ? DK : p.kt, vt = STAGED ? DV : p.vt;
        // raw elements of token r: values of dimensions 4 lane .. 4 lane + 3; a key unit as (a0, a1), (b0, b1)
        auto values = [&](int r) {
            if constexpr (KEYS != KEYS_SINGLE) {
                return *reinterpret_cast<const uint2*>(vp + r * vt);
            } else {
                const uint16_t* q = reinterpret_cast<const uint16_t*>(vp + r * vt);
                return make_uint2(q[0] | static_cast<uint32_t>(q[1]) << 16, q[2] | static_cast<uint32_t>(q[3]) << 16);
            }
        };
        auto keys = [&](int r, int m) {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(kp + r * kt);
            if constexpr (KEYS == KEYS_QUADS) {   // a0 b0 a1 b1
                const uint2 x = *reinterpret_cast<const uint2*>(q + da[m][0]);
                return make_uint2(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.x, x.y, 0x7632));
            } else if constexpr (KEYS == KEYS_HALVES) {
                // rotated: neighbours (a0, a1) and (b0, b1); else (a0, b0) and (a1, b1)
                const bool turned = 2 * unit[m] < p.r.dim / 2;
                const uint32_t x = *reinterpret_cast<const uint32_t*>(q + da[m][0]);
                const uint32_t y = *reinterpret_cast<const uint32_t*>(q + (turned ? db[m][0] : da[m][1]));
                return turned ? make_uint2(x, y) : make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
            } else {
                return make_uint2(q[da[m][0]] | static_cast<uint32_t>(q[da[m][1]]) << 16, q[db[m][0]] | static_cast<uint32_t>(q[db[m][1]]) << 16);
            }
        };
        auto rotated = [&](uint2 w, int r, int m, float2& ya, float2& yb) {
            const float2 a = two_floats<T>(w.x), c = two_floats<T>(w.y);
            ya = a;
            yb = c;
            if (rotates) {
                const float4 t = turn[r][unit[m]];
                const float2 cs = make_float2(t.x, t.y), sn = make_float2(t.z, t.w);
                ya = fma2(c, make_float2(-sn.x, -sn.y), mul2(a, cs));
                yb = fma2(a, sn, mul2(c, cs));
            }
        };
        // largest magnitudes: of the raw elements as integers of 16 bits (NaN above infinity above all), of the rotated keys
        uint32_t vmax = 0, raw = 0, flat = 0;   // flat: of keys that are not rotated
        float kmax = 0.0f;
#pragma unroll 8
        for (int r = lo; r < hi; ++r) {
            const uint2 v = values(r);
            vmax = __vimax3_u16x2(vmax, v.x & 0x7fff7fffu, v.y & 0x7fff7fffu);
        }
#pragma unroll
        for (int m = 0; m < KU; ++m) {
            if (spins[m]) {
#pragma unroll 4
                for (int r = lo; r < hi; ++r) {
                    const uint2 w = keys(r, m);
                    float2 ya, yb;
                    rotated(w, r, m, ya, yb);
                    raw = __vimax3_u16x2(raw, w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
                    kmax = fmaxf(fmaxf(kmax, fmaxf(fabsf(ya.x), fabsf(ya.y))), fmaxf(fabsf(yb.x), fabsf(yb.y)));
                }
            } else {
#pragma unroll 8
                for (int r = lo; r < hi; ++r) {
                    const uint2 w = keys(r, m);
                    flat = __vimax3_u16x2(flat, w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
                }
            }
        }
        flat = max(flat & 0xffffu, flat >> 16);
        kmax = fmaxf(kmax, two_floats<T>(flat).x);
        vmax = max(vmax & 0xffffu, vmax >> 16);
        raw = max(max(raw & 0xffffu, raw >> 16), flat);
        // A token with an element that is not finite has no key of its own, and does not count for the key's scale; of its values the
        // finite ones stay. (A rotated key's overflow is an infinity in one of its pair at least, never a NaN: the products are
        // summed unrounded.)
        uint32_t bad = 0;
        auto finite_only = [&](uint32_t w) {
            if ((w & 0x7fffu) >= INF_BITS<T>) w &= 0xffff0000u;
            if ((w >> 16 & 0x7fffu) >= INF_BITS<T>) w &= 0xffffu;
            return w;
        };
        const bool odd = __any_sync(0xffffffffu, vmax >= INF_BITS<T> || raw >= INF_BITS<T> || !finite(kmax));
        if (odd) {
            vmax = 0;
            kmax = 0.0f;
#pragma unroll 1
            for (int r = lo; r < hi; ++r) {
                const uint2 v = values(r);
                const uint32_t x = finite_only(v.x), y = finite_only(v.y);
                bool strange = x != v.x || y != v.y;
                float top = 0.0f;
#pragma unroll
                for (int m = 0; m < KU; ++m) {
                    float2 ya, yb;
                    rotated(keys(r, m), r, m, ya, yb);
                    strange |= !finite(ya.x) || !finite(ya.y) || !finite(yb.x) || !finite(yb.y);
                    top = fmaxf(fmaxf(top, fmaxf(fabsf(ya.x), fabsf(ya.y))), fmaxf(fabsf(yb.x), fabsf(yb.y)));
                }
                vmax = max(max(vmax, max(x & 0x7fffu, x >> 16 & 0x7fffu)), max(y & 0x7fffu, y >> 16 & 0x7fffu));
                if (__any_sync(0xffffffffu, strange)) bad |= 1u << r;
                else kmax = fmaxf(kmax, top);
            }
        }
        const int ve = max(scale_byte(__float_as_uint(two_floats<T>(__reduce_max_sync(0xffffffffu, vmax)).x)), vbyte);
        const int ke = max(scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(kmax))), kbyte);
        const float vinv = inv_scale(ve), kinv = inv_scale(ke);
        if (lo > 0 && ke > kbyte) {   // the older keys: lo rows of DK bytes, contiguous
            const float m = kinv * kv_scale(kbyte);
            for (int i = lane; i < lo * DK / 2; i += 32) {
                uint16_t* q = reinterpret_cast<uint16_t*>(kc) + i;
                *q = static_cast<uint16_t>(e4m3_scaled(*q, m));
            }
        }
        auto put_key = [&](float2 ya, float2 yb, int r, int m) {
            uint32_t x = e4m3x2(ya.x * kinv, ya.y * kinv), y = e4m3x2(yb.x * kinv, yb.y * kinv);   // (a0, a1), (b0, b1)
            if (!has[m]) return;
            uint8_t* q = kc + r * DK;
            if constexpr (KEYS == KEYS_SINGLE) {
                q[da[m][0]] = static_cast<uint8_t>(x);
                q[da[m][1]] = static_cast<uint8_t>(x >> 8);
                q[db[m][0]] = static_cast<uint8_t>(y);
                q[db[m][1]] = static_cast<uint8_t>(y >> 8);
            } else {
                const uint32_t w = __byte_perm(x, y, 0x5140);   // a0 b0 a1 b1
                if constexpr (KEYS == KEYS_QUADS) {
                    *reinterpret_cast<uint32_t*>(q + da[m][0]) = w;
                } else {
                    const bool turned = 2 * unit[m] < p.r.dim / 2;
                    *reinterpret_cast<uint16_t*>(q + da[m][0]) = static_cast<uint16_t>(turned ? x : w);
                    *reinterpret_cast<uint16_t*>(q + (turned ? db[m][0] : da[m][1])) = static_cast<uint16_t>(turned ? y : w >> 16);
                }
            }
        };
#pragma unroll
        for (int m = 0; m < KU; ++m) {
            if (spins[m]) {
#pragma unroll 4
                for (int r = lo; r < hi; ++r) {
                    float2 ya, yb;
                    rotated(keys(r, m), r, m, ya, yb);
                    put_key(ya, yb, r, m);
                }
            } else {
#pragma unroll 4
                for (int r = lo; r < hi; ++r) {
                    const uint2 w = keys(r, m);
                    put_key(two_floats<T>(w.x), two_floats<T>(w.y), r, m);
                }
            }
        }
        if (bad) {
            __syncwarp();   // (after the codes of these rows)
#pragma unroll 1
            for (int r = lo; r < hi; ++r)
                if (bad >> r & 1)
                    for (int i = lane; i < DK; i += 32) kc[r * DK + i] = 0x7f;
        }
        if constexpr (STAGED)
            if (h + nwarps < p.c.kv_heads) stage_keys(h + nwarps);
        // values: 16 tokens of a dimension are 16 bytes
        if (vlane) {
            const bool grown = lo > 0 && ve > vbyte, merge = !WHOLE && (lo > 0 || hi < KV_BLOCK);   // the block holds, or may hold, others' bytes
            const float moves = vinv * kv_scale(vbyte);
            uint32_t in[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint4 was = make_uint4(0, 0, 0, 0);
                if (merge) was = *reinterpret_cast<const uint4*>(vc + static_cast<int64_t>(4 * lane + j) * KV_PAGE);
                in[j][0] = was.x, in[j][1] = was.y, in[j][2] = was.z, in[j][3] = was.w;
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) {   // tokens 2 t, 2 t + 1
                const bool fresh0 = 2 * t >= lo && 2 * t < hi, fresh1 = 2 * t + 1 >= lo && 2 * t + 1 < hi;
                if (merge && !fresh0 && !fresh1 && !(grown && 2 * t < lo)) continue;
                uint2 v0 = fresh0 ? values(2 * t) : make_uint2(0, 0), v1 = fresh1 ? values(2 * t + 1) : make_uint2(0, 0);
                if (odd) {
                    v0 = make_uint2(finite_only(v0.x), finite_only(v0.y));
                    v1 = make_uint2(finite_only(v1.x), finite_only(v1.y));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 x = two_floats<T>(j < 2 ? v0.x : v0.y), y = two_floats<T>(j < 2 ? v1.x : v1.y);
                    uint32_t two = e4m3x2((j % 2 ? x.y : x.x) * vinv, (j % 2 ? y.y : y.x) * vinv);
                    if (merge) {
                        const uint32_t old = in[j][t / 2] >> (t % 2 * 16) & 0xffffu;
                        const uint32_t moved = grown ? e4m3_scaled(old, moves) : old;
                        const uint32_t a = 2 * t < lo ? moved : fresh0 ? two : old, c = 2 * t + 1 < lo ? moved : fresh1 ? two : old;
                        two = (a & 0xffu) | (c & 0xff00u);
                    }
                    in[j][t / 2] = t % 2 ? (in[j][t / 2] & 0xffffu) | two << 16 : (in[j][t / 2] & 0xffff0000u) | two;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint4*>(vc + static_cast<int64_t>(4 * lane + j) * KV_PAGE) = make_uint4(in[j][0], in[j][1], in[j][2], in[j][3]);
        }
        if constexpr (STAGED)
            if (h + nwarps < p.c.kv_heads) stage_values(h + nwarps);
        __syncwarp();   // every lane has read the old scales
        if (lane == 0) {
            *ks = static_cast<uint8_t>(ke);
            *vs = static_cast<uint8_t>(ve);
        }
        return true;
    };
    const bool fills = lo == 0 && hi == KV_BLOCK;
    for (int h = warp; h < p.c.kv_heads; h += nwarps)
        if (!(fills ? one_head(std::true_type{}, h) : one_head(std::false_type{}, h))) return;
}

template <typename T, int DK, int DV, int KEYS> static cudaError_t append_staged(const AppendArgs& p, unsigned grid, dim3 threads, cudaStream_t st)
{
    static std::atomic<uint64_t> done{0};
    constexpr int EACH = KV_BLOCK * (DK + DV) * sizeof(T);   // of a warp
    const auto kernel = &kv_append_kernel<T, DK, DV, KEYS, true>;
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), APPEND_WARPS * EACH, done);
    if (e != cudaSuccess) return e;
    return launch_after(*kernel, dim3(grid), threads, static_cast<size_t>(threads.x / 32 * EACH), st, p);
}

template <typename T, int DK, int DV> static cudaError_t append_launch(const AppendArgs& p, int keys, bool staged, unsigned grid, cudaStream_t st)
{
    const dim3 threads(32 * (p.c.kv_heads < APPEND_WARPS ? p.c.kv_heads : APPEND_WARPS));
    if (staged) return keys == KEYS_QUADS ? append_staged<T, DK, DV, KEYS_QUADS>(p, grid, threads, st) : append_staged<T, DK, DV, KEYS_HALVES>(p, grid, threads, st);
    if (keys == KEYS_QUADS) return launch_after(kv_append_kernel<T, DK, DV, KEYS_QUADS, false>, dim3(grid), threads, 0, st, p);
    if (keys == KEYS_HALVES) return launch_after(kv_append_kernel<T, DK, DV, KEYS_HALVES, false>, dim3(grid), threads, 0, st, p);
    return launch_after(kv_append_kernel<T, DK, DV, KEYS_SINGLE, false>, dim3(grid), threads, 0, st, p);
}

template <typename T> static cudaError_t append_typed(const AppendArgs& p, cudaStream_t st)
{
    const int64_t grid = static_cast<int64_t>(p.b.seqs) * p.blocks;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    // Four dimensions at a time where rows, heads and the rotation's halves lie on their boundaries, else one by one; staged where
    // every row begins on a bulk copy's 16 bytes (the prompts above: 73 us, 118 without).
    const uint64_t off = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                         static_cast<uint64_t>(p.kt | p.kh | p.vt | p.vh) * 2;
    const bool quads = p.r.interleaved || p.r.dim == 0;
    const int keys = off % 8 != 0 ? KEYS_SINGLE : quads ? KEYS_QUADS : p.r.dim % 4 == 0 ? KEYS_HALVES : KEYS_SINGLE;
    const bool staged = off % 16 == 0 && keys != KEYS_SINGLE;
    const unsigned g = static_cast<unsigned>(grid);
    if (p.c.key_dim == 64) return append_launch<T, 64, 64>(p, keys, staged, g, st);
    if (p.c.key_dim == 128) return append_launch<T, 128, 128>(p, keys, staged, g, st);
    return append_launch<T, 192, 128>(p, keys, staged, g, st);
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
    const int most = batch->max_q < batch->tokens ? batch->max_q : batch->tokens;   // rows of a sequence
    p.blocks = (most + KV_BLOCK - 2) / KV_BLOCK + 1;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == EVA_DTYPE_BF16 ? append_typed<__nv_bfloat16>(p, st) : append_typed<__half>(p, st);
    return e == cudaSuccess ? EVA_OK : EVA_ERR_CUDA;
}
