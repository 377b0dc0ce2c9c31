// Attention over the paged 8-bit cache on the tensor cores: many rows per sequence and key/value head (prompts).
//
// A CTA holds 256 rows (token, query head of the group) of one sequence and key/value head as two tiles of 128, and walks
// the sequence's tokens 128 at a time: S = Q K^T (tcgen05.mma, M 128, N 128), softmax, O += P V with P as the A
// operand in tensor memory. The two tiles alternate: while the tensor cores multiply for one, eight warps (a thread per row)
// do the softmax of the other. Tensor memory is full: two S of 128 columns (P, 16-bit, overwrites its own S) and two O.
//
// Four more warps turn the cache's codes into fp16 (exact) in the 128-byte swizzled layout, straight from global memory: a page's
// keys are rows of key_dim, its values rows of 64 tokens, so both are K-major operands without a transposition. Converting for
// two tiles at once halves that work. The scales stay outside, as in the decode kernel: a block's key scale multiplies its
// scores, its value scale 2^e goes into the exponent t = score + e, and out = sum 2^(t - M) code / sum 2^(t - M) 2^-e.
// M is raised (and O rescaled in tensor memory) only when a row's maximum has grown by more than 2^8: weights are fp16 up to
// 2^15, 2^7 at M, so that tokens down to 2^-21 of the largest keep 11 bits, and 2^-31 is the smallest.
//
// The (sequence, head, row block, token tile) units of a call form one line that is cut into equal pieces, one per SM, so
// causal rows of different lengths and ragged batches fill the GPU alike; row blocks cut between pieces leave fp32 partial
// sums that kv_prompt_combine joins in their order.
#include <algorithm>

#include "decode_tc.cuh"
#include "kv_attend.cuh"
#include "tc.cuh"

#include <cuda_fp8.h>

namespace eva {

constexpr int PR_TILE = 128, PR_ROWS = 2 * PR_TILE;       // rows of a tile, of a CTA; tokens of a step
constexpr int PR_CONV = 4, PR_WARPS = 8 + PR_CONV + 1;    // softmax, converter and MMA warps
constexpr float PR_BIAS = 7.0f, PR_SLACK = 8.0f;
constexpr int PR_SCALES = 4;                              // steps whose scales are kept

template <int DK, int DV> struct PrCfg {
    static constexpr int KC = DK / 64;                    // 64-element chunks of a query or key row
    static constexpr int CHUNK = PR_TILE * 128;           // 128 rows x 128 bytes
    static constexpr int VCHUNK = DV * 128;               // a page of values
    static constexpr int Q = 2 * KC * CHUNK, K = KC * CHUNK, V = 2 * VCHUNK;
    static constexpr int KST = DK == 192 ? 1 : 2, VST = 2;
    static constexpr int SMEM = Q + KST * K + VST * V + 1024;
};

struct PrBars {
    uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sready[2], pready[2], pvdone[2], qfull[2], scfull[PR_SCALES];
    uint32_t tmem;
};

// Row block qb of a sequence: its rows' tokens, the token range they see and the steps over it.
struct PrItem {
    int lo, hi, t0, tiles;
};

__device__ __forceinline__ PrItem pr_item(const KvSeq& s, int group, int window, int qb)
{
    const int rows = s.n * group, r0 = qb * PR_ROWS, r1 = min(r0 + PR_ROWS, rows) - 1;
    PrItem it;
    it.hi = max(s.ctx + r1 / group + 1, 0);
    it.lo = window > 0 ? max(0, s.ctx + r0 / group + 1 - window) : 0;
    it.t0 = it.lo / PR_TILE;
    it.tiles = it.hi > 0 ? (it.hi + PR_TILE - 1) / PR_TILE - it.t0 : 1;
    return it;
}

__device__ __forceinline__ int pr_blocks(const KvSeq& s, int group) { return (s.n * group + PR_ROWS - 1) / PR_ROWS; }

// Steps of one head of a sequence (whole warp).
__device__ __forceinline__ int64_t pr_units(const KvSeq& s, int group, int window)
{
    int64_t sum = 0;
    for (int qb = threadIdx.x & 31; qb < pr_blocks(s, group); qb += 32) sum += pr_item(s, group, window, qb).tiles;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

constexpr int PR_SPANS = 256;   // runs of sequences whose steps are summed in shared memory

// A piece of the line: where it begins and how many steps it has.
struct PrPlace {
    int b, h, qb, off;
    int64_t left, begin, total;
    int pieces;
};

// Consecutive steps of one row block within a piece.
struct PrSeg {
    int b, h, qb, t0, t1, after;   // steps t0 .. t1 - 1, `after` more in later pieces
    bool first;                    // holds the row block's first step
    PrItem item;
};

struct PrCursor {
    PrPlace at;
    KvSeq s;

    __device__ __forceinline__ bool next(const AttendArgs& p, PrSeg& g)
    {
        if (at.left <= 0) return false;
        g.b = at.b, g.h = at.h, g.qb = at.qb;
        g.item = pr_item(s, p.group, p.window, at.qb);
        const int have = g.item.tiles - at.off;
        const int take = static_cast<int>(min(static_cast<int64_t>(have), at.left));
        if (take <= 0) {   // lengths changed under the call
            at.left = 0;
            return false;
        }
        g.t0 = g.item.t0 + at.off;
        g.t1 = g.t0 + take;
        g.first = at.off == 0;
        g.after = have - take;
        at.left -= take;
        at.off = 0;
        if (at.left > 0 && ++at.qb == pr_blocks(s, p.group)) {
            at.qb = 0;
            if (++at.h == p.c.kv_heads) {
                at.h = 0;
                do {
                    if (++at.b >= p.b.seqs) {
                        at.left = 0;
                        break;
                    }
                    s = kv_seq(p.b, at.b, p.c.status);
                } while (s.n == 0);
            }
        }
        return true;
    }
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_st32f(uint32_t taddr, const float (&v)[32])
{
    uint32_t r[16];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[16 * k + i]);
        tmem_st16(taddr + 16 * k, r);
    }
}

// 16 codes (16 bytes) as two 16-byte units of halves
__device__ __forceinline__ void codes_to_halves(uint4 c, uint4& lo, uint4& hi)
{
    lo = make_uint4(e4m3_halves(c.x), e4m3_halves(c.x >> 16), e4m3_halves(c.y), e4m3_halves(c.y >> 16));
    hi = make_uint4(e4m3_halves(c.z), e4m3_halves(c.z >> 16), e4m3_halves(c.w), e4m3_halves(c.w >> 16));
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Byte offset of 16-byte unit u of row r in a 128-byte swizzled chunk
__device__ __forceinline__ uint32_t sw128(int r, int u) { return static_cast<uint32_t>(r * 128 + ((u ^ (r & 7)) << 4)); }

template <int DK, int DV, typename T>
__global__ void __launch_bounds__(PR_WARPS * 32, 1) kv_prompt_kernel(const AttendArgs p)
{
    using C = PrCfg<DK, DV>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PrBars B;
    __shared__ float4 scales[PR_SCALES][8];               // of a step's blocks: key scale, value exponent, 1 / value scale
    __shared__ unsigned long long spans[PR_SPANS];
    __shared__ PrPlace place;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* smem = align1024(smem_raw);
    const uint32_t sq = smem_u32(smem), sk = sq + C::Q, sv = sk + C::KST * C::K;
    int* const status = p.c.status;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.kfull[i], PR_CONV);
            mbar_init(&B.kempty[i], 1);
            mbar_init(&B.vfull[i], PR_CONV);
            mbar_init(&B.vempty[i], 1);
            mbar_init(&B.sready[i], 1);
            mbar_init(&B.pready[i], 4);
            mbar_init(&B.pvdone[i], 1);
            mbar_init(&B.qfull[i], 4);
        }
        for (int i = 0; i < PR_SCALES; ++i) mbar_init(&B.scfull[i], 1);
        fence_barrier_init();
    }
    if (warp == PR_WARPS - 1) tmem_alloc(&B.tmem, 512);
    for (int i = threadIdx.x; i < PR_SPANS; i += PR_WARPS * 32) spans[i] = 0;
    __syncthreads();
    // this CTA's piece of the line
    const int span = (p.b.seqs + PR_SPANS - 1) / PR_SPANS;
    for (int b = warp; b < p.b.seqs; b += PR_WARPS) {
        const int64_t u = pr_units(kv_seq(p.b, b, status), p.group, p.window);
        if (lane == 0 && u > 0) atomicAdd(&spans[b / span], static_cast<unsigned long long>(u));
    }
    __syncthreads();
    if (warp == 0) {
        int64_t total = 0;
        for (int i = lane; i < PR_SPANS; i += 32) total += static_cast<int64_t>(spans[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const int heads = p.c.kv_heads;
        total *= heads;
        PrPlace w{};
        w.total = total;
        w.pieces = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));
        const int c = blockIdx.x;
        if (c < w.pieces) {
            w.begin = total * c / w.pieces;
            w.left = total * (c + 1) / w.pieces - w.begin;
            int64_t rem = w.begin;
            int i = 0;
            while (i < PR_SPANS - 1 && rem >= static_cast<int64_t>(spans[i]) * heads) rem -= static_cast<int64_t>(spans[i++]) * heads;
            bool found = false;
            for (int b = i * span; b < min(p.b.seqs, (i + 1) * span) && !found; ++b) {
                const KvSeq s = kv_seq(p.b, b, status);
                const int64_t u = pr_units(s, p.group, p.window);
                if (rem >= u * heads) {
                    rem -= u * heads;
                    continue;
                }
                w.b = b;
                w.h = static_cast<int>(rem / u);
                rem -= w.h * u;
                for (int q0 = 0; q0 < pr_blocks(s, p.group); q0 += 32) {
                    int t = q0 + lane < pr_blocks(s, p.group) ? pr_item(s, p.group, p.window, q0 + lane).tiles : 0;
                    int64_t sum = t;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
                        if (lane >= o) sum += x;
                    }
                    const uint32_t hit = __ballot_sync(0xffffffffu, sum > rem);
                    if (hit) {
                        const int l = __ffs(hit) - 1;
                        w.qb = q0 + l;
                        w.off = static_cast<int>(rem - __shfl_sync(0xffffffffu, sum - t, l));
                        found = true;
                        break;
                    }
                    rem -= __shfl_sync(0xffffffffu, sum, 31);
                }
                break;
            }
            if (!found) w.left = 0;   // lengths changed under the call
        }
        if (lane == 0) place = w;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = B.tmem;
    PrCursor cur;
    cur.at = place;
    cur.s = cur.at.left > 0 ? kv_seq(p.b, cur.at.b, status) : KvSeq{0, 0, 0, 0};
    PrSeg g;

    if (warp < 8) {
        // ---- softmax: thread = row of tile `tile`
        const int tile = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + tile * PR_TILE, to = tmem + lanes + 2 * PR_TILE + tile * DV;
        uint32_t it = 0;                      // steps so far
        int4 head = make_int4(-1, 0, 0, 0);   // the row block that begins here and goes on in later pieces
        int64_t at = cur.at.begin;
        KvSeq s = cur.s;
        while (cur.next(p, g)) {
            const int r = g.qb * PR_ROWS + tile * PR_TILE + row, tok = r / p.group;
            const bool in = tok < s.n;
            const int64_t head_row = (static_cast<int64_t>(s.row0) + tok);
            const int qh = g.h * p.group + (r - tok * p.group);
            float c;
            {
                // the row, scaled by a power of two to [1, 2) at its largest, as fp16
                const T* q = static_cast<const T*>(p.q) + head_row * p.qt + static_cast<int64_t>(qh) * p.qh;
                float big = 0.0f;
                bool odd = false;
#pragma unroll 4
                for (int u = 0; u < DK / 8; ++u) {
                    const uint4 v = in ? *reinterpret_cast<const uint4*>(q + u * 8) : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = two_floats<T>(w[e]);
                        big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
                        odd |= f.x != f.x || f.y != f.y;
                    }
                }
                odd |= big == INFINITY;
                const int e2 = min(max(static_cast<int>(__float_as_uint(big) >> 23), 1), 252);
                const float down = __uint_as_float(static_cast<uint32_t>(254 - e2) << 23);
                c = odd ? __uint_as_float(0x7fc00000u) : p.scale * __uint_as_float(static_cast<uint32_t>(e2) << 23);
#pragma unroll 4
                for (int u = 0; u < DK / 8; ++u) {
                    const uint4 v = in ? *reinterpret_cast<const uint4*>(q + u * 8) : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    uint32_t o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = two_floats<T>(w[e]);
                        o[e] = half2_bits(f.x * down, f.y * down);
                    }
                    st_shared16(sq + (tile * C::KC + u / 8) * C::CHUNK + sw128(row, u % 8), make_uint4(o[0], o[1], o[2], o[3]));
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.qfull[tile]);
            }
            // rows without a token see nothing; rows behind the sequence are not written and need no mask
            const int hi = in ? s.ctx + tok + 1 : 0x7fffffff;
            const int lo = in && p.window > 0 ? hi - p.window : 0;
            const int all_hi = __reduce_min_sync(0xffffffffu, hi), all_lo = __reduce_max_sync(0xffffffffu, lo);
            float m = -INFINITY, l = 0.0f;
            for (int t = g.t0; t < g.t1; ++t, ++it) {
                const float4* sc = scales[it % PR_SCALES];
                const int tok0 = t * PR_TILE;
                const bool part = tok0 + PR_TILE > all_hi || tok0 < all_lo;
                mbar_wait(&B.scfull[it % PR_SCALES], (it / PR_SCALES) & 1, status);
                mbar_wait(&B.sready[tile], it & 1, status);
                tc_fence_after();
                float mx = -INFINITY;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float v[32];
                    tmem_ld32(ts + 32 * k, v);
                    if (part) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int tk = tok0 + 32 * k + i;
                            v[i] = tk >= lo && tk < hi ? v[i] : -INFINITY;
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float b = v[16 * x];
#pragma unroll
                        for (int i = 1; i < 16; ++i) b = fmaxf(b, v[16 * x + i]);
                        const float4 f = sc[2 * k + x];
                        mx = fmaxf(mx, fmaf(b, f.x * c, f.y));
                    }
                }
                const bool grow = mx > m + PR_SLACK || (m == -INFINITY && mx > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float down = grow ? ex2(m - mx) : 1.0f;
                    if (grow) m = mx;
                    l *= down;
                    if (t > g.t0) {
                        mbar_wait(&B.pvdone[tile], (it - 1) & 1, status);
                        tc_fence_after();
#pragma unroll 1
                        for (int k = 0; k < DV; k += 32) {
                            float v[32];
                            tmem_ld32(to + k, v);
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] *= down;
                            tmem_st32f(to + k, v);
                        }
                    }
                }
                const float ref = PR_BIAS - (m == -INFINITY ? 0.0f : m);
                // far from 0 the rounding of M must be the score's own, else their difference is not small at the largest
                const bool careful = part || __any_sync(0xffffffffu, m != -INFINITY && fabsf(m) > 4096.0f);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float v[32];
                    tmem_ld32(ts + 32 * k, v);
                    uint32_t w[16];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float4 f = sc[2 * k + x];
                        const float fc = f.x * c, add = f.y + ref;
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float a = fmaf(v[16 * x + i], fc, add), b = fmaf(v[16 * x + i + 1], fc, add);
                            if (careful) {
                                const int tk = tok0 + 32 * k + 16 * x + i;
                                a = fmaf(v[16 * x + i], fc, f.y) + ref;
                                b = fmaf(v[16 * x + i + 1], fc, f.y) + ref;
                                a = tk >= lo && tk < hi ? a : -INFINITY;
                                b = tk + 1 >= lo && tk + 1 < hi ? b : -INFINITY;
                            }
                            a = ex2(a);
                            b = ex2(b);
                            sum += a + b;
                            w[8 * x + i / 2] = half2_bits(a, b);
                        }
                        l = fmaf(sum, f.z, l);
                    }
                    tmem_st16(ts + 16 * k, w);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.pready[tile]);
            }
            // the row block's output, or its partial sums
            mbar_wait(&B.pvdone[tile], (it - 1) & 1, status);
            tc_fence_after();
            const bool whole = g.first && g.after == 0;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* out = static_cast<T*>(p.out) + (head_row * p.heads + qh) * DV;
            const int pr = tile * PR_TILE + row;
            float* part = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + (g.first ? 1 : 0)) * PR_ROWS * (DV + 2);
            if (!whole && in) {
                part[pr] = m;
                part[PR_ROWS + pr] = l;
            }
            float* po = part + 2 * PR_ROWS + static_cast<int64_t>(pr) * DV;
#pragma unroll 1
            for (int k = 0; k < DV; k += 32) {
                float v[32];
                __syncwarp();
                tmem_ld32(to + k, v);
                if (in && whole) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        *reinterpret_cast<uint4*>(out + k + i) =
                            make_uint4(two_bits<T>(v[i] * inv, v[i + 1] * inv), two_bits<T>(v[i + 2] * inv, v[i + 3] * inv),
                                       two_bits<T>(v[i + 4] * inv, v[i + 5] * inv), two_bits<T>(v[i + 6] * inv, v[i + 7] * inv));
                } else if (in) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(po + k + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            tc_fence_before();
            at += g.t1 - g.t0;
            if (g.first && g.after > 0)
                head = make_int4(g.b, g.h, g.qb, static_cast<int>(((at + g.after) * cur.at.pieces - 1) / cur.at.total));
            s = cur.s;
        }
        if (threadIdx.x == 0) p.heads_of[blockIdx.x] = head;
    } else if (warp < 8 + PR_CONV) {
        // ---- converters: 64-byte quarters of 8 rows per warp and load
        const int cw = warp - 8, unit = lane & 3, sub = cw * 8 + (lane >> 2);
        uint4 kr[DK / 64][4], vr[2][DV / 32];
        float4 mine = make_float4(1.0f, 0.0f, 1.0f, 0.0f);   // scales of block `lane` of the step (lanes 0 .. 7 of warp 8)
        int pages = -1, pages_at = -64, pages_b = -1;        // lane l: page pages_at + l of sequence pages_b
        KvSeq s = cur.s;
        bool more = cur.next(p, g);
        int t = more ? g.t0 : 0, pg[2] = {-1, -1}, len = s.len;

        // pages of step t
        auto find = [&]() {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int i = 2 * t + x;
                if (g.b != pages_b || i < pages_at || i >= pages_at + 32) {
                    pages_b = g.b;
                    pages_at = i;
                    const int want = i + lane;
                    pages = static_cast<int64_t>(want) * KV_PAGE < s.len ? kv_page(p.c, p.b, g.b, want, status) : -1;
                }
                pg[x] = __shfl_sync(0xffffffffu, pages, i - pages_at);
            }
        };
        auto load_k = [&]() {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r = sub + 32 * k, page = pg[k >> 1];   // row r: token r % 64 of page r / 64
                const uint8_t* src = static_cast<const uint8_t*>(p.c.k) +
                                     ((static_cast<int64_t>(max(page, 0)) * p.c.kv_heads + g.h) * KV_PAGE + (r & 63)) * DK + unit * 16;
#pragma unroll
                for (int ch = 0; ch < DK / 64; ++ch)
                    kr[ch][k] = page >= 0 ? *reinterpret_cast<const uint4*>(src + ch * 64) : make_uint4(0, 0, 0, 0);
            }
            if (cw == 0 && lane < 8) {
                const int page = pg[lane >> 2];
                mine = make_float4(1.0f, -INFINITY, 0.0f, 0.0f);   // no page: no weight
                if (page >= 0) {
                    const int64_t i = (static_cast<int64_t>(page) * p.c.kv_heads + g.h) * KV_PAGE_BLOCKS + (lane & 3);
                    const uint32_t ks = static_cast<const uint8_t*>(p.c.k_scale)[i];
                    const uint32_t vs = min(max(static_cast<uint32_t>(static_cast<const uint8_t*>(p.c.v_scale)[i]), 1u), 253u);
                    mine = make_float4(kv_scale(ks), static_cast<float>(static_cast<int>(vs) - 127),
                                       __uint_as_float((254u - vs) << 23), 0.0f);
                }
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint8_t* src = static_cast<const uint8_t*>(p.c.v) +
                                     ((static_cast<int64_t>(max(pg[x], 0)) * p.c.kv_heads + g.h) * DV + sub) * KV_PAGE + unit * 16;
#pragma unroll
                for (int k = 0; k < DV / 32; ++k)
                    vr[x][k] = pg[x] >= 0 ? *reinterpret_cast<const uint4*>(src + k * 32 * KV_PAGE) : make_uint4(0, 0, 0, 0);
                // behind the sequence's end a page may hold anything, NaN codes too, and 0 x NaN would count
                const int live = len - (2 * t + x) * KV_PAGE - unit * 16;
                if (live < 16) {
                    uint32_t keep[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int n = live - 4 * e;
                        keep[e] = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
                    }
#pragma unroll
                    for (int k = 0; k < DV / 32; ++k) {
                        vr[x][k].x &= keep[0];
                        vr[x][k].y &= keep[1];
                        vr[x][k].z &= keep[2];
                        vr[x][k].w &= keep[3];
                    }
                }
            }
        };
        if (more) {
            find();
            load_k();
            load_v();
        }
        for (uint32_t it = 0; more; ++it) {
            const uint32_t ks = it % C::KST, vs = it % C::VST;
            mbar_wait(&B.kempty[ks], ((it / C::KST) & 1) ^ 1, status);
#pragma unroll
            for (int ch = 0; ch < DK / 64; ++ch)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint4 a, b;
                    codes_to_halves(kr[ch][k], a, b);
                    const uint32_t dst = sk + ks * C::K + ch * C::CHUNK;
                    st_shared16(dst + sw128(sub + 32 * k, 2 * unit), a);
                    st_shared16(dst + sw128(sub + 32 * k, 2 * unit + 1), b);
                }
            if (cw == 0 && lane < 8) scales[it % PR_SCALES][lane] = mine;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.kfull[ks]);
            if (cw == 0 && lane == 0) mbar_arrive(&B.scfull[it % PR_SCALES]);
            if (++t == g.t1) {
                s = cur.s;
                more = cur.next(p, g);
                t = g.t0;
                len = s.len;
            }
            if (more) {
                find();
                load_k();
            }
            mbar_wait(&B.vempty[vs], ((it / C::VST) & 1) ^ 1, status);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int k = 0; k < DV / 32; ++k) {
                    uint4 a, b;
                    codes_to_halves(vr[x][k], a, b);
                    const uint32_t dst = sv + vs * C::V + x * C::VCHUNK;
                    st_shared16(dst + sw128(sub + 32 * k, 2 * unit), a);
                    st_shared16(dst + sw128(sub + 32 * k, 2 * unit + 1), b);
                }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.vfull[vs]);
            if (more) load_v();
        }
    } else if (lane == 0) {
        // ---- MMA issue
        constexpr uint32_t iqk = umma_idesc_f16(PR_TILE, PR_TILE), ipv = umma_idesc_f16(PR_TILE, DV);
        uint32_t it = 0, segs = 0;
        auto qk = [&](int tile, uint32_t n) {
            const uint32_t k0 = sk + (n % C::KST) * C::K, q0 = sq + tile * C::KC * C::CHUNK;
#pragma unroll
            for (int j = 0; j < DK / 16; ++j)
                umma_f16(tmem + tile * PR_TILE, umma_desc_sw128(q0 + (j >> 2) * C::CHUNK + (j & 3) * 32),
                         umma_desc_sw128(k0 + (j >> 2) * C::CHUNK + (j & 3) * 32), iqk, j > 0);
            umma_commit(&B.sready[tile]);
        };
        while (cur.next(p, g)) {
            const int n = g.t1 - g.t0;
            for (int tile = 0; tile < 2; ++tile) {
                mbar_wait(&B.qfull[tile], segs & 1, status);
                if (tile == 0) mbar_wait(&B.kfull[it % C::KST], (it / C::KST) & 1, status);
                tc_fence_after();
                qk(tile, it);
            }
            umma_commit(&B.kempty[it % C::KST]);
            for (int j = 0; j < n; ++j, ++it) {
                for (int tile = 0; tile < 2; ++tile) {
                    if (tile == 0) mbar_wait(&B.vfull[it % C::VST], (it / C::VST) & 1, status);
                    mbar_wait(&B.pready[tile], it & 1, status);
                    tc_fence_after();
                    const uint32_t v0 = sv + (it % C::VST) * C::V;
#pragma unroll
                    for (int k = 0; k < PR_TILE / 16; ++k)
                        umma_f16_ta(tmem + 2 * PR_TILE + tile * DV, tmem + tile * PR_TILE + k * 8,
                                    umma_desc_sw128(v0 + (k >> 2) * C::VCHUNK + (k & 3) * 32), ipv, j > 0 || k > 0);
                    umma_commit(&B.pvdone[tile]);
                    if (j + 1 < n) {
                        if (tile == 0) {
                            mbar_wait(&B.kfull[(it + 1) % C::KST], ((it + 1) / C::KST) & 1, status);
                            tc_fence_after();
                        }
                        qk(tile, it + 1);
                    }
                }
                umma_commit(&B.vempty[it % C::VST]);
                if (j + 1 < n) umma_commit(&B.kempty[(it + 1) % C::KST]);
            }
            ++segs;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == PR_WARPS - 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

constexpr int PR_COMBINE_ROWS = COMBINE_THREADS / 32;   // rows of a combining block, one per warp

// Joins the partial sums of the row block that begins in piece blockIdx.x and ends in a later one.
template <int DV, typename T>
__global__ void __launch_bounds__(COMBINE_THREADS) kv_prompt_combine(const AttendArgs p)
{
    const int g = blockIdx.x, lane = threadIdx.x & 31;
    const int4 head = p.heads_of[g];
    if (head.x < 0) return;
    const KvSeq s = kv_seq(p.b, head.x, p.c.status);
    const int pr = blockIdx.y * PR_COMBINE_ROWS + (threadIdx.x >> 5), r = head.z * PR_ROWS + pr, tok = r / p.group;
    if (tok >= s.n) return;
    const int step = PR_ROWS * (DV + 2), parts = head.w - g + 1;
    const float* base = p.part + static_cast<int64_t>(g) * 2 * step;
    auto part = [&](int k) { return base + (k == 0 ? step : static_cast<int64_t>(k) * 2 * step); };
    float m = -INFINITY;
    for (int k = lane; k < parts; k += 32) m = fmaxf(m, part(k)[pr]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ref = m == -INFINITY ? 0.0f : m;
    const int d = (lane * 4) % DV;
    float o[4] = {}, l = 0.0f;
    for (int k0 = 0; k0 < parts; k0 += 32) {
        float w = 0.0f;
        if (k0 + lane < parts) {
            w = ex2(part(k0 + lane)[pr] - ref);
            l = fmaf(part(k0 + lane)[PR_ROWS + pr], w, l);
        }
        const int n = min(32, parts - k0);
#pragma unroll 8
        for (int k = 0; k < n; ++k) {
            const float wk = __shfl_sync(0xffffffffu, w, k);
            const float4 v = *reinterpret_cast<const float4*>(part(k0 + k) + 2 * PR_ROWS + static_cast<int64_t>(pr) * DV + d);
            o[0] = fmaf(v.x, wk, o[0]);
            o[1] = fmaf(v.y, wk, o[1]);
            o[2] = fmaf(v.z, wk, o[2]);
            o[3] = fmaf(v.w, wk, o[3]);
        }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(p.out) + ((static_cast<int64_t>(s.row0) + tok) * p.heads + head.y * p.group + (r - tok * p.group)) * DV;
    if (lane * 4 < DV)
        *reinterpret_cast<uint2*>(out + d) = make_uint2(two_bits<T>(o[0] * inv, o[1] * inv), two_bits<T>(o[2] * inv, o[3] * inv));
}

template <int DK, int DV, typename T> static cudaError_t prompt_launch(const AttendArgs& p, cudaStream_t st)
{
    using C = PrCfg<DK, DV>;
    cudaError_t e = cudaFuncSetAttribute(kv_prompt_kernel<DK, DV, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    const int pieces = num_sms();
    kv_prompt_kernel<DK, DV, T><<<pieces, PR_WARPS * 32, C::SMEM, st>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    kv_prompt_combine<DV, T><<<dim3(pieces, PR_ROWS / PR_COMBINE_ROWS), COMBINE_THREADS, 0, st>>>(p);
    return cudaGetLastError();
}

size_t prompt_workspace(int dv)
{
    return num_sms() * (sizeof(int4) + 2 * sizeof(float) * PR_ROWS * (dv + 2));
}

cudaError_t launch_prompt(AttendArgs p, void* workspace, bool bf16, cudaStream_t st)
{
    p.part_rows = PR_ROWS;
    p.heads_of = static_cast<int4*>(workspace);
    p.part = reinterpret_cast<float*>(p.heads_of + num_sms());
    const int dk = p.c.key_dim;
    if (dk == 64) return bf16 ? prompt_launch<64, 64, __nv_bfloat16>(p, st) : prompt_launch<64, 64, __half>(p, st);
    if (dk == 128) return bf16 ? prompt_launch<128, 128, __nv_bfloat16>(p, st) : prompt_launch<128, 128, __half>(p, st);
    return bf16 ? prompt_launch<192, 128, __nv_bfloat16>(p, st) : prompt_launch<192, 128, __half>(p, st);
}

}  // namespace eva
