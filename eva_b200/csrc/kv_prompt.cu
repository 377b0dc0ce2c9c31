// Attention over the paged 8-bit cache on the tensor cores: many rows per sequence and key/value head (prompts).
//
// A CTA holds 256 rows (token, query head of the group) of one sequence and key/value head as two tiles of 128, and walks
// the sequence's tokens 128 at a time: S = Q K^T (tcgen05.mma, M 128, N 128), softmax, O += P V with P as the A
// operand in tensor memory. The two tiles alternate: while the tensor cores multiply for one, eight warps (a thread per row)
// do the softmax of the other. Tensor memory is full: two S of 128 columns (P, 16-bit, overwrites its own S) and two O.
//
// Bulk copies bring a page's codes as they are; four more warps turn them into fp16 (exact) in the 128-byte swizzled layout: a page's
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
// Four warpgroups: 8 softmax warps, 4 converter warps, the MMA warp (and three idle ones). Registers move to the
// softmax threads, which hold a row's 128 scores: 2 x 184 + 96 + 48 = 4 x 128, the launch's own.
constexpr int PR_CONV = 4, PR_MMA = 8 + PR_CONV, PR_WARPS = 16;
constexpr int PR_REGS_SOFTMAX = 184, PR_REGS_CONV = 96, PR_REGS_MMA = 48;
constexpr float PR_BIAS = 7.0f, PR_SLACK = 8.0f;
constexpr int PR_SCALES = 4, PR_SEGS = 4;                 // steps whose scales are kept, segments in flight

template <int DK, int DV> struct PrCfg {
    static constexpr int KC = DK / 64;                    // 64-element chunks of a query or key row
    static constexpr int CHUNK = PR_TILE * 128;           // 128 rows x 128 bytes
    static constexpr int VCHUNK = DV * 128;               // a page of values
    static constexpr int Q = 2 * KC * CHUNK, K = KC * CHUNK, V = 2 * VCHUNK;
    static constexpr int RK = 2 * KV_PAGE * DK, RV = 2 * KV_PAGE * DV;   // a step's codes as they are in the cache
    static constexpr int KST = DK == 192 ? 1 : 2, VST = DK == 192 ? 1 : 2;
    static constexpr int SMEM = Q + KST * K + VST * V + RK + RV + 1024;
    static_assert(SMEM <= 227 * 1024 - 1536, "shared memory");
};

struct PrBars {
    uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sready[2], pready[2], pvdone[2], qfull[2], scfull[PR_SCALES], segfull[PR_SEGS], segempty[PR_SEGS];
    uint64_t rkfull, rkempty, rvfull, rvempty;
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
    int b, h, qb, off, left, pieces;
    int64_t begin, total;
};


// Consecutive steps of one row block within a piece; t1 == 0 ends the piece.
struct PrSeg {
    int b, h, qb, t0, t1;          // steps t0 .. t1 - 1
    int first, after, done;        // holds the row block's first step; steps of it in later pieces; of the piece before
    KvSeq s;
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// One lane of the (whole) warp
__device__ __forceinline__ uint32_t elect_one()
{
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r;
}

__device__ __forceinline__ void umma_f16_if(uint32_t lead, uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
        "l"(da), "l"(db), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}

__device__ __forceinline__ void umma_f16_ta_if(uint32_t lead, uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc,
                                               uint32_t acc)
{
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
        "r"(tmem_a), "l"(db), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}

__device__ __forceinline__ void umma_commit_if(uint32_t lead, uint64_t* bar)
{
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)), "r"(lead)
        : "memory");
}

// 32 columns into r, valid after tmem_wait_ld() and tied()
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Keeps the uses of r[0 .. 31] behind this point
__device__ __forceinline__ void tied(uint32_t* r)
{
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

// Two 32-bit products and sums in one instruction
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float m, float c)
{
    asm("{\n .reg .b64 p, q, r;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %4};\n mov.b64 r, {%5, %5};\n"
        " fma.rn.f32x2 p, p, q, r;\n mov.b64 {%0, %1}, p;\n}\n"
        : "=f"(x), "=f"(y)
        : "f"(a), "f"(b), "f"(m), "f"(c));
}

__device__ __forceinline__ void add2(float& x, float& y, float a, float b)
{
    asm("{\n .reg .b64 p, q;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n add.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}\n"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}

// Largest t = score * scale + exponent over a step's scores r; with MASK over those that are seen (bit i of the words)
template <bool MASK>
__device__ __forceinline__ float pr_max(const uint32_t (&r)[128], const float4* sc, float c, int lo, int hi)
{
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        float b = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float v = __uint_as_float(r[16 * x + i]);
            b = fmaxf(b, !MASK || (16 * x + i >= lo && 16 * x + i < hi) ? v : -INFINITY);
        }
        mx = fmaxf(mx, fmaf(b, sc[x].x * c, sc[x].y));
    }
    return mx;
}

// Weights 2^(t + ref) of a step's scores as fp16 into tensor memory (over the scores); returns their sum, each divided
// by its value scale. CAREFUL: with the mask, and rounding t as pr_max did.
template <bool CAREFUL>
__device__ __forceinline__ float pr_weights(const uint32_t (&r)[128], const float4* sc, float c, float ref, int lo, int hi, uint32_t ts)
{
    float l = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t w[16];
#pragma unroll
        for (int x = 2 * k; x < 2 * k + 2; ++x) {
            const float4 f = sc[x];
            const float fc = f.x * c, add = f.y + ref;
            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
            for (int i = 16 * x; i < 16 * x + 16; i += 2) {
                float a = __uint_as_float(r[i]), b = __uint_as_float(r[i + 1]);
                if constexpr (CAREFUL) {
                    a = i >= lo && i < hi ? fmaf(a, fc, f.y) + ref : -INFINITY;
                    b = i + 1 >= lo && i + 1 < hi ? fmaf(b, fc, f.y) + ref : -INFINITY;
                } else {
                    fma2(a, b, a, b, fc, add);
                }
                a = ex2(a);
                b = ex2(b);
                add2(s0, s1, a, b);
                w[i / 2 - 16 * k] = half2_bits(a, b);
            }
            l = fmaf(s0 + s1, f.z, l);
        }
        tmem_st16(ts + 16 * k, w);
    }
    return l;
}

// 16 codes (16 bytes) as two 16-byte units of halves
__device__ __forceinline__ void codes_to_halves(uint4 c, uint4& lo, uint4& hi)
{
    lo = make_uint4(e4m3_halves(c.x), e4m3_halves(c.x >> 16), e4m3_halves(c.y), e4m3_halves(c.y >> 16));
    hi = make_uint4(e4m3_halves(c.z), e4m3_halves(c.z >> 16), e4m3_halves(c.w), e4m3_halves(c.w >> 16));
}

__device__ __forceinline__ uint4 ld_shared16(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
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
    __shared__ PrPlace place;
    __shared__ PrSeg segs[PR_SEGS];
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform for the compiler
    uint8_t* smem = align1024(smem_raw);
    const uint32_t sq = smem_u32(smem), sk = sq + C::Q, sv = sk + C::KST * C::K;
    uint8_t* const rawk = smem + C::Q + C::KST * C::K + C::VST * C::V;
    uint8_t* const rawv = rawk + C::RK;
    unsigned long long* const spans = reinterpret_cast<unsigned long long*>(smem);   // until the first query
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
        for (int i = 0; i < PR_SEGS; ++i) {
            mbar_init(&B.segfull[i], 1);
            mbar_init(&B.segempty[i], 8 + PR_CONV + 2);
        }
        mbar_init(&B.rkfull, 1);
        mbar_init(&B.rvfull, 1);
        mbar_init(&B.rkempty, PR_CONV);
        mbar_init(&B.rvempty, PR_CONV);
        fence_barrier_init();
    }
    if (warp == PR_MMA) tmem_alloc(&B.tmem, 512);
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
            w.left = static_cast<int>(total * (c + 1) / w.pieces - w.begin);
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
    // Segment i of the piece, for every lane of a warp (or the one thread that calls)
    auto segment = [&](uint32_t i) -> const PrSeg& {
        mbar_wait(&B.segfull[i % PR_SEGS], (i / PR_SEGS) & 1, status);
        return segs[i % PR_SEGS];
    };

    if (warp < 8) {
        // ---- softmax: thread = row of tile `tile`
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PR_REGS_SOFTMAX));
        const int tile = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + tile * PR_TILE, to = tmem + lanes + 2 * PR_TILE + tile * DV;
        uint32_t it = 0, seg = 0;             // steps and segments so far
        uint4 raw[DK / 8];                    // the row's query
        int pos = 0, t0 = 0, t1 = 0;          // position of the row, -1 - pos where it is behind the sequence
        T* dst = nullptr;                     // its output, or partial sums
        bool in = false, whole = false;
        if (threadIdx.x == 0) p.heads_of[blockIdx.x] = make_int4(-1, 0, 0, 0);
        // takes the next segment's row up (its loads are under way when this returns)
        auto take = [&]() -> bool {
            const PrSeg& g = segment(seg);
            t0 = g.t0;
            t1 = g.t1;
            if (t1 == 0) return false;
            const int r = g.qb * PR_ROWS + tile * PR_TILE + row, tok = r / p.group, qh = g.h * p.group + (r - tok * p.group);
            in = tok < g.s.n;
            pos = g.s.ctx + tok;
            whole = g.first && g.after == 0;
            const int64_t qrow = static_cast<int64_t>(g.s.row0) + tok;
            if (whole)
                dst = static_cast<T*>(p.out) + (qrow * p.heads + qh) * DV;
            else
                dst = reinterpret_cast<T*>(p.part + (static_cast<int64_t>(blockIdx.x) * 2 + g.first) * PR_ROWS * (DV + 2));
            if (threadIdx.x == 0 && g.first && g.after > 0)
                p.heads_of[blockIdx.x] =
                    make_int4(g.b, g.h, g.qb,
                              static_cast<int>(((place.begin + g.done + (t1 - t0) + g.after) * place.pieces - 1) / place.total));
            const T* q = static_cast<const T*>(p.q) + qrow * p.qt + static_cast<int64_t>(qh) * p.qh;
#pragma unroll
            for (int u = 0; u < DK / 8; ++u) raw[u] = in ? *reinterpret_cast<const uint4*>(q + u * 8) : make_uint4(0, 0, 0, 0);
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.segempty[seg % PR_SEGS]);
            ++seg;
            return true;
        };
        float m = 0.0f, l = 0.0f;
        for (bool pending = false;; pending = true) {
            const bool was_whole = whole, was_in = in;
            T* const out = dst;
            const bool more = take();
            if (pending) {
                // the row block's output, or its partial sums, while the next query is on its way
                mbar_wait(&B.pvdone[tile], (it - 1) & 1, status);
                tc_fence_after();
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int pr = tile * PR_TILE + row;
                float* part = reinterpret_cast<float*>(out);
                if (!was_whole && was_in) {
                    part[pr] = m;
                    part[PR_ROWS + pr] = l;
                }
                float* po = part + 2 * PR_ROWS + pr * DV;
#pragma unroll 1
                for (int k = 0; k < DV; k += 32) {
                    float v[32];
                    __syncwarp();
                    tmem_ld32(to + k, v);
                    if (was_in && was_whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                            *reinterpret_cast<uint4*>(out + k + i) =
                                make_uint4(two_bits<T>(v[i] * inv, v[i + 1] * inv), two_bits<T>(v[i + 2] * inv, v[i + 3] * inv),
                                           two_bits<T>(v[i + 4] * inv, v[i + 5] * inv), two_bits<T>(v[i + 6] * inv, v[i + 7] * inv));
                    } else if (was_in) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<float4*>(po + k + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
                }
                tc_fence_before();
            }
            if (!more) break;
            // the row, scaled by a power of two to [1, 2) at its largest, as fp16
            float c, big = 0.0f;
            bool odd = false;
#pragma unroll
            for (int u = 0; u < DK / 8; ++u) {
                const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
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
#pragma unroll
            for (int u = 0; u < DK / 8; ++u) {
                const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
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
            // rows without a token see nothing; rows behind the sequence are not written and need no mask
            const int hi = in ? pos + 1 : 0x7fffffff, lo = in && p.window > 0 ? max(hi - p.window, 0) : 0;
            const int all_hi = __reduce_min_sync(0xffffffffu, hi), all_lo = __reduce_max_sync(0xffffffffu, lo);
            m = -INFINITY, l = 0.0f;
            const int first = t0;
            for (int t = t0; t < t1; ++t, ++it) {
                const float4* sc = scales[it % PR_SCALES];
                const int tok0 = t * PR_TILE;
                const bool part = tok0 + PR_TILE > all_hi || tok0 < all_lo;
                mbar_wait(&B.scfull[it % PR_SCALES], (it / PR_SCALES) & 1, status);
                mbar_wait(&B.sready[tile], it & 1, status);
                tc_fence_after();
                uint32_t v[128];
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_ld32_async(ts + 32 * k, v + 32 * k);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 4; ++k) tied(v + 32 * k);
                const float mx = part ? pr_max<true>(v, sc, c, lo - tok0, hi - tok0) : pr_max<false>(v, sc, c, 0, 0);
                const bool grow = mx > m + PR_SLACK || (m == -INFINITY && mx > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float fall = grow ? ex2(m - mx) : 1.0f;
                    if (grow) m = mx;
                    l *= fall;
                    if (t > first) {
                        mbar_wait(&B.pvdone[tile], (it - 1) & 1, status);
                        tc_fence_after();
#pragma unroll 1
                        for (int k = 0; k < DV; k += 16) {
                            uint32_t o[16];
                            tmem_ld32x32_x16(to + k, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fall);
                            tmem_st16(to + k, o);
                        }
                    }
                }
                const float ref = PR_BIAS - (m == -INFINITY ? 0.0f : m);
                // far from 0 the rounding of M must be the score's own, else their difference is not small at the largest
                const bool careful = part || __any_sync(0xffffffffu, m != -INFINITY && fabsf(m) > 4096.0f);
                l += careful ? pr_weights<true>(v, sc, c, ref, part ? lo - tok0 : 0, part ? hi - tok0 : PR_TILE, ts)
                             : pr_weights<false>(v, sc, c, ref, 0, 0, ts);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.pready[tile]);
            }
        }
    } else if (warp < 8 + PR_CONV) {
        // ---- converters: 64-byte quarters of 8 rows per warp and load
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PR_REGS_CONV));
        const int unit = lane & 3, sub = (warp - 8) * 8 + (lane >> 2);
        // Eight lanes read and write 128 bytes without a bank conflict where two rows of a quarter are 64 or 192 bytes apart;
        // rows of 128 bytes take the one half from the even and the other from the odd row.
        const int odd = DK == 128 ? sub & 1 : 0;
        const uint32_t u0 = sw128(sub, 2 * unit), u1 = sw128(sub, 2 * unit + 1);
        uint32_t it = 0;
        for (uint32_t seg = 0;; ++seg) {
            const PrSeg& g = segment(seg);
            const int t0 = g.t0, t1 = g.t1, len = g.s.len;
            if (t1 == 0) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.segempty[seg % PR_SEGS]);
            for (int t = t0; t < t1; ++t, ++it) {
                const uint32_t ks = it % C::KST, vs = it % C::VST;
                mbar_wait(&B.rkfull, it & 1, status);
                mbar_wait(&B.kempty[ks], ((it / C::KST) & 1) ^ 1, status);
#pragma unroll 1
                for (int ch = 0; ch < DK / 64; ++ch) {
                    const uint32_t src = smem_u32(rawk) + sub * DK + ((ch ^ odd) * 64 + unit * 16);
                    const uint32_t dst = sk + ks * C::K + (ch ^ odd) * C::CHUNK;
                    uint4 c[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) c[k] = ld_shared16(src + k * 32 * DK);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint4 a, b;
                        codes_to_halves(c[k], a, b);
                        st_shared16(dst + k * 32 * 128 + u0, a);
                        st_shared16(dst + k * 32 * 128 + u1, b);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&B.kfull[ks]);
                    mbar_arrive(&B.rkempty);
                }
                mbar_wait(&B.rvfull, it & 1, status);
                mbar_wait(&B.vempty[vs], ((it / C::VST) & 1) ^ 1, status);
#pragma unroll 1
                for (int x = 0; x < 2; ++x) {
                    const uint32_t src = smem_u32(rawv) + (x * DV + sub) * KV_PAGE + unit * 16;
                    const uint32_t dst = sv + vs * C::V + x * C::VCHUNK;
                    uint4 c[DV / 32];
#pragma unroll
                    for (int k = 0; k < DV / 32; ++k) c[k] = ld_shared16(src + k * 32 * KV_PAGE);
                    // behind the sequence's end a page may hold anything, NaN codes too, and 0 x NaN would count
                    const int live = len - (2 * t + x) * KV_PAGE - unit * 16;
                    if (__any_sync(0xffffffffu, live < 16)) {
                        uint32_t keep[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int n = live - 4 * e;
                            keep[e] = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
                        }
#pragma unroll
                        for (int k = 0; k < DV / 32; ++k) {
                            c[k].x &= keep[0];
                            c[k].y &= keep[1];
                            c[k].z &= keep[2];
                            c[k].w &= keep[3];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < DV / 32; ++k) {
                        uint4 a, b;
                        codes_to_halves(c[k], a, b);
                        st_shared16(dst + k * 32 * 128 + u0, a);
                        st_shared16(dst + k * 32 * 128 + u1, b);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&B.vfull[vs]);
                    mbar_arrive(&B.rvempty);
                }
            }
        }
    } else {
        // ---- MMA issue: a whole warp walks through, so that descriptors stay in uniform registers, and one lane issues
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PR_REGS_MMA));
        if (warp == PR_MMA) {
            const uint32_t lead = elect_one();
        constexpr uint32_t iqk = umma_idesc_f16(PR_TILE, PR_TILE), ipv = umma_idesc_f16(PR_TILE, DV);
        uint32_t it = 0, seg = 0;
        // Rolled loops: this warp runs each product once a step, and straight-line code would come from memory every time.
        auto qk = [&](int tile, uint32_t n) {
            uint64_t a = umma_desc_sw128(sq + tile * C::KC * C::CHUNK), b = umma_desc_sw128(sk + (n % C::KST) * C::K);
#pragma unroll 1
            for (int j = 0; j < DK / 16; ++j) {
                umma_f16_if(lead, tmem + tile * PR_TILE, a, b, iqk, j > 0);
                const uint32_t up = (j & 3) == 3 ? (C::CHUNK - 96) >> 4 : 2;   // 32 bytes on, or the next chunk
                a += up;
                b += up;
            }
            umma_commit_if(lead, &B.sready[tile]);
        };
        auto pv = [&](int tile, uint32_t n, bool add) {
            uint64_t b = umma_desc_sw128(sv + (n % C::VST) * C::V);
#pragma unroll 1
            for (int k = 0; k < PR_TILE / 16; ++k) {
                umma_f16_ta_if(lead, tmem + 2 * PR_TILE + tile * DV, tmem + tile * PR_TILE + k * 8, b, ipv, add || k > 0);
                b += (k & 3) == 3 ? (C::VCHUNK - 96) >> 4 : 2;
            }
            umma_commit_if(lead, &B.pvdone[tile]);
        };
        for (;; ++seg) {
            const PrSeg& g = segment(seg);
            const int n = g.t1 - g.t0;
            if (g.t1 == 0) break;
            __syncwarp();
            if (lead) mbar_arrive(&B.segempty[seg % PR_SEGS]);
            for (int tile = 0; tile < 2; ++tile) {
                mbar_wait(&B.qfull[tile], seg & 1, status);
                if (tile == 0) mbar_wait(&B.kfull[it % C::KST], (it / C::KST) & 1, status);
                tc_fence_after();
                qk(tile, it);
            }
            umma_commit_if(lead, &B.kempty[it % C::KST]);
            for (int j = 0; j < n; ++j, ++it) {
                for (int tile = 0; tile < 2; ++tile) {
                    if (tile == 0) mbar_wait(&B.vfull[it % C::VST], (it / C::VST) & 1, status);
                    mbar_wait(&B.pready[tile], it & 1, status);
                    tc_fence_after();
                    pv(tile, it, j > 0);
                    if (j + 1 < n) {
                        if (tile == 0) {
                            mbar_wait(&B.kfull[(it + 1) % C::KST], ((it + 1) / C::KST) & 1, status);
                            tc_fence_after();
                        }
                        qk(tile, it + 1);
                    }
                }
                umma_commit_if(lead, &B.vempty[it % C::VST]);
                if (j + 1 < n) umma_commit_if(lead, &B.kempty[(it + 1) % C::KST]);
            }
        }
        } else if (warp == PR_MMA + 2) {
            // ---- copies: a step's pages into shared memory as they are, and its blocks' scales
            int pages = -1, pages_at = -64, pages_b = -1;   // lane l: page pages_at + l of sequence pages_b
            uint32_t it = 0;
            float4 mine = make_float4(1.0f, -INFINITY, 0.0f, 0.0f);
            for (uint32_t seg = 0;; ++seg) {
                const PrSeg& g = segment(seg);
                const int b = g.b, h = g.h, t0 = g.t0, t1 = g.t1, len = g.s.len;
                if (t1 == 0) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.segempty[seg % PR_SEGS]);
                for (int t = t0; t < t1; ++t, ++it) {
                    int pg[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int i = 2 * t + x;
                        if (b != pages_b || i < pages_at || i >= pages_at + 32) {
                            pages_b = b;
                            pages_at = i;
                            const int want = i + lane;
                            pages = static_cast<int64_t>(want) * KV_PAGE < len ? kv_page(p.c, p.b, b, want, status) : -1;
                        }
                        pg[x] = __shfl_sync(0xffffffffu, pages, i - pages_at);
                    }
                    // a page that is not there: codes of zero and no weight
                    if (lane < 8) {
                        const int page = pg[lane >> 2];
                        mine = make_float4(1.0f, -INFINITY, 0.0f, 0.0f);
                        if (page >= 0) {
                            const int64_t i = (static_cast<int64_t>(page) * p.c.kv_heads + h) * KV_PAGE_BLOCKS + (lane & 3);
                            const uint32_t ks = static_cast<const uint8_t*>(p.c.k_scale)[i];
                            const uint32_t vs = min(max(static_cast<uint32_t>(static_cast<const uint8_t*>(p.c.v_scale)[i]), 1u), 253u);
                            mine = make_float4(kv_scale(ks), static_cast<float>(static_cast<int>(vs) - 127),
                                               __uint_as_float((254u - vs) << 23), 0.0f);
                        }
                    }
                    mbar_wait(&B.rkempty, (it & 1) ^ 1, status);
                    if (pg[0] < 0 || pg[1] < 0) {
                        for (int x = 0; x < 2; ++x)
                            if (pg[x] < 0)
                                for (int i = lane; i < KV_PAGE * DK / 16; i += 32)
                                    st_shared16(smem_u32(rawk) + x * KV_PAGE * DK + i * 16, make_uint4(0, 0, 0, 0));
                        __syncwarp();
                    }
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&B.rkfull, ((pg[0] >= 0) + (pg[1] >= 0)) * KV_PAGE * DK);
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            if (pg[x] >= 0)
                                bulk_g2s(rawk + x * KV_PAGE * DK,
                                         static_cast<const uint8_t*>(p.c.k) + (static_cast<int64_t>(pg[x]) * p.c.kv_heads + h) * KV_PAGE * DK,
                                         KV_PAGE * DK, &B.rkfull);
                    }
                    __syncwarp();
                    mbar_wait(&B.rvempty, (it & 1) ^ 1, status);
                    if (pg[0] < 0 || pg[1] < 0) {
                        for (int x = 0; x < 2; ++x)
                            if (pg[x] < 0)
                                for (int i = lane; i < KV_PAGE * DV / 16; i += 32)
                                    st_shared16(smem_u32(rawv) + x * KV_PAGE * DV + i * 16, make_uint4(0, 0, 0, 0));
                        __syncwarp();
                    }
                    if (lane < 8) scales[it % PR_SCALES][lane] = mine;
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&B.rvfull, ((pg[0] >= 0) + (pg[1] >= 0)) * KV_PAGE * DV);
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            if (pg[x] >= 0)
                                bulk_g2s(rawv + x * KV_PAGE * DV,
                                         static_cast<const uint8_t*>(p.c.v) + (static_cast<int64_t>(pg[x]) * p.c.kv_heads + h) * KV_PAGE * DV,
                                         KV_PAGE * DV, &B.rvfull);
                        mbar_arrive(&B.scfull[it % PR_SCALES]);
                    }
                    __syncwarp();
                }
            }
        } else if (warp == PR_MMA + 1 && lane == 0) {
            // ---- the segments of the piece
            int b = place.b, h = place.h, qb = place.qb, off = place.off, left = place.left, done = 0;
            KvSeq s = left > 0 ? kv_seq(p.b, b, status) : KvSeq{0, 0, 0, 0};
            for (uint32_t i = 0;; ++i) {
                mbar_wait(&B.segempty[i % PR_SEGS], ((i / PR_SEGS) & 1) ^ 1, status);
                PrSeg& g = segs[i % PR_SEGS];
                PrItem item{};
                int have = 0;
                if (left > 0) {
                    item = pr_item(s, p.group, p.window, qb);
                    have = item.tiles - off;
                }
                const int n = min(have, left);
                if (n <= 0) {   // the end (or lengths that changed under the call)
                    g.t0 = g.t1 = 0;
                    mbar_arrive(&B.segfull[i % PR_SEGS]);
                    break;
                }
                g.b = b, g.h = h, g.qb = qb, g.s = s, g.done = done;
                g.t0 = item.t0 + off;
                g.t1 = g.t0 + n;
                g.first = off == 0;
                g.after = have - n;
                mbar_arrive(&B.segfull[i % PR_SEGS]);
                left -= n;
                done += n;
                off = 0;
                if (left > 0 && ++qb == pr_blocks(s, p.group)) {
                    qb = 0;
                    if (++h == p.c.kv_heads) {
                        h = 0;
                        do {
                            if (++b >= p.b.seqs) {
                                left = 0;
                                break;
                            }
                            s = kv_seq(p.b, b, status);
                        } while (s.n == 0);
                    }
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == PR_MMA) {
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
