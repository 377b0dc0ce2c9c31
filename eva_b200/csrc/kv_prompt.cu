// Attention over the paged 8-bit cache on the tensor cores: many rows per sequence and key/value head (prompts).
//
// A CTA holds 256 rows (token, query head of the group) of one sequence and key/value head as two tiles of 128, and walks
// the sequence's tokens a page (64) at a step: S = Q K^T (tcgen05.mma, M 128, N 64), softmax, O += P V with P as the A
// operand in tensor memory. A tile has two S (of even and odd steps; P, 16-bit, overwrites its own S), and four warps for each, a
// thread per row: scores run two steps ahead, and consecutive steps overlap but for the running maximum M, which
// the warps of one parity hand to those of the other. Tensor memory is full: four S of 64 columns and two O of value_dim.
//
// Bulk copies bring a page's codes as they are; four more warps turn them into fp16 (exact) in the 128-byte swizzled layout: a page's
// keys are rows of key_dim, its values rows of 64 tokens, so both are K-major operands without a transposition. Converting for
// two tiles at once halves that work. The scales stay outside, as in the decode kernel: a block's key scale multiplies its
// scores, its value scale 2^e goes into the exponent t = score + e, and out = sum 2^(t - M) code / sum 2^(t - M) 2^-e.
// M is raised (and O rescaled in tensor memory) only when a row's maximum has grown by more than 2^12: weights are fp16 up to 2^15,
// 2^3 at M, so that tokens down to 2^-17 of it keep 11 bits, and 2^-27 is the step below.
//
// The (sequence, head, row block, token step) units of a call form one line that is cut into pieces of equal cost, one per SM, so
// causal rows of different lengths and ragged batches fill the GPU alike; row blocks cut between pieces leave fp32 partial
// sums that kv_prompt_combine joins in their order.
//
// 8192 new tokens, 16 query heads on 4 of 128 + 128 dimensions: 355 us, 275 GFLOP at 775 TFLOP/s (0.46 of the 1679 that a library
// product reaches); three sequences of up to 700 tokens behind 20000, 16 heads of 192 + 128: 352 us, 730 TFLOP/s. What bounds
// it is one step's chain: scores, maximum, weights, their product take 1900 clocks of tensor core and 3200 of softmax for each tile
// and parity, of which two overlap, so 2550 a step; the tensor pipe is 39 % busy, exponentials 39 %, issue 51 %. Steps there
// (prompt, pieces): one S per tile and 128 tokens a step 835, 625 us; scores read from tensor memory once 646, 494; products issued from
// rolled loops (straight-line code that one warp runs once a step comes from memory every time) 579, 451; codes by bulk copies
// 570, 357; two S a tile 548, 351; parities with warps of their own 493, 358; row blocks weighed 355, 352. Slower: 128 tokens a step with
// a row's scores in registers, two threads a row, one pass with a maximum that lags.
#include <algorithm>

#include "decode_tc.cuh"
#include "kv_attend.cuh"
#include "tc.cuh"

namespace eva {

constexpr int PR_TILE = 128, PR_ROWS = 2 * PR_TILE;       // rows of a tile, of a CTA
constexpr int PR_STEP = KV_PAGE;                          // tokens of a step
// 16 softmax warps (for each tile four for the even and four for the odd steps), 4 converter warps, two that issue the
// MMAs, one each for the segments and the copies.
constexpr int PR_SOFT = 16, PR_CONV = 4, PR_MMA = PR_SOFT + PR_CONV, PR_WARPS = PR_MMA + 4;
constexpr float PR_BIAS = 3.0f, PR_SLACK = 12.0f;         // exponents of a weight at M, and by which it may pass M
constexpr int PR_BLOCK_COST = 6;                          // steps that a row block's beginning and end take
constexpr int PR_SCALES = 8, PR_SEGS = 4;                 // steps whose scales are kept, segments in flight

template <int DK, int DV> struct PrCfg {
    static constexpr int KC = DK / 64;                    // 64-element chunks of a query or key row
    static constexpr int QCHUNK = PR_TILE * 128, KCHUNK = PR_STEP * 128;   // rows x 128 bytes
    static constexpr int Q = 2 * KC * QCHUNK, K = KC * KCHUNK, V = DV * 128;
    static constexpr int RK = PR_STEP * DK, RV = PR_STEP * DV;   // a step's codes as they are in the cache
    static constexpr int KST = DK == 192 ? 2 : 3, VST = KST, RST = 2;   // stages
    static constexpr int SMEM = Q + KST * K + VST * V + RST * (RK + RV) + 1024;
};

struct PrBars {
    uint64_t kfull[3], kempty[3], vfull[3], vempty[3], rkfull[2], rkempty[2], rvfull[2], rvempty[2];
    uint64_t sready[2][2], pready[2][2], pvdone[2][2], qfull[2];   // [tile][step & 1]
    uint64_t mready[2][4][2];                                   // [tile][warp][step & 1]
    uint64_t scfull[PR_SCALES], segfull[PR_SEGS], segempty[PR_SEGS];
    uint64_t pair[2][4];                                        // [tile][warp]: both parities' warps are here
    uint64_t mmadone[2];                                        // [tile], of a CTA that gave up
    uint32_t tmem, copied_k, copied_v;                          // steps whose codes the copying warp has asked for
    int gave_up;
};

// mbar_wait that sleeps in the barrier unit for up to 100 us a try: many warps wait here at any time, and short tries would
// fill the queue to shared memory, exponentials and tensor memory that the others work through. The loop for a wait
// that is not over by then stays out of line. A wait of the CTA that gives up ends the others of that CTA, and no more: the status
// word is the cache's, and a bit that an earlier launch left in it says nothing of this one.
__device__ __forceinline__ bool try_wait_long(uint64_t* bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(100000)
        : "memory");
    return ok != 0;
}

__device__ __noinline__ bool wait_more(uint64_t* bar, uint32_t parity, int* gave_up, int* status, uint64_t limit)
{
    const uint64_t t0 = globaltimer();
    while (ld_volatile(gave_up) == 0) {
        if (try_wait_long(bar, parity)) return true;
        if (globaltimer() - t0 > limit) {
            *static_cast<volatile int*>(gave_up) = 1;
            atomicOr(status, ST_TIMEOUT);
        }
    }
    return false;
}

// Before a CTA that gave up leaves: what it has in flight, whatever the others do.
__device__ __noinline__ void wait_for_own(uint64_t* bar, uint32_t parity)
{
    const uint64_t t0 = globaltimer();
    while (!try_wait_long(bar, parity) && globaltimer() - t0 <= WAIT_LIMIT_NS) {}
}

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
    it.t0 = it.lo / PR_STEP;
    it.tiles = it.hi > 0 ? (it.hi + PR_STEP - 1) / PR_STEP - it.t0 : 1;
    return it;
}

__device__ __forceinline__ int pr_blocks(const KvSeq& s, int group) { return (s.n * group + PR_ROWS - 1) / PR_ROWS; }

// Cost of one head of a sequence in steps (whole warp): a row block counts its steps and, before them, PR_BLOCK_COST for the time
// its query, first scores and output take (15k clocks, against 2.5k of a step; without it the 8192 tokens above take 485 us, not 352).
__device__ __forceinline__ int64_t pr_units(const KvSeq& s, int group, int window)
{
    int64_t sum = 0;
    for (int qb = threadIdx.x & 31; qb < pr_blocks(s, group); qb += 32) sum += pr_item(s, group, window, qb).tiles + PR_BLOCK_COST;
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
    int first, after, end;         // holds the row block's first step; steps of it in later pieces; cost from the piece's begin to its end
    KvSeq s;
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r)
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

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Largest t = score * scale + exponent of a step's scores
__device__ __forceinline__ float pr_max(uint32_t ts, const float4* sc, float c)
{
    float mx = -INFINITY;
    uint32_t r[64];
    tmem_ld32_async(ts, r);
    tmem_ld32_async(ts + 32, r + 32);
    tmem_wait_ld();
    tied(r);
    tied(r + 32);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        float b = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i += 2) b = max3(b, __uint_as_float(r[16 * x + i]), __uint_as_float(r[16 * x + i + 1]));
        mx = fmaxf(mx, fmaf(b, sc[x].x * c, sc[x].y));
    }
    return mx;
}

// Weights 2^(t + ref) as fp16 into tensor memory (over the scores); returns their sum, each divided by its value scale.
__device__ __forceinline__ float pr_weights(uint32_t ts, const float4* sc, float c, float ref)
{
    float l = 0.0f;
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        uint32_t r[32], w[16];
        tmem_ld32_async(ts + 32 * k, r);
        tmem_wait_ld();
        tied(r);
        // A pair's exponentials are issued four pairs before their sum and rounding, which would wait for them.
        constexpr int AHEAD = 4;
        float4 f[2] = {sc[2 * k], sc[2 * k + 1]};
        float sum[2][2] = {};
#pragma unroll
        for (int i = 0; i < 16 + AHEAD; ++i) {
            if (i < 16) {
                float a, b;
                fma2(a, b, __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), f[i / 8].x * c, f[i / 8].y + ref);
                r[2 * i] = __float_as_uint(ex2(a));
                r[2 * i + 1] = __float_as_uint(ex2(b));
            }
            if (i >= AHEAD) {
                const int j = i - AHEAD;
                const float a = __uint_as_float(r[2 * j]), b = __uint_as_float(r[2 * j + 1]);
                add2(sum[j / 8][0], sum[j / 8][1], a, b);
                w[j] = half2_bits(a, b);
            }
        }
        l = fmaf(sum[0][0] + sum[0][1], f[0].z, l);
        l = fmaf(sum[1][0] + sum[1][1], f[1].z, l);
        tmem_st16(ts + 16 * k, w);
    }
    return l;
}

// The same two for a step of which a row sees tokens lo .. hi - 1 only, that has a block of very small values (value_scale), or whose
// scores lie far from 0, where M must be rounded as t is, else their difference is not small at the largest: 16 columns at a time, since this is seldom run and long code would
// come from memory.
__device__ __noinline__ float pr_max_masked(uint32_t ts, const float4* sc, float c, int lo, int hi)
{
    float mx = -INFINITY;
#pragma unroll 1
    for (int x = 0; x < 4; ++x) {
        uint32_t r[16];
        tmem_ld32x32_x16(ts + 16 * x, r);
        const float fc = sc[x].x * c, add = sc[x].y;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            mx = fmaxf(mx, 16 * x + i >= lo && 16 * x + i < hi ? fmaf(__uint_as_float(r[i]), fc, add) : -INFINITY);
    }
    return mx;
}

__device__ __noinline__ float pr_weights_masked(uint32_t ts, const float4* sc, float c, float ref, int lo, int hi)
{
    float l = 0.0f;
#pragma unroll 1
    for (int x = 0; x < 4; ++x) {
        uint32_t r[16], w[8];
        tmem_ld32x32_x16(ts + 16 * x, r);
        const float4 f = sc[x];
        const float fc = f.x * c, less = fabsf(f.w);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float a = 16 * x + i >= lo && 16 * x + i < hi ? ex2(fmaf(__uint_as_float(r[i]), fc, f.y) + ref) : 0.0f;
            const float b = 16 * x + i + 1 >= lo && 16 * x + i + 1 < hi ? ex2(fmaf(__uint_as_float(r[i + 1]), fc, f.y) + ref) : 0.0f;
            s += a + b;
            w[i / 2] = half2_bits(a * less, b * less);
        }
        l = fmaf(s, f.z, l);
        tmem_st32x32_x8(ts + 8 * x, w);
    }
    return l;
}

// A row's output so far, times fall
template <int DV> __device__ __noinline__ void pr_rescale(uint32_t to, float fall)
{
#pragma unroll 1
    for (int k = 0; k < DV; k += 32) {
        uint32_t o[32];
        tmem_ld32_async(to + k, o);
        tmem_wait_ld();
        tied(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fall);
        tmem_st16(to + k, o);
        tmem_st16(to + k + 16, o + 16);
    }
}

// 16 codes (16 bytes) as two 16-byte units of halves
__device__ __forceinline__ void codes_to_halves(uint4 c, uint4& lo, uint4& hi)
{
    e4m3_halves(c.x, lo.x, lo.y);
    e4m3_halves(c.y, lo.z, lo.w);
    e4m3_halves(c.z, hi.x, hi.y);
    e4m3_halves(c.w, hi.z, hi.w);
}

__device__ __forceinline__ uint4 ld_shared16(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// 16 bytes from global to shared memory, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Byte offset of 16-byte unit u of row r in a 128-byte swizzled chunk
__device__ __forceinline__ uint32_t sw128(int r, int u) { return static_cast<uint32_t>(r * 128 + ((u ^ (r & 7)) << 4)); }

template <int DK, int DV, typename T>
__global__ void __launch_bounds__(PR_WARPS * 32, 1) kv_prompt_kernel(AttendArgs p)
{
    using C = PrCfg<DK, DV>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PrBars B;
    __shared__ float4 scales[PR_SCALES][4];               // of a step's blocks: key scale, value exponent, 2^-exponent, -+ factor of the weights
    __shared__ PrPlace place;
    __shared__ PrSeg segs[PR_SEGS];
    __shared__ float qscale[2][PR_TILE];                  // of a row's query: its power of two times the call's scale
    __shared__ float top[2][PR_TILE];                     // the running M of a tile's rows
    __shared__ float2 sums[2][2][PR_TILE];                // [tile][step & 1]: M and sum of a row as its steps left them
    static_assert(C::SMEM + sizeof(B) + sizeof(scales) + sizeof(place) + sizeof(segs) + sizeof(qscale) + sizeof(top) + sizeof(sums) + 7 * 16 <=
                      227 * 1024,
                  "shared memory, each array at a multiple of 16");
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform for the compiler
    uint8_t* smem = align1024(smem_raw);
    const uint32_t sq = smem_u32(smem), sk = sq + C::Q, sv = sk + C::KST * C::K;
    uint8_t* const rawk = smem + C::Q + C::KST * C::K + C::VST * C::V;
    uint8_t* const rawv = rawk + C::RST * C::RK;
    unsigned long long* const spans = reinterpret_cast<unsigned long long*>(smem);   // until the first query
    int* const status = p.c.status;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 3; ++i) {
            mbar_init(&B.kfull[i], PR_CONV);
            mbar_init(&B.kempty[i], 2);
            mbar_init(&B.vfull[i], PR_CONV);
            mbar_init(&B.vempty[i], 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.rkfull[i], 1);
            mbar_init(&B.rvfull[i], 1);
            mbar_init(&B.rkempty[i], PR_CONV);
            mbar_init(&B.rvempty[i], PR_CONV);
            for (int j = 0; j < 2; ++j) {
                mbar_init(&B.sready[i][j], 1);
                mbar_init(&B.pready[i][j], 4);
                mbar_init(&B.pvdone[i][j], 1);
                for (int k = 0; k < 4; ++k) mbar_init(&B.mready[i][k][j], 1);
            }
            mbar_init(&B.qfull[i], 8);
            mbar_init(&B.mmadone[i], 1);
            for (int k = 0; k < 4; ++k) mbar_init(&B.pair[i][k], 2);
        }
        for (int i = 0; i < PR_SCALES; ++i) mbar_init(&B.scfull[i], 1);
        for (int i = 0; i < PR_SEGS; ++i) {
            mbar_init(&B.segfull[i], 1);
            mbar_init(&B.segempty[i], PR_SOFT + PR_CONV + 3);
        }
        B.gave_up = 0;
        fence_barrier_init();
    }
    if (warp == PR_MMA) tmem_alloc(&B.tmem, 512);
    for (int i = threadIdx.x; i < PR_SPANS; i += PR_WARPS * 32) spans[i] = 0;
    __syncthreads();
    after_previous();
    // this CTA's piece of the line
    const int span = (p.b.seqs + PR_SPANS - 1) / PR_SPANS;
    // a warp for each sequence's row blocks where there are few sequences, else a thread: 1000 sequences of one block 57 us, 88 by warps
    if (p.b.seqs < 64) {
        for (int b = warp; b < p.b.seqs; b += PR_WARPS) {
            const int64_t u = pr_units(kv_seq(p.b, b, status), p.group, p.window);
            if (lane == 0 && u > 0) atomicAdd(&spans[b / span], static_cast<unsigned long long>(u));
        }
    } else {
        for (int b = threadIdx.x; b < p.b.seqs; b += PR_WARPS * 32) {
            const KvSeq s = kv_seq(p.b, b, status);
            int64_t u = 0;
            for (int qb = 0; qb < pr_blocks(s, p.group); ++qb) u += pr_item(s, p.group, p.window, qb).tiles + PR_BLOCK_COST;
            if (u > 0) atomicAdd(&spans[b / span], static_cast<unsigned long long>(u));
        }
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
                    int t = q0 + lane < pr_blocks(s, p.group) ? pr_item(s, p.group, p.window, q0 + lane).tiles + PR_BLOCK_COST : 0;
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
    // ok: no wait of the thread has given up. What a wait was for is garbage then, but harmless: warps vote on ok once a step, before
    // anything leaves the CTA, and end.
    bool ok = true;
    auto wait_on = [&](uint64_t* bar, uint32_t parity) {
        if (!try_wait_long(bar, parity)) ok &= wait_more(bar, parity, &B.gave_up, status, WAIT_LIMIT_NS);
    };
    auto all_ok = [&] { return __all_sync(0xffffffffu, ok) != 0; };
    // Segment i of the piece, for every lane of a warp
    auto segment = [&](uint32_t i) -> const PrSeg& {
        wait_on(&B.segfull[i % PR_SEGS], (i / PR_SEGS) & 1);
        return segs[i % PR_SEGS];
    };

    if (warp < PR_SOFT) {
        // ---- softmax: thread = row of tile `tile`, in the steps of one parity. A step's maximum joins the other parity's M of the
        // step before; all else of consecutive steps overlaps.
        const int tile = warp >> 3, odd_steps = (warp >> 2) & 1, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t ts = tmem + lanes + tile * PR_TILE + odd_steps * PR_STEP, to = tmem + lanes + 2 * PR_TILE + tile * DV;
        uint32_t it = 0, met = 0;             // steps so far; meetings with the other parity's warp
        auto meet = [&] {
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.pair[tile][quad]);
            wait_on(&B.pair[tile][quad], met++ & 1);
        };
        if (threadIdx.x == 0) p.heads_of[blockIdx.x] = make_int4(-1, 0, 0, 0);
        for (uint32_t seg = 0;; ++seg) {
            const PrSeg& g = segment(seg);
            const int t0 = g.t0, t1 = g.t1;
            if (!all_ok() || t1 == 0) break;
            const int qb = g.qb, h = g.h, rows = g.s.n, row0 = g.s.row0;
            const int r = qb * PR_ROWS + tile * PR_TILE + row, tok = r / p.group, qh = h * p.group + (r - tok * p.group);
            const bool in = tok < rows, whole = g.first && g.after == 0;
            const int64_t qrow = static_cast<int64_t>(g.s.row0) + tok;
            // rows without a token see nothing; rows behind the sequence are not written and need no mask
            const int hi = in ? g.s.ctx + tok + 1 : 0x7fffffff, lo = in && p.window > 0 ? max(hi - p.window, 0) : 0;
            // its output, or its piece's partial sums
            T* const out = static_cast<T*>(p.out) + (qrow * p.heads + qh) * DV;
            float* const part = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + g.first) * PR_ROWS * (DV + 2);
            if (threadIdx.x == 0 && g.first && g.after > 0)
                p.heads_of[blockIdx.x] =
                    make_int4(g.b, g.h, g.qb,
                              static_cast<int>(((place.begin + g.end) * place.pieces - 1) / place.total));
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.segempty[seg % PR_SEGS]);
            // The 32 rows (16 by each parity's warp), each scaled by a power of two to [1, 2) at its largest, as fp16: eight lanes a row, so that copies and
            // stores take whole 128-byte lines, four rows at a time; first as they are to their places, then scaled there.
            {
                const int l8 = lane & 7, sub4 = quad * 32 + (lane >> 3);
                const uint32_t dst = sq + tile * C::KC * C::QCHUNK;
#pragma unroll 1
                for (int x = 16 * odd_steps; x < 16 * odd_steps + 16; x += 4) {
                    const int r4 = qb * PR_ROWS + tile * PR_TILE + sub4 + x, tok4 = r4 / p.group;
                    const T* q = static_cast<const T*>(p.q) + (static_cast<int64_t>(row0) + tok4) * p.qt +
                                 (static_cast<int64_t>(h) * p.group + (r4 - tok4 * p.group)) * p.qh + l8 * 8;
#pragma unroll
                    for (int j = 0; j < C::KC; ++j) copy16(dst + j * C::QCHUNK + sw128(sub4 + x, l8), tok4 < rows ? q + j * 64 : p.q, tok4 < rows);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
#pragma unroll 1
                for (int x = 16 * odd_steps; x < 16 * odd_steps + 16; x += 4) {
                    uint4 raw[C::KC];
                    float big = 0.0f;
                    bool odd = false;
#pragma unroll
                    for (int j = 0; j < C::KC; ++j) raw[j] = ld_shared16(dst + j * C::QCHUNK + sw128(sub4 + x, l8));
#pragma unroll
                    for (int j = 0; j < C::KC; ++j) {
                        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = two_floats<T>(w[e]);
                            big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
                            odd |= f.x != f.x || f.y != f.y;
                        }
                    }
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                    odd = (__ballot_sync(0xffffffffu, odd) >> (lane & 24) & 0xffu) != 0 || big == INFINITY;
                    const int e2 = min(max(static_cast<int>(__float_as_uint(big) >> 23), 1), 252);
                    const float down = __uint_as_float(static_cast<uint32_t>(254 - e2) << 23);
                    if (l8 == 0)
                        qscale[tile][sub4 + x] = odd ? __uint_as_float(0x7fc00000u) : p.scale * __uint_as_float(static_cast<uint32_t>(e2) << 23);
#pragma unroll
                    for (int j = 0; j < C::KC; ++j) {
                        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
                        uint32_t o[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = two_floats<T>(w[e]);
                            o[e] = half2_bits(f.x * down, f.y * down);
                        }
                        st_shared16(dst + j * C::QCHUNK + sw128(sub4 + x, l8), make_uint4(o[0], o[1], o[2], o[3]));
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.qfull[tile]);
            }
            meet();
            const float c = qscale[tile][row];
            const int all_hi = __reduce_min_sync(0xffffffffu, hi), all_lo = __reduce_max_sync(0xffffffffu, lo);
            const uint32_t first = it, end = it + (t1 - t0);
            float m = -INFINITY, l = 0.0f;
#pragma unroll 1
            for (it += (it ^ odd_steps) & 1; it < end; it += 2) {
                const float4* sc = scales[it % PR_SCALES];
                const int tok0 = (t0 + static_cast<int>(it - first)) * PR_STEP;
                const bool part_seen = tok0 + PR_STEP > all_hi || tok0 < all_lo;
                wait_on(&B.scfull[it % PR_SCALES], (it / PR_SCALES) & 1);
                wait_on(&B.sready[tile][odd_steps], (it >> 1) & 1);
                tc_fence_after();
                const float mx = part_seen ? pr_max_masked(ts, sc, c, lo - tok0, hi - tok0) : pr_max(ts, sc, c);
                float was = -INFINITY;
                if (it > first) {
                    wait_on(&B.mready[tile][quad][odd_steps ^ 1], ((it - 1) >> 1) & 1);
                    was = top[tile][row];
                }
                const bool grow = mx > was + PR_SLACK || (was == -INFINITY && mx > was);
                const float now = grow ? mx : was;
                top[tile][row] = now;
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.mready[tile][quad][odd_steps]);
                if (it > first && __any_sync(0xffffffffu, grow)) {
                    const float fall = grow ? ex2(was - now) : 1.0f;
                    wait_on(&B.pvdone[tile][odd_steps ^ 1], ((it - 1) >> 1) & 1);
                    tc_fence_after();
                    pr_rescale<DV>(to, fall);
                }
                if (m != now) l *= m == -INFINITY ? 1.0f : ex2(m - now);   // (a sum that is not 0 there is NaN, and stays it)
                m = now;
                const float ref = PR_BIAS - (m == -INFINITY ? 0.0f : m);
                if (!part_seen && sc[0].w > 0.0f && !__any_sync(0xffffffffu, m != -INFINITY && fabsf(m) > 4096.0f))
                    l += pr_weights(ts, sc, c, ref);
                else
                    l += pr_weights_masked(ts, sc, c, ref, lo - tok0, hi - tok0);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.pready[tile][odd_steps]);
                if (!all_ok()) break;
            }
            it = end;
            // both parities' sums, then half of the output each
            sums[tile][odd_steps][row] = make_float2(m, l);
            meet();
            const float2 s0 = sums[tile][0][row], s1 = sums[tile][1][row];
            m = fmaxf(s0.x, s1.x);
            l = s0.y * (s0.x == -INFINITY ? 1.0f : ex2(s0.x - m)) + s1.y * (s1.x == -INFINITY ? 1.0f : ex2(s1.x - m));
            wait_on(&B.pvdone[tile][(it - 1) & 1], ((it - 1) >> 1) & 1);
            tc_fence_after();
            if (!all_ok()) break;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int pr = tile * PR_TILE + row;
            if (!whole && in && odd_steps == 0) {
                part[pr] = m;
                part[PR_ROWS + pr] = l;
            }
#pragma unroll 1
            for (int k = odd_steps * (DV / 2); k < (odd_steps + 1) * (DV / 2); k += 16) {
                uint32_t v[16];
                __syncwarp();
                tmem_ld32x32_x16(to + k, v);
                if (in && whole) {
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = two_bits<T>(__uint_as_float(v[i + 2 * e]) * inv, __uint_as_float(v[i + 2 * e + 1]) * inv);
                        *reinterpret_cast<uint4*>(out + k + i) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else if (in) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<uint4*>(part + 2 * PR_ROWS + pr * DV + k + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            tc_fence_before();
        }
    } else if (warp < PR_MMA) {
        // ---- converters: 64-byte quarters of 8 rows per warp and load
        const int unit = lane & 3, sub = (warp - PR_SOFT) * 8 + (lane >> 2);
        // Eight lanes read and write 128 bytes without a bank conflict where two rows of a quarter are 64 or 192 bytes apart;
        // rows of 128 bytes take the one half from the even and the other from the odd row.
        const int odd = DK == 128 ? sub & 1 : 0;
        const uint32_t u0 = sw128(sub, 2 * unit), u1 = sw128(sub, 2 * unit + 1);
        uint32_t it = 0;
        for (uint32_t seg = 0;; ++seg) {
            const PrSeg& g = segment(seg);
            const int t0 = g.t0, t1 = g.t1, len = g.s.len;
            if (!all_ok() || t1 == 0) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.segempty[seg % PR_SEGS]);
#pragma unroll 1
            for (int t = t0; t < t1; ++t, ++it) {
                const uint32_t ks = it % C::KST, vs = it % C::VST, rs = it % C::RST;
                wait_on(&B.rkfull[rs], (it / C::RST) & 1);
                wait_on(&B.kempty[ks], ((it / C::KST) & 1) ^ 1);
                {
                    const uint32_t src = smem_u32(rawk) + rs * C::RK + sub * DK + unit * 16, dst = sk + ks * C::K;
                    uint4 c[C::KC][2];
#pragma unroll
                    for (int ch = 0; ch < C::KC; ++ch)
#pragma unroll
                        for (int k = 0; k < 2; ++k) c[ch][k] = ld_shared16(src + (ch ^ odd) * 64 + k * 32 * DK);
#pragma unroll
                    for (int ch = 0; ch < C::KC; ++ch)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint4 a, b;
                            codes_to_halves(c[ch][k], a, b);
                            st_shared16(dst + (ch ^ odd) * C::KCHUNK + k * 32 * 128 + u0, a);
                            st_shared16(dst + (ch ^ odd) * C::KCHUNK + k * 32 * 128 + u1, b);
                        }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&B.kfull[ks]);
                    mbar_arrive(&B.rkempty[rs]);
                }
                wait_on(&B.rvfull[rs], (it / C::RST) & 1);
                wait_on(&B.vempty[vs], ((it / C::VST) & 1) ^ 1);
                {
                    const uint32_t src = smem_u32(rawv) + rs * C::RV + sub * KV_PAGE + unit * 16, dst = sv + vs * C::V;
                    uint4 c[DV / 32];
#pragma unroll
                    for (int k = 0; k < DV / 32; ++k) c[k] = ld_shared16(src + k * 32 * KV_PAGE);
                    // behind the sequence's end a page may hold anything, NaN codes too, and 0 x NaN would count
                    const int live = len - t * PR_STEP - unit * 16;
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
                    mbar_arrive(&B.rvempty[rs]);
                }
                if (!all_ok()) break;
            }
        }
    } else {
        if (warp == PR_MMA || warp == PR_MMA + 3) {
            // ---- MMA issue, a warp for each tile, so that the one's waits do not hold the other's products up. A whole warp walks
            // through, so that descriptors stay in uniform registers, and one lane issues. Loops stay rolled: each product is
            // issued once a step, and straight-line code would come from memory every time.
            constexpr uint32_t iqk = umma_idesc_f16(PR_TILE, PR_STEP), ipv = umma_idesc_f16(PR_TILE, DV);
            const uint32_t lead = elect_one();
            const int tile = warp == PR_MMA ? 0 : 1;
            const uint32_t ts = tmem + tile * PR_TILE, to = tmem + 2 * PR_TILE + tile * DV;
            const uint64_t dq = umma_desc_sw128(sq + tile * C::KC * C::QCHUNK);
            uint32_t it = 0;
            for (uint32_t seg = 0;; ++seg) {
                const PrSeg& g = segment(seg);
                const int n = g.t1 - g.t0;
                if (!all_ok() || g.t1 == 0) break;
                __syncwarp();
                if (lead) mbar_arrive(&B.segempty[seg % PR_SEGS]);
                wait_on(&B.qfull[tile], seg & 1);
                // scores run two steps ahead of the weights' products
                it -= 2;
#pragma unroll 1
                for (int j = -2; j < n; ++j, ++it) {
                    if (j >= 0) {
                        wait_on(&B.vfull[it % C::VST], (it / C::VST) & 1);
                        wait_on(&B.pready[tile][it & 1], (it >> 1) & 1);
                        tc_fence_after();
                        uint64_t b = umma_desc_sw128(sv + (it % C::VST) * C::V);
                        uint32_t a = ts + (it & 1) * PR_STEP;
#pragma unroll 1
                        for (int k = 0; k < PR_STEP / 16; ++k, a += 8, b += 2) umma_f16_ta_if(lead, to, a, b, ipv, j > 0 || k > 0);
                        umma_commit_if(lead, &B.pvdone[tile][it & 1]);
                        umma_commit_if(lead, &B.vempty[it % C::VST]);
                    }
                    if (j + 2 < n) {
                        const uint32_t ahead = it + 2, ks = ahead % C::KST;
                        wait_on(&B.kfull[ks], (ahead / C::KST) & 1);
                        tc_fence_after();
                        uint64_t a = dq, b = umma_desc_sw128(sk + ks * C::K);
#pragma unroll 1
                        for (int k = 0; k < DK / 16; ++k) {
                            umma_f16_if(lead, ts + (it & 1) * PR_STEP, a, b, iqk, k > 0);
                            a += (k & 3) == 3 ? (C::QCHUNK - 96) >> 4 : 2;   // 32 bytes on, or the next chunk
                            b += (k & 3) == 3 ? (C::KCHUNK - 96) >> 4 : 2;
                        }
                        umma_commit_if(lead, &B.sready[tile][it & 1]);
                        umma_commit_if(lead, &B.kempty[ks]);
                    }
                    if (!all_ok()) break;
                }
            }
        } else if (warp == PR_MMA + 2) {
            // ---- copies: a step's page into shared memory as it is, and its blocks' scales
            int pages = -1, pages_at = -64, pages_b = -1;   // lane l: page pages_at + l of sequence pages_b
            uint32_t it = 0, half = 0;
            for (uint32_t seg = 0;; ++seg) {
                const PrSeg& g = segment(seg);
                const int b = g.b, h = g.h, t0 = g.t0, t1 = g.t1, len = g.s.len;
                if (!all_ok() || t1 == 0) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.segempty[seg % PR_SEGS]);
#pragma unroll 1
                for (int t = t0; t < t1; ++t, ++it) {
                    const uint32_t rs = it % C::RST, par = ((it / C::RST) & 1) ^ 1;
                    if (b != pages_b || t < pages_at || t >= pages_at + 32) {
                        pages_b = b;
                        pages_at = t;
                        const int want = t + lane;
                        pages = static_cast<int64_t>(want) * KV_PAGE < len ? kv_page(p.c, p.b, b, want, status) : -1;
                    }
                    const int page = __shfl_sync(0xffffffffu, pages, t - pages_at);
                    const int64_t ph = static_cast<int64_t>(max(page, 0)) * p.c.kv_heads + h;
                    float4 mine = make_float4(1.0f, -INFINITY, 0.0f, 1.0f);   // no page: codes of zero and no weight
                    if (lane < 4 && page >= 0) {
                        const uint32_t ks = static_cast<const uint8_t*>(p.c.k_scale)[ph * KV_PAGE_BLOCKS + lane];
                        const uint32_t vs = static_cast<const uint8_t*>(p.c.v_scale)[ph * KV_PAGE_BLOCKS + lane];
                        const ValueScale v = value_scale(vs);
                        mine = make_float4(kv_scale(ks), v.e, v.inv, v.less);
                    }
                    if (__any_sync(0xffffffffu, mine.w != 1.0f)) mine.w = -mine.w;   // a step with such a block: pr_weights_masked
                    wait_on(&B.rkempty[rs], par);
                    if (!all_ok()) break;   // the stage is not free: nothing is copied into it
                    if (page < 0) {
                        for (int i = lane; i < C::RK / 16; i += 32) st_shared16(smem_u32(rawk) + rs * C::RK + i * 16, make_uint4(0, 0, 0, 0));
                        __syncwarp();
                    }
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&B.rkfull[rs], page >= 0 ? C::RK : 0);
                        if (page >= 0) bulk_g2s(rawk + rs * C::RK, static_cast<const uint8_t*>(p.c.k) + ph * C::RK, C::RK, &B.rkfull[rs]);
                    }
                    wait_on(&B.rvempty[rs], par);
                    if (!all_ok()) {
                        half = 1;
                        break;
                    }
                    if (page < 0)
                        for (int i = lane; i < C::RV / 16; i += 32) st_shared16(smem_u32(rawv) + rs * C::RV + i * 16, make_uint4(0, 0, 0, 0));
                    if (lane < 4) scales[it % PR_SCALES][lane] = mine;
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&B.rvfull[rs], page >= 0 ? C::RV : 0);
                        if (page >= 0) bulk_g2s(rawv + rs * C::RV, static_cast<const uint8_t*>(p.c.v) + ph * C::RV, C::RV, &B.rvfull[rs]);
                        mbar_arrive(&B.scfull[it % PR_SCALES]);
                    }
                    __syncwarp();
                }
            }
            if (lane == 0) B.copied_k = it + half, B.copied_v = it;
        } else if (warp == PR_MMA + 1 && lane == 0) {
            // ---- the segments of the piece
            int b = place.b, h = place.h, qb = place.qb, off = place.off, left = place.left, done = 0;
            KvSeq s = left > 0 ? kv_seq(p.b, b, status) : KvSeq{0, 0, 0, 0};
            for (uint32_t i = 0;; ++i) {
                // (the others may be a whole segment's steps away)
                if (!try_wait_long(&B.segempty[i % PR_SEGS], ((i / PR_SEGS) & 1) ^ 1) &&
                    !wait_more(&B.segempty[i % PR_SEGS], ((i / PR_SEGS) & 1) ^ 1, &B.gave_up, status, WAIT_LIMIT_NS + 20000ull * done))
                    break;
                PrSeg& g = segs[i % PR_SEGS];
                PrItem item{};
                int n = 0, lo = 0, hi = 0, after = 0;
                while (left > 0 && hi <= lo) {   // the next row block with a step in this piece
                    item = pr_item(s, p.group, p.window, qb);
                    const int have = item.tiles + PR_BLOCK_COST - off;
                    n = min(have, left);
                    if (n <= 0) break;   // lengths changed under the call
                    lo = max(off - PR_BLOCK_COST, 0);
                    hi = off + n - PR_BLOCK_COST;
                    after = have - n;
                    if (hi <= lo) left = 0;   // the piece ends before the row block's first step
                }
                if (hi <= lo) {
                    g.t0 = g.t1 = 0;
                    mbar_arrive(&B.segfull[i % PR_SEGS]);
                    break;
                }
                g.b = b, g.h = h, g.qb = qb, g.s = s;
                g.t0 = item.t0 + lo;
                g.t1 = item.t0 + hi;
                g.first = lo == 0;
                g.after = after;
                g.end = done + n + after;
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
    if (B.gave_up) {   // (what this needs is kept in shared memory: values held in registers until here cost the loops above 7 %)
        if (warp == PR_MMA || warp == PR_MMA + 3) {
            uint64_t* const bar = &B.mmadone[warp == PR_MMA ? 0 : 1];
            umma_commit_if(elect_one(), bar);   // the same lane as before
            wait_for_own(bar, 0);
        } else if (warp == PR_MMA + 2) {
            const uint32_t k = B.copied_k, v = B.copied_v;
            for (uint32_t i = 1; i <= C::RST; ++i) {
                if (k >= i) wait_for_own(&B.rkfull[(k - i) % C::RST], ((k - i) / C::RST) & 1);
                if (v >= i) wait_for_own(&B.rvfull[(v - i) % C::RST], ((v - i) / C::RST) & 1);
            }
        }
        __syncthreads();
    }
    if (warp == PR_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

constexpr int PR_COMBINE_ROWS = COMBINE_THREADS / 32;   // rows of a combining block, one per warp

// Joins the partial sums of the row block that begins in piece blockIdx.x and ends in a later one.
template <int DV, typename T>
__global__ void __launch_bounds__(COMBINE_THREADS) kv_prompt_combine(AttendArgs p)
{
    const int g = blockIdx.x, lane = threadIdx.x & 31;
    after_previous();
    const int4 head = p.heads_of[g];
    if (head.x < 0) return;
    const KvSeq s = kv_seq(p.b, head.x, p.c.status);
    const int pr = blockIdx.y * PR_COMBINE_ROWS + (threadIdx.x >> 5), r = head.z * PR_ROWS + pr, tok = r / p.group;
    if (tok >= s.n) return;
    const int step = PR_ROWS * (DV + 2), parts = head.w - g + 1;
    const float* base = p.part + static_cast<int64_t>(g) * 2 * step;
    auto part = [&](int k) { return base + (k == 0 ? step : static_cast<int64_t>(k) * 2 * step); };
    float m, l, o[4];
    join_parts<DV>(part, parts, pr, PR_ROWS + pr, 2 * PR_ROWS + static_cast<int64_t>(pr) * DV, lane, m, l, o);
    put_row<DV, T>(static_cast<T*>(p.out) + ((static_cast<int64_t>(s.row0) + tok) * p.heads + head.y * p.group + (r - tok * p.group)) * DV, l, o, lane);
}

template <int DK, int DV, typename T> static cudaError_t prompt_launch(AttendArgs p, cudaStream_t st)
{
    using C = PrCfg<DK, DV>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(&kv_prompt_kernel<DK, DV, T>), C::SMEM, done);
    if (e != cudaSuccess) return e;
    const int pieces = num_sms();
    e = launch_after(kv_prompt_kernel<DK, DV, T>, dim3(pieces), dim3(PR_WARPS * 32), C::SMEM, st, p);
    if (e != cudaSuccess) return e;
    return launch_after(kv_prompt_combine<DV, T>, dim3(pieces, PR_ROWS / PR_COMBINE_ROWS), dim3(COMBINE_THREADS), 0, st, p);
}

size_t prompt_workspace(int dv)
{
    return num_sms() * (sizeof(int4) + 2 * sizeof(float) * PR_ROWS * (dv + 2));
}

cudaError_t launch_prompt(AttendArgs p, void* workspace, bool bf16, cudaStream_t st)
{
    p.heads_of = static_cast<int4*>(workspace);
    p.part = reinterpret_cast<float*>(p.heads_of + num_sms());
    const int dk = p.c.key_dim;
    if (dk == 64) return bf16 ? prompt_launch<64, 64, __nv_bfloat16>(p, st) : prompt_launch<64, 64, __half>(p, st);
    if (dk == 128) return bf16 ? prompt_launch<128, 128, __nv_bfloat16>(p, st) : prompt_launch<128, 128, __half>(p, st);
    return bf16 ? prompt_launch<192, 128, __nv_bfloat16>(p, st) : prompt_launch<192, 128, __half>(p, st);
}

}  // namespace eva
