// Attention over the paged 8-bit cache: few rows per sequence and key/value head (decoding), entry point.
//
// At most 16 rows (new tokens x query heads of a group) share each key and value, so the cache's bytes are the cost: every
// one is read once. The tokens of all sequences and heads, in tiles of a page (64), form one line of work that is cut
// into equal pieces whatever the lengths are, one per warp of the GPU or, in short lines, fewer (DEC_PIECE, DEC_SPREAD); a warp's tiles come through its own
// two-stage ring of bulk copies (a page of a head is contiguous). Scores and outputs are m16n8k16 products with fp32 sums,
// transposed: keys and values are the 16-row operand and the query rows the 8-column one, so that up to eight rows cost what one
// does and no product is padding (an accumulator in tensor memory has 128 rows; the tensor pipes are at 19 % here, DRAM is the
// bound). The codes themselves are multiplied (e4m3 is exact in fp16); their scales stay outside: a
// token's key scale multiplies its score, its value scale 2^e joins the exponent, t = score + e, and the softmax's running
// maximum is that of t:
//   out = sum 2^(t - M) code / sum 2^(t - M) 2^-e.
// Weights are rounded to fp16, the operand's type, with 2^14 as the largest, so that tokens down to 2^-28 of the largest keep 11 bits; their sum
// is of the unrounded ones.
// The order of a tile's tokens within a product is free, and chosen so that both operands are 16-byte shared-memory loads and
// the weights need no exchange but movmatrix: product e of a tile has, in its rows r and r + 8, tokens
// 16 (r / 2) + 4 e + (0, 2) + r % 2, and lane quad q holds of the values tokens 16 q .. 16 q + 15.
// An item (sequence and head) whose tiles fall to several warps leaves fp32 partial sums, which
// kv_combine_kernel joins in their order, so results do not depend on timing.
//
// 128 + 128 dimensions, 8 heads of keys: 64 sequences of up to 8192 tokens, 4 rows: 581 MB in 106 us, 5.5 TB/s (0.84 of the 6.5 a
// copy reaches); two of 131072, 8 rows: 537 MB in 101 us, 5.3 TB/s; 16 heads of 192 + 128, one row each: 1365 MB in 236 us, 5.8 TB/s. Smaller calls are latency: 16 sequences of some 3000 tokens
// within a window of 4096, 4 heads, 16 rows: 54 MB in 36.5 us, of which a warp's six to eight tiles one behind the other take 25.
#include <algorithm>

#include "kv.cuh"
#include "kv_attend.cuh"

namespace eva {

constexpr int DEC_ROWS = 16;
// Tiles of a piece at least, but for calls that this leaves fewer than DEC_SPREAD pieces for each SM: see kv_decode_kernel
constexpr int DEC_PIECE = 8, DEC_SPREAD = 4, DEC_JOIN = 16;   // DEC_JOIN: parts of an item that one warp joins
constexpr float P_BIAS = 14.0f;   // weights are at most 2^14

template <int DK, int DV> struct DecCfg {
    static constexpr int KB = KV_PAGE * DK, VB = KV_PAGE * DV, STAGE = KB + VB, STAGES = 2;
    static constexpr int W = 224 * 1024 / (STAGES * STAGE) < 12 ? 224 * 1024 / (STAGES * STAGE) : 12;   // warps
    static constexpr int SMEM = W * STAGES * STAGE + 128;
};

static int dec_warps(int dk, int dv)
{
    return dk == 64 ? DecCfg<64, 64>::W : dk == 128 ? DecCfg<128, 128>::W : DecCfg<192, 128>::W;
}

// fp32 values of one partial sum of R rows: M and l of each row, then [R][DV]
static __host__ __device__ inline int part_floats(int R, int dv) { return R * (dv + 2); }

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transposes an 8 x 8 matrix of halves whose row lane / 4 has its columns 2 (lane % 4), + 1 in x.
__device__ __forceinline__ uint32_t transposed(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Tiles of one head of a sequence: the pages from the first token that its first row sees to its last one. A sequence with
// rows but no token has one (empty) tile, so that its rows are written.
__device__ __forceinline__ int dec_tiles(const KvSeq& s, int window, int* first)
{
    const int lo = window > 0 ? max(0, max(s.ctx, 0) + 1 - window) : 0;
    *first = lo / KV_PAGE;
    return s.n > 0 ? max(1, (s.len + KV_PAGE - 1) / KV_PAGE - *first) : 0;
}

struct DecTile {   // what the consumer of a tile needs
    int b, h, n, row0, len, tok;     // tok: first token; -1: nothing to read
    bool first, last;                // of its item
    int index, left;                 // tiles of the item before and after this one
    uint32_t ks, vs;                 // scale bytes of the block of the lane's scores (lane / 8)
};

struct alignas(16) DecRest {   // partial sums that a piece leaves of an item: its first (-1: none left) and last piece, rows, head
    int first, last, row0, n, h;
};

constexpr size_t DEC_RECORD = 2 * sizeof(DecRest) + DEC_ROWS * sizeof(int);   // of a piece: its two rests and counters

// NT: groups of eight rows
template <int DK, int DV, typename T, int NT>
__global__ void __launch_bounds__(DecCfg<DK, DV>::W * 32, 1) kv_decode_kernel(AttendArgs p)
{
    using C = DecCfg<DK, DV>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(8) uint64_t bars[C::W][C::STAGES];
    __shared__ int64_t spans[C::W * 32];   // tiles of a head, by runs of sequences
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, r8 = lane >> 2;
    uint8_t* ring = smem_raw + ((128 - (smem_u32(smem_raw) & 127)) & 127) + warp * C::STAGES * C::STAGE;
    if (lane == 0) {
        for (int i = 0; i < C::STAGES; ++i) mbar_init(&bars[warp][i], 1);
        fence_barrier_init();
    }
    after_previous();
    // length of the line of work: a thread sums a span of sequences
    const int span = (p.b.seqs + C::W * 32 - 1) / (C::W * 32);
    int at0;
    int64_t mine = 0;
    for (int b = threadIdx.x * span; b < min(p.b.seqs, static_cast<int>(threadIdx.x + 1) * span); ++b)
        mine += dec_tiles(kv_seq(p.b, b, p.c.status), p.window, &at0);
    spans[threadIdx.x] = mine;
    __syncthreads();
    int64_t total = 0;
    for (int i = lane; i < C::W * 32; i += 32) total += spans[i];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    total *= p.c.kv_heads;
    const int g = warp * gridDim.x + blockIdx.x;
    // Pieces, none of them empty. Every piece that cuts an item leaves partial sums to be joined, every tile waits for the one before it:
    // a decode step (rotation and append too) of 24 sequences of up to 3000 tokens takes 42.6 us in pieces of 8 tiles, 45 of 6, 45.7
    // with one for every warp; but 16 sequences of 2000 tokens and one head 19 us in four pieces for each SM, 25.5 in one.
    const int64_t most = static_cast<int64_t>(C::W) * gridDim.x, spread = static_cast<int64_t>(DEC_SPREAD) * gridDim.x;
    const int nw = static_cast<int>(min(min(most, total), max(spread, total / DEC_PIECE)));
    const int64_t begin = g < nw ? total * g / nw : 0;
    int64_t end = g < nw ? total * (g + 1) / nw : 0;
    DecRest lead{}, tail{};   // of an item that began before the piece, and of one that goes on behind it
    lead.first = tail.first = -1;
    if (begin < end) {
        // the sequence, head and tile at `begin`
        int b = 0, h = 0, i = 0, tiles = 0, first = 0;
        KvSeq s{};
        {
            int64_t rem = begin;
            bool found = false;
            // the lane, of 32 that hold t (and so many heads of it), whose part of the line holds tile `rem`; -1 and the next tile
            auto holder = [&](int64_t t, int64_t& own) {
                int64_t sum = t;
#pragma unroll
                for (int x = 1; x < 32; x <<= 1) {
                    const int64_t y = __shfl_up_sync(0xffffffffu, sum, x);
                    if (lane >= x) sum += y;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, sum * p.c.kv_heads > rem);
                const int l = hit ? __ffs(hit) - 1 : 31;
                rem -= __shfl_sync(0xffffffffu, hit ? sum - t : sum, l) * p.c.kv_heads;
                own = __shfl_sync(0xffffffffu, t, l);
                return hit ? l : -1;
            };
            for (int i0 = 0; i0 < C::W * 32 && !found; i0 += 32) {
                int64_t own;
                int l = holder(spans[i0 + lane], own);
                if (l < 0) continue;
                const int b1 = min(p.b.seqs, (i0 + l + 1) * span);
                for (int b0 = (i0 + l) * span; b0 < b1 && !found; b0 += 32) {
                    const int t = b0 + lane < b1 ? dec_tiles(kv_seq(p.b, b0 + lane, p.c.status), p.window, &at0) : 0;
                    l = holder(t, own);
                    if (l < 0) continue;
                    tiles = static_cast<int>(own);
                    b = b0 + l;
                    h = static_cast<int>(rem / tiles);
                    i = static_cast<int>(rem - static_cast<int64_t>(h) * tiles);
                    found = true;
                }
                break;
            }
            if (found) {
                s = kv_seq(p.b, b, p.c.status);
                dec_tiles(s, p.window, &first);
            } else {
                end = begin;   // lengths changed under the call
            }
        }
        int pages = 0, pages_at = -64;   // lane l: page of tile pages_at + l of sequence b
        int64_t next = begin;            // the tile that issue() takes, b / h / i are its place

        auto issue = [&](int slot) -> DecTile {
            DecTile t{};
            t.b = b, t.h = h, t.n = s.n, t.row0 = s.row0, t.len = s.len, t.first = i == 0, t.index = i, t.left = tiles - 1 - i;
            t.last = t.left == 0;
            t.tok = -1;
            if (s.len > 0) {
                const int pi = first + i;
                if (pi - pages_at >= 32 || pi < pages_at) {
                    pages_at = pi;
                    const int want = pi + lane;
                    pages = want * KV_PAGE < s.len ? kv_page(p.c, p.b, b, want, p.c.status) : -1;
                }
                const int page = __shfl_sync(0xffffffffu, pages, pi - pages_at);
                if (page >= 0) {
                    t.tok = pi * KV_PAGE;
                    const int64_t ph = static_cast<int64_t>(page) * p.c.kv_heads + h;
                    t.ks = static_cast<const uint8_t*>(p.c.k_scale)[ph * KV_PAGE_BLOCKS + (lane >> 3)];
                    t.vs = static_cast<const uint8_t*>(p.c.v_scale)[ph * KV_PAGE_BLOCKS + (lane >> 3)];
                    if (lane == 0) {
                        uint8_t* dst = ring + slot * C::STAGE;
                        mbar_arrive_expect_tx(&bars[warp][slot], C::STAGE);
                        bulk_g2s(dst, static_cast<const uint8_t*>(p.c.k) + ph * C::KB, C::KB, &bars[warp][slot]);
                        bulk_g2s(dst + C::KB, static_cast<const uint8_t*>(p.c.v) + ph * C::VB, C::VB, &bars[warp][slot]);
                    }
                }
            }
            ++next;
            if (++i == tiles && next < end) {
                i = 0;
                if (++h == p.c.kv_heads) {
                    h = 0;
                    tiles = 0;
                    while (tiles == 0 && ++b < p.b.seqs) {
                        s = kv_seq(p.b, b, p.c.status);
                        tiles = dec_tiles(s, p.window, &first);
                    }
                    if (tiles == 0) end = next;   // lengths changed under the call
                }
                pages_at = h == 0 ? -64 : pages_at;   // the same pages for the next head
            }
            return t;
        };

        uint32_t phase = 0;
        // the first item's queries, 1 us away, while its first tiles are looked up
        if (r8 < s.n * p.group) {
            const int tok = r8 / p.group;
            const T* q = static_cast<const T*>(p.q) + (static_cast<int64_t>(s.row0) + tok) * p.qt +
                         (static_cast<int64_t>(h) * p.group + (r8 - tok * p.group)) * p.qh + quad * 16;
#pragma unroll
            for (int j = 0; j < DK / 64; ++j) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + j * 64));
        }
        DecTile cur{}, nxt{};
        if (next < end) cur = issue(0);
        if (next < end) nxt = issue(1);
        // of each group of rows: the query as B operand, the output (rows 2 quad, + 1 of dimensions r8, r8 + 8 of each 16), and of
        // rows 2 quad, + 1 maximum, sum, factor and range of tokens
        uint32_t qf[NT][DK / 16][2];
        float o[NT][DV / 16][4], m[NT][2], l[NT][2], c[NT][2];
        int hi[NT][2], lo[NT][2];
        bool whole = false;
        for (int64_t at = begin; at < end; ++at) {
            const int slot = static_cast<int>(at - begin) & 1;
            if (cur.first || at == begin) {
                whole = cur.first;
#pragma unroll
                for (int g8 = 0; g8 < NT; ++g8) {
#pragma unroll
                    for (int j = 0; j < DV / 16; ++j) o[g8][j][0] = o[g8][j][1] = o[g8][j][2] = o[g8][j][3] = 0.0f;
                    // query row r8 of the group, scaled by a power of two to [1, 2) at its largest
                    const int r = 8 * g8 + r8, tok = r / p.group;
                    const bool in = tok < cur.n;
                    const T* q = static_cast<const T*>(p.q) + (static_cast<int64_t>(cur.row0) + tok) * p.qt +
                                 (static_cast<int64_t>(cur.h) * p.group + (r - tok * p.group)) * p.qh + quad * 16;
                    uint4 raw[DK / 64][2];
                    float big = 0.0f;
#pragma unroll
                    for (int j = 0; j < DK / 64; ++j)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            raw[j][k] = in ? *reinterpret_cast<const uint4*>(q + j * 64 + k * 8) : make_uint4(0, 0, 0, 0);
                    bool odd = false;
#pragma unroll
                    for (int j = 0; j < DK / 64; ++j)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t w[4] = {raw[j][k].x, raw[j][k].y, raw[j][k].z, raw[j][k].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 f = two_floats<T>(w[e]);
                                big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
                                odd |= f.x != f.x || f.y != f.y;
                            }
                        }
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                    odd = (__ballot_sync(0xffffffffu, odd) >> (r8 * 4) & 15u) != 0 || big == INFINITY;
                    const int e2 = min(max(static_cast<int>(__float_as_uint(big) >> 23), 1), 252);
                    const float down = __uint_as_float(static_cast<uint32_t>(254 - e2) << 23);
                    const float own = odd ? __uint_as_float(0x7fc00000u) : p.scale * __uint_as_float(static_cast<uint32_t>(e2) << 23);
#pragma unroll
                    for (int j = 0; j < DK / 64; ++j)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t w[4] = {raw[j][k].x, raw[j][k].y, raw[j][k].z, raw[j][k].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 f = two_floats<T>(w[e]);
                                // elements 8 k + 2 e, + 1 of the lane's 16: product 2 k + e / 2, k index pair e % 2
                                qf[g8][j * 4 + 2 * k + e / 2][e % 2] = half2_bits(f.x * down, f.y * down);
                            }
                        }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int t = (8 * g8 + 2 * quad + x) / p.group;
                        c[g8][x] = __shfl_sync(0xffffffffu, own, 8 * quad + 4 * x);
                        hi[g8][x] = t < cur.n ? cur.len - cur.n + t + 1 : 0;
                        lo[g8][x] = p.window > 0 ? max(0, hi[g8][x] - p.window) : 0;
                        m[g8][x] = -INFINITY;
                        l[g8][x] = 0.0f;
                    }
                }
            }
            if (cur.tok >= 0) {
                const uint8_t* K = ring + slot * C::STAGE;
                const uint8_t* V = K + C::KB;
                if (!copies_arrived(&bars[warp][slot], phase >> slot & 1, p.c.status)) {
                    copies_late(&bars[warp][slot], phase >> slot & 1, p.c.status);
                    if (at + 1 < end && nxt.tok >= 0) copies_late(&bars[warp][slot ^ 1], phase >> (slot ^ 1) & 1, p.c.status);
                    break;   // the item stays unfinished
                }
                phase ^= 1u << slot;
                float sc[NT][4][4];   // product e: tokens t0 + 4 e + (0, 0, 2, 2), rows 2 quad + (0, 1, 0, 1)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int g8 = 0; g8 < NT; ++g8) sc[g8][e][0] = sc[g8][e][1] = sc[g8][e][2] = sc[g8][e][3] = 0.0f;
                    const uint8_t* kr = K + (16 * (r8 >> 1) + 4 * e + (r8 & 1)) * DK + quad * 16;
#pragma unroll
                    for (int j = 0; j < DK / 64; ++j) {
                        const uint4 x4 = *reinterpret_cast<const uint4*>(kr + j * 64);
                        const uint4 y4 = *reinterpret_cast<const uint4*>(kr + 2 * DK + j * 64);
                        const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t a0, a1, a2, a3;
                            e4m3_halves(x[k], a0, a2);
                            e4m3_halves(y[k], a1, a3);
#pragma unroll
                            for (int g8 = 0; g8 < NT; ++g8) mma_f16(sc[g8][e], a0, a1, a2, a3, qf[g8][j * 4 + k][0], qf[g8][j * 4 + k][1]);
                        }
                    }
                }
                const float ks = kv_scale(cur.ks);
                const ValueScale vsc = value_scale(cur.vs);
                const int t0 = cur.tok + 16 * (r8 >> 1) + (r8 & 1);
                const bool part = cur.tok + KV_PAGE > cur.len - cur.n + 1 || (p.window > 0 && cur.tok < cur.len - p.window);   // not for all rows
                uint32_t pf[NT][4][2];
#pragma unroll
                for (int g8 = 0; g8 < NT; ++g8) {
                    float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float a = sc[g8][e][k] * (ks * c[g8][k & 1]) + vsc.e;
                            if (part) {
                                const int t = t0 + 4 * e + (k & 2);
                                a = t >= lo[g8][k & 1] && t < hi[g8][k & 1] ? a : -INFINITY;
                            }
                            sc[g8][e][k] = a;
                            x[k & 1] = fmaxf(x[k & 1], a);
                        }
#pragma unroll
                    for (int s2 = 4; s2 < 32; s2 <<= 1) {
                        x[0] = fmaxf(x[0], __shfl_xor_sync(0xffffffffu, x[0], s2));
                        x[1] = fmaxf(x[1], __shfl_xor_sync(0xffffffffu, x[1], s2));
                    }
                    if (__any_sync(0xffffffffu, x[0] > m[g8][0] || x[1] > m[g8][1])) {
                        float fall[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float now = fmaxf(m[g8][k], x[k]);
                            fall[k] = m[g8][k] == -INFINITY ? 1.0f : ex2(m[g8][k] - now);   // (nothing there yet, or NaN)
                            l[g8][k] *= fall[k];
                            m[g8][k] = now;
                        }
#pragma unroll
                        for (int j = 0; j < DV / 16; ++j)
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[g8][j][k] *= fall[k & 1];
                    }
                    const float ref[2] = {P_BIAS - (m[g8][0] == -INFINITY ? 0.0f : m[g8][0]), P_BIAS - (m[g8][1] == -INFINITY ? 0.0f : m[g8][1])};
                    float sum[2] = {0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            w[k] = ex2(sc[g8][e][k] + ref[k & 1]);
                            sum[k & 1] += w[k];
                        }
                        pf[g8][e][0] = transposed(half2_bits(w[0] * vsc.less, w[1] * vsc.less));
                        pf[g8][e][1] = transposed(half2_bits(w[2] * vsc.less, w[3] * vsc.less));
                    }
                    l[g8][0] = fmaf(sum[0], vsc.inv, l[g8][0]);
                    l[g8][1] = fmaf(sum[1], vsc.inv, l[g8][1]);
                }
                // tokens of the quad's block; what lies behind the sequence's end may be anything, NaN codes too
                const int live = cur.len - cur.tok - 16 * quad;
                const bool tail = cur.tok + KV_PAGE > cur.len;
                uint32_t keep[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = live - 4 * e;
                    keep[e] = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
                }
#pragma unroll
                for (int j = 0; j < DV / 16; ++j) {
                    const uint4 x4 = *reinterpret_cast<const uint4*>(V + (16 * j + r8) * KV_PAGE + quad * 16);
                    const uint4 y4 = *reinterpret_cast<const uint4*>(V + (16 * j + r8 + 8) * KV_PAGE + quad * 16);
                    uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (tail) x[e] &= keep[e], y[e] &= keep[e];
                        uint32_t a0, a1, a2, a3;
                        e4m3_halves(x[e], a0, a2);
                        e4m3_halves(y[e], a1, a3);
#pragma unroll
                        for (int g8 = 0; g8 < NT; ++g8) mma_f16(o[g8][j], a0, a1, a2, a3, pf[g8][e][0], pf[g8][e][1]);
                    }
                }
                __syncwarp();   // every lane has read the stage
            }
            const DecTile done = cur;
            cur = nxt;
            if (next < end) nxt = issue(slot);
            if (done.last || at == end - 1) {
                const int rows = done.n * p.group;
                const bool out = whole && done.last;
                // partial: slot 1 where the item begins here, slot 0 where it began in an earlier warp
                const int R = p.part_rows;
                float* dst = p.part + (static_cast<int64_t>(g) * 2 + (whole ? 1 : 0)) * part_floats(R, DV);
#pragma unroll
                for (int g8 = 0; g8 < NT; ++g8)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float sum = l[g8][x];
#pragma unroll
                        for (int s2 = 4; s2 < 32; s2 <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s2);
                        const int r = 8 * g8 + 2 * quad + x, tok = r / p.group;
                        if (r >= rows) continue;
                        if (out) {
                            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                            T* row = static_cast<T*>(p.out) +
                                     ((static_cast<int64_t>(done.row0) + tok) * p.heads + done.h * p.group + (r - tok * p.group)) * DV + r8;
#pragma unroll
                            for (int j = 0; j < DV / 16; ++j) {
                                row[16 * j] = one_of<T>(o[g8][j][x] * inv);
                                row[16 * j + 8] = one_of<T>(o[g8][j][2 + x] * inv);
                            }
                        } else {
                            if (r8 == 0) {
                                dst[r] = m[g8][x];
                                dst[R + r] = sum;
                            }
#pragma unroll
                            for (int j = 0; j < DV / 16; ++j) {
                                dst[2 * R + r * DV + r8 + 16 * j] = o[g8][j][x];
                                dst[2 * R + r * DV + r8 + 16 * j + 8] = o[g8][j][2 + x];
                            }
                        }
                    }
                if (!out) {
                    // the item's pieces: those that hold its first and its last tile
                    DecRest& rest = whole ? tail : lead;
                    rest.first = static_cast<int>(((at - done.index + 1) * nw - 1) / total);
                    rest.last = static_cast<int>(((at + done.left + 1) * nw - 1) / total);
                    rest.row0 = done.row0, rest.n = done.n, rest.h = done.h;
                }
            }
        }
    }
    if (lane == 0) {
        DecRest* to = reinterpret_cast<DecRest*>(p.heads_of) + 2 * g;
        to[0] = lead;
        to[1] = tail;
    }
    // counters of the joining kernel's groups
    int* count = reinterpret_cast<int*>(reinterpret_cast<DecRest*>(p.heads_of) + 2 * C::W * gridDim.x) + g * DEC_ROWS;
    if (lane < DEC_ROWS) count[lane] = 0;
}

// Joins the partial sums of the items that lie in several pieces. The parts of an item are joined in groups of 16 by the warp of
// the group's first piece (and row); where there are more groups, the one that is done last joins the groups, in their
// order whichever that is, so that an item of a thousand pieces takes as long as ten loads, not a hundred. A second level costs 5 us,
// eight more parts one: groups of 8, 16, 32 take 38.5, 36.6, 36.6 us for the drafted tokens above, 99.2, 98.4, 100.2 for the two of 131072.
template <int DV, typename T>
__global__ void __launch_bounds__(COMBINE_THREADS) kv_combine_kernel(AttendArgs p, int pieces)
{
    const int lane = threadIdx.x & 31, R = p.part_rows, step = part_floats(R, DV);
    const int64_t task = static_cast<int64_t>(blockIdx.x) * (COMBINE_THREADS / 32) + (threadIdx.x >> 5);
    const int g = static_cast<int>(task / R), r = static_cast<int>(task - static_cast<int64_t>(g) * R);
    if (g >= pieces) return;
    after_previous();
    const DecRest* rests = reinterpret_cast<const DecRest*>(p.heads_of);
    int* counts = reinterpret_cast<int*>(reinterpret_cast<DecRest*>(p.heads_of) + 2 * pieces);
    for (int slot = 0; slot < 2; ++slot) {
        const DecRest rest = rests[2 * g + slot];
        const int i = g - rest.first;   // this piece's part of the item
        if (rest.first < 0 || i % DEC_JOIN != 0 || r >= rest.n * p.group) continue;
        // part k of the item: its first piece, slot 1, then the next pieces, slot 0
        float* base = p.part + static_cast<int64_t>(rest.first) * 2 * step;
        auto part = [&](int k) { return base + (k == 0 ? step : static_cast<int64_t>(k) * 2 * step); };
        const int parts = rest.last - rest.first + 1, groups = (parts + DEC_JOIN - 1) / DEC_JOIN, tok = r / p.group;
        T* out = static_cast<T*>(p.out) + ((static_cast<int64_t>(rest.row0) + tok) * p.heads + rest.h * p.group + (r - tok * p.group)) * DV;
        float m, l, o[4];
        join_parts<DV>([&](int k) { return part(i + k); }, min(DEC_JOIN, parts - i), r, R + r, 2 * R + r * DV, lane, m, l, o);
        if (groups > 1) {
            float* own = part(i);   // no other warp reads this row of it
            __syncwarp();
            if (lane == 0) own[r] = m, own[R + r] = l;
            if (lane * 4 < DV) {
                *reinterpret_cast<float2*>(own + 2 * R + r * DV + lane * 4) = make_float2(o[0], o[1]);
                *reinterpret_cast<float2*>(own + 2 * R + r * DV + lane * 4 + 2) = make_float2(o[2], o[3]);
            }
            __threadfence();
            __syncwarp();
            int before = 0;
            if (lane == 0) before = atomicAdd(counts + rest.first * DEC_ROWS + r, 1);
            if (__shfl_sync(0xffffffffu, before, 0) != groups - 1) continue;
            __threadfence();
            join_parts<DV>([&](int k) { return part(DEC_JOIN * k); }, groups, r, R + r, 2 * R + r * DV, lane, m, l, o);
        }
        put_row<DV, T>(out, l, o, lane);
    }
}

template <int DK, int DV, typename T, int NT> static cudaError_t decode_launch(AttendArgs p, int pieces, cudaStream_t st)
{
    using C = DecCfg<DK, DV>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(&kv_decode_kernel<DK, DV, T, NT>), C::SMEM, done);
    if (e != cudaSuccess) return e;
    e = launch_after(kv_decode_kernel<DK, DV, T, NT>, dim3(pieces / C::W), dim3(C::W * 32), C::SMEM, st, p);
    if (e != cudaSuccess) return e;
    const int64_t tasks = static_cast<int64_t>(pieces) * p.part_rows, each = COMBINE_THREADS / 32;
    return launch_after(kv_combine_kernel<DV, T>, dim3(static_cast<unsigned>((tasks + each - 1) / each)), dim3(COMBINE_THREADS), 0, st, p, pieces);
}

template <typename T> static cudaError_t decode_typed(const AttendArgs& p, int pieces, cudaStream_t st)
{
    const bool one = p.part_rows <= 8;   // a group of eight rows or two: 4 rows 103 us, 142 with an empty second group
    if (p.c.key_dim == 64) return one ? decode_launch<64, 64, T, 1>(p, pieces, st) : decode_launch<64, 64, T, 2>(p, pieces, st);
    if (p.c.key_dim == 128) return one ? decode_launch<128, 128, T, 1>(p, pieces, st) : decode_launch<128, 128, T, 2>(p, pieces, st);
    return one ? decode_launch<192, 128, T, 1>(p, pieces, st) : decode_launch<192, 128, T, 2>(p, pieces, st);
}

}  // namespace eva

using namespace eva;

static bool attend_ok(const EvaKvCache* cache, const EvaKvBatch* batch, int32_t heads)
{
    return kv_cache_ok(cache) && kv_batch_ok(batch) && heads >= 1 && heads % cache->kv_heads == 0;
}

// Rows that share a key and value head's tokens. Up to 16 the decode kernel takes them: 64 sequences of 8000 tokens and 16 rows 61 us,
// 90 in the prompt kernel, 4 rows 103 against 332 (8 heads); one of 16 x 2000 19 against 23. More rows than two products' columns
// would reload the queries and halve the decode kernel's warps; 24 rows are 90 us in the prompt kernel, as 16 are.
static int64_t shared_rows(const EvaKvCache& c, const EvaKvBatch& b, int heads)
{
    return static_cast<int64_t>(b.max_q) * (heads / c.kv_heads);
}

extern "C" size_t eva_kv_attend_workspace(const EvaKvCache* cache, const EvaKvBatch* batch, int32_t heads)
{
    if (!attend_ok(cache, batch, heads)) return 0;
    const int64_t rows = shared_rows(*cache, *batch, heads);
    if (rows > DEC_ROWS) return prompt_workspace(cache->value_dim);
    const size_t pieces = static_cast<size_t>(num_sms()) * dec_warps(cache->key_dim, cache->value_dim);
    return pieces * (DEC_RECORD + 2 * sizeof(float) * part_floats(static_cast<int>(rows), cache->value_dim));
}

extern "C" int eva_kv_attend(const EvaKvCache* cache, const EvaKvBatch* batch, const void* q, int32_t dtype, int32_t heads,
                             int64_t q_token_stride, int64_t q_head_stride, float scale, int32_t window, void* workspace,
                             size_t workspace_bytes, void* out, void* stream)
{
    if (!attend_ok(cache, batch, heads) || (dtype != EVA_DTYPE_F16 && dtype != EVA_DTYPE_BF16) || window < 0 ||
        !(scale >= 0.0f) || scale > 2.0e38f)   // times log2(e) is finite
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
    p.window = window < (1 << 30) ? window : 0;   // the longest sequence: no window, and no sum of it passes 32 bits
    p.scale = scale * 1.4426950408889634f;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t rows = shared_rows(*cache, *batch, heads);
    cudaError_t e;
    if (rows <= DEC_ROWS) {
        const int pieces = num_sms() * dec_warps(cache->key_dim, cache->value_dim);
        p.part_rows = static_cast<int>(rows);
        p.heads_of = static_cast<int4*>(workspace);
        p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + pieces * DEC_RECORD);
        e = dtype == EVA_DTYPE_BF16 ? decode_typed<__nv_bfloat16>(p, pieces, st) : decode_typed<__half>(p, pieces, st);
    } else {
        e = launch_prompt(p, workspace, dtype == EVA_DTYPE_BF16, st);
    }
    return e == cudaSuccess ? EVA_OK : EVA_ERR_CUDA;
}
