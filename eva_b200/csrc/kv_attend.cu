// Attention over the paged 8-bit cache: few rows per sequence and key/value head (decoding), entry point.
//
// At most 16 rows (new tokens x query heads of a group) share each key and value, so the cache's bytes are the cost: every
// one is read once. The tokens of all sequences and heads, in tiles of a page (64), form one line of work that is cut
// into equal pieces, one per warp of the GPU, whatever the lengths are; a warp's tiles come through its own
// two-stage ring of bulk copies (a page of a head is contiguous). Scores and outputs are m16n8k16 products with fp32 sums
// on the codes themselves (e4m3 is exact in fp16). Their scales stay outside: a token's key scale multiplies its
// score, its value scale 2^e joins the exponent, t = score + e, and the softmax's running maximum is that of t:
//   out = sum 2^(t - M) code / sum 2^(t - M) 2^-e.
// Weights are rounded to fp16 with 2^14 as the largest, so that tokens down to 2^-28 of the largest keep 11 bits.
// The order of a tile's tokens within a product is free, and chosen so that both operands are 16-byte shared-memory loads:
// lane quad q holds tokens 16 q .. 16 q + 15 (one scale block) and, of the keys, dimensions 16 q .. 16 q + 15 of each 64.
// An item (sequence and head) whose tiles fall to several warps leaves fp32 partial sums, which
// kv_combine_kernel joins in their order, so results do not depend on timing.
#include <algorithm>

#include "kv.cuh"
#include "kv_attend.cuh"

#include <cuda_fp8.h>

namespace eva {

constexpr int DEC_ROWS = 16;
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
    int left;                        // tiles of the item after this one
    uint32_t ks, vs;                 // scale bytes of the lane quad's block
};

template <int DK, int DV, typename T>
__global__ void __launch_bounds__(DecCfg<DK, DV>::W * 32, 1) kv_decode_kernel(const AttendArgs p)
{
    using C = DecCfg<DK, DV>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(8) uint64_t bars[C::W][C::STAGES];
    __shared__ int sums[C::W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, n8 = lane >> 2;
    uint8_t* ring = smem_raw + ((128 - (smem_u32(smem_raw) & 127)) & 127) + warp * C::STAGES * C::STAGE;
    if (lane == 0) {
        for (int i = 0; i < C::STAGES; ++i) mbar_init(&bars[warp][i], 1);
        fence_barrier_init();
    }
    // length of the line of work
    int mine = 0, at0;
    for (int b = threadIdx.x; b < p.b.seqs; b += C::W * 32) mine += dec_tiles(kv_seq(p.b, b, p.c.status), p.window, &at0);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int i = 0; i < C::W; ++i) total += sums[i];
    total *= p.c.kv_heads;
    const int g = warp * gridDim.x + blockIdx.x;
    const int nw = static_cast<int>(min(static_cast<int64_t>(C::W * gridDim.x), total));   // pieces, none of them empty
    const int64_t begin = g < nw ? total * g / nw : 0;
    int64_t end = g < nw ? total * (g + 1) / nw : 0;
    int4 head = make_int4(-1, 0, 0, 0);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (begin < end) {
        // the sequence, head and tile at `begin`
        int b = 0, h = 0, i = 0, tiles = 0, first = 0;
        KvSeq s{};
        {
            int64_t before = 0;
            bool found = false;
            for (int b0 = 0; b0 < p.b.seqs; b0 += 32) {
                int t = b0 + lane < p.b.seqs ? dec_tiles(kv_seq(p.b, b0 + lane, p.c.status), p.window, &at0) : 0, sum = t;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += x;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, before + static_cast<int64_t>(sum) * p.c.kv_heads > begin);
                if (hit) {
                    const int l = __ffs(hit) - 1;
                    b = b0 + l;
                    const int64_t rem =
                        begin - before - static_cast<int64_t>(__shfl_sync(0xffffffffu, sum - t, l)) * p.c.kv_heads;
                    tiles = __shfl_sync(0xffffffffu, t, l);
                    h = static_cast<int>(rem / tiles);
                    i = static_cast<int>(rem - static_cast<int64_t>(h) * tiles);
                    found = true;
                    break;
                }
                before += static_cast<int64_t>(__shfl_sync(0xffffffffu, sum, 31)) * p.c.kv_heads;
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
            t.b = b, t.h = h, t.n = s.n, t.row0 = s.row0, t.len = s.len, t.first = i == 0, t.left = tiles - 1 - i;
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
                    t.ks = static_cast<const uint8_t*>(p.c.k_scale)[ph * KV_PAGE_BLOCKS + quad];
                    t.vs = static_cast<const uint8_t*>(p.c.v_scale)[ph * KV_PAGE_BLOCKS + quad];
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
        DecTile cur{}, nxt{};
        if (next < end) cur = issue(0);
        if (next < end) nxt = issue(1);
        uint32_t qf[DK / 16][4];
        float o[DV / 8][4], m0 = 0, m1 = 0, l0 = 0, l1 = 0, c0 = 0, c1 = 0;
        int hi0 = 0, hi1 = 0, lo0 = 0, lo1 = 0;
        bool whole = false;
        for (int64_t at = begin; at < end; ++at) {
            const int slot = static_cast<int>(at - begin) & 1;
            if (cur.first || at == begin) {
                whole = cur.first;
                m0 = m1 = -INFINITY;
                l0 = l1 = 0.0f;
#pragma unroll
                for (int j = 0; j < DV / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
                // query rows n8 and n8 + 8, scaled by a power of two to [1, 2) at their largest
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int r = n8 + 8 * half, tok = r / p.group;
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
                    const uint32_t some_odd = __ballot_sync(0xffffffffu, odd);
                    odd = (some_odd >> (n8 * 4) & 15u) != 0 || big == INFINITY;
                    const int e2 = min(max(static_cast<int>(__float_as_uint(big) >> 23), 1), 252);
                    const float down = __uint_as_float(static_cast<uint32_t>(254 - e2) << 23);
                    const float c = odd ? __uint_as_float(0x7fc00000u)
                                        : p.scale * __uint_as_float(static_cast<uint32_t>(e2) << 23);
#pragma unroll
                    for (int j = 0; j < DK / 64; ++j)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t w[4] = {raw[j][k].x, raw[j][k].y, raw[j][k].z, raw[j][k].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 f = two_floats<T>(w[e]);
                                // elements 8 k + 2 e, + 1 of the lane's 16: step 2 k + e / 2, k index pair e % 2
                                qf[j * 4 + 2 * k + e / 2][half + 2 * (e % 2)] = half2_bits(f.x * down, f.y * down);
                            }
                        }
                    const int hi = in ? cur.len - cur.n + tok + 1 : 0;
                    const int lo = p.window > 0 ? max(0, hi - p.window) : 0;
                    if (half == 0) c0 = c, hi0 = hi, lo0 = lo;
                    else c1 = c, hi1 = hi, lo1 = lo;
                }
            }
            if (cur.tok >= 0) {
                const uint8_t* K = ring + slot * C::STAGE;
                const uint8_t* V = K + C::KB;
                mbar_wait(&bars[warp][slot], phase >> slot & 1, p.c.status);
                phase ^= 1u << slot;
                float sc[8][4];   // 4-token step i, half h: [2 i + h]; columns: tokens 16 quad + 4 i + 2 h + {0, 1}
#pragma unroll
                for (int ih = 0; ih < 8; ++ih) {
                    sc[ih][0] = sc[ih][1] = sc[ih][2] = sc[ih][3] = 0.0f;
                    const uint8_t* kr = K + (16 * (n8 >> 1) + 2 * ih + (n8 & 1)) * DK + quad * 16;
#pragma unroll
                    for (int j = 0; j < DK / 64; ++j) {
                        const uint4 w4 = *reinterpret_cast<const uint4*>(kr + j * 64);
                        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            uint32_t k0, k1;
                            e4m3_halves(w[e], k0, k1);
                            mma_f16(sc[ih], qf[j * 4 + e][0], qf[j * 4 + e][1], qf[j * 4 + e][2], qf[j * 4 + e][3], k0, k1);
                        }
                    }
                }
                const float ks = kv_scale(cur.ks), vlog = static_cast<float>(static_cast<int>(max(cur.vs, 1u)) - 127);
                const float f0 = ks * c0, f1 = ks * c1;
                const int t0 = cur.tok + 16 * quad;
                const bool part = cur.tok + KV_PAGE > cur.len - cur.n + 1 || p.window > 0;   // some row does not see all
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int ih = 0; ih < 8; ++ih)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float a = sc[ih][e] * f0 + vlog, c = sc[ih][2 + e] * f1 + vlog;
                        if (part) {
                            const int t = t0 + 2 * ih + e;
                            a = t >= lo0 && t < hi0 ? a : -INFINITY;
                            c = t >= lo1 && t < hi1 ? c : -INFINITY;
                        }
                        sc[ih][e] = a;
                        sc[ih][2 + e] = c;
                        x0 = fmaxf(x0, a);
                        x1 = fmaxf(x1, c);
                    }
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
                x0 = fmaxf(m0, fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2)));
                x1 = fmaxf(m1, fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2)));
                if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
                    const float d0 = m0 == -INFINITY ? 0.0f : ex2(m0 - x0), d1 = m1 == -INFINITY ? 0.0f : ex2(m1 - x1);
                    l0 *= d0;
                    l1 *= d1;
#pragma unroll
                    for (int j = 0; j < DV / 8; ++j) o[j][0] *= d0, o[j][1] *= d0, o[j][2] *= d1, o[j][3] *= d1;
                    m0 = x0;
                    m1 = x1;
                }
                const float r0 = P_BIAS - (m0 == -INFINITY ? 0.0f : m0), r1 = P_BIAS - (m1 == -INFINITY ? 0.0f : m1);
                float w0 = 0.0f, w1 = 0.0f;
                uint32_t pf[4][4];
#pragma unroll
                for (int ih = 0; ih < 8; ++ih) {
                    const float a0 = ex2(sc[ih][0] + r0), a1 = ex2(sc[ih][1] + r0);
                    const float b0 = ex2(sc[ih][2] + r1), b1 = ex2(sc[ih][3] + r1);
                    w0 += a0 + a1;
                    w1 += b0 + b1;
                    pf[ih >> 1][2 * (ih & 1)] = half2_bits(a0, a1);
                    pf[ih >> 1][2 * (ih & 1) + 1] = half2_bits(b0, b1);
                }
                const float iv = __uint_as_float((254u - min(max(cur.vs, 1u), 253u)) << 23);   // 2^-vlog
                l0 = fmaf(w0, iv, l0);
                l1 = fmaf(w1, iv, l1);
                const int live = cur.len - t0;   // tokens of the quad's block; what lies behind may be anything, NaN codes too
                const bool tail = cur.tok + KV_PAGE > cur.len;
                uint32_t keep[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = live - 4 * e;
                    keep[e] = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
                }
#pragma unroll
                for (int j = 0; j < DV / 8; ++j) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(V + (8 * j + n8) * KV_PAGE + quad * 16);
                    uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (tail) w[e] &= keep[e];
                        uint32_t v0, v1;
                        e4m3_halves(w[e], v0, v1);
                        mma_f16(o[j], pf[e][0], pf[e][1], pf[e][2], pf[e][3], v0, v1);
                    }
                }
                __syncwarp();   // every lane has read the stage
            }
            const DecTile done = cur;
            cur = nxt;
            if (next < end) nxt = issue(slot);
            if (done.last || at == end - 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
                l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
                l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
                l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
                const int rows = done.n * p.group;
                if (whole && done.last) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int r = n8 + 8 * half, tok = r / p.group;
                        if (r < rows) {
                            const float l = half ? l1 : l0, inv = l == 0.0f ? 0.0f : 1.0f / l;
                            T* out = static_cast<T*>(p.out) +
                                     ((static_cast<int64_t>(done.row0) + tok) * p.heads + done.h * p.group + (r - tok * p.group)) * DV +
                                     2 * quad;
#pragma unroll
                            for (int j = 0; j < DV / 8; ++j)
                                *reinterpret_cast<uint32_t*>(out + 8 * j) =
                                    two_bits<T>(o[j][2 * half] * inv, o[j][2 * half + 1] * inv);
                        }
                    }
                } else {
                    // partial: slot 1 where the item begins here, slot 0 where it began in an earlier warp
                    const int R = p.part_rows;
                    float* dst = p.part + (static_cast<int64_t>(g) * 2 + (whole ? 1 : 0)) * part_floats(R, DV);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int r = n8 + 8 * half;
                        if (r < rows) {
                            if (quad == 0) {
                                dst[r] = half ? m1 : m0;
                                dst[R + r] = half ? l1 : l0;
                            }
#pragma unroll
                            for (int j = 0; j < DV / 8; ++j)
                                *reinterpret_cast<float2*>(dst + 2 * R + r * DV + 8 * j + 2 * quad) =
                                    make_float2(o[j][2 * half], o[j][2 * half + 1]);
                        }
                    }
                    if (whole) {
                        // last warp with a tile of the item: the one whose piece holds tile at + left
                        const int64_t last = at + done.left;
                        head = make_int4(done.b, done.h, static_cast<int>(((last + 1) * nw - 1) / total), 0);
                    }
                }
            }
        }
    }
    if (lane == 0) p.heads_of[g] = head;
}

// Joins the partial sums of the item that begins in piece blockIdx.x and ends in a later one; row blockIdx.y.
template <int DV, typename T>
__global__ void __launch_bounds__(COMBINE_THREADS) kv_combine_kernel(const AttendArgs p)
{
    constexpr int GROUPS = COMBINE_THREADS / DV;
    __shared__ float acc[GROUPS][DV], ls[GROUPS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int g = blockIdx.x, r = blockIdx.y;
    const int4 head = p.heads_of[g];
    if (head.x < 0) return;
    const KvSeq s = kv_seq(p.b, head.x, p.c.status);
    if (r >= s.n * p.group) return;
    const int R = p.part_rows, step = part_floats(R, DV);
    const int d = threadIdx.x % DV, grp = threadIdx.x / DV;
    // part k of the item: piece g, slot 1, then pieces g + 1 .. head.z, slot 0
    const float* base = p.part + static_cast<int64_t>(g) * 2 * step;
    const int parts = head.z - g + 1;
    auto part = [&](int k) { return base + (k == 0 ? step : static_cast<int64_t>(k) * 2 * step); };
    float m = -INFINITY;
    for (int k = 0; k < parts; ++k) m = fmaxf(m, part(k)[r]);
    const float ref = m == -INFINITY ? 0.0f : m;
    float o = 0.0f, l = 0.0f;
#pragma unroll 4
    for (int k = grp; k < parts; k += GROUPS) {
        const float* q = part(k);
        const float w = ex2(q[r] - ref);
        l = fmaf(q[R + r], w, l);
        o = fmaf(q[2 * R + r * DV + d], w, o);
    }
    acc[grp][d] = o;
    if (d == 0) ls[grp] = l;
    __syncthreads();
    if (grp == 0) {
        l = o = 0.0f;
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
            l += ls[k];
            o += acc[k][d];
        }
        const int tok = r / p.group;
        static_cast<T*>(p.out)[((static_cast<int64_t>(s.row0) + tok) * p.heads + head.y * p.group + (r - tok * p.group)) * DV + d] =
            one_of<T>(l == 0.0f ? 0.0f : o / l);
    }
}

template <int DK, int DV, typename T> static cudaError_t decode_launch(const AttendArgs& p, int pieces, cudaStream_t st)
{
    using C = DecCfg<DK, DV>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(&kv_decode_kernel<DK, DV, T>), C::SMEM, done);
    if (e != cudaSuccess) return e;
    kv_decode_kernel<DK, DV, T><<<pieces / C::W, C::W * 32, C::SMEM, st>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // launched while the decode kernel runs; its blocks wait for that kernel's end before they read
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(pieces, p.part_rows);
    cfg.blockDim = dim3(COMBINE_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_combine_kernel<DV, T>, p);
}

template <typename T> static cudaError_t decode_typed(const AttendArgs& p, int pieces, cudaStream_t st)
{
    if (p.c.key_dim == 64) return decode_launch<64, 64, T>(p, pieces, st);
    if (p.c.key_dim == 128) return decode_launch<128, 128, T>(p, pieces, st);
    return decode_launch<192, 128, T>(p, pieces, st);
}

}  // namespace eva

using namespace eva;

static bool attend_ok(const EvaKvCache* cache, const EvaKvBatch* batch, int32_t heads)
{
    return kv_cache_ok(cache) && kv_batch_ok(batch) && heads >= 1 && heads % cache->kv_heads == 0;
}

// Rows that share a key and value head's tokens, and whether the decode kernel takes them.
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
    return pieces * (sizeof(int4) + 2 * sizeof(float) * part_floats(static_cast<int>(rows), cache->value_dim));
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
    p.scale = scale * 1.4426950408889634f;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t rows = shared_rows(*cache, *batch, heads);
    cudaError_t e;
    if (rows <= DEC_ROWS) {
        const int pieces = num_sms() * dec_warps(cache->key_dim, cache->value_dim);
        p.part_rows = static_cast<int>(rows);
        p.heads_of = static_cast<int4*>(workspace);
        p.part = reinterpret_cast<float*>(p.heads_of + pieces);
        e = dtype == EVA_DTYPE_BF16 ? decode_typed<__nv_bfloat16>(p, pieces, st) : decode_typed<__half>(p, pieces, st);
    } else {
        e = launch_prompt(p, workspace, dtype == EVA_DTYPE_BF16, st);
    }
    return e == cudaSuccess ? EVA_OK : EVA_ERR_CUDA;
}
