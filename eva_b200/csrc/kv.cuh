// Shared by the paged-cache kernels: sequence and page lookup with every index checked, element access.
#pragma once

#include "common.cuh"
#include "internal.h"

namespace eva {

constexpr int KV_PAGE = EVA_KV_PAGE, KV_BLOCK = EVA_KV_BLOCK, KV_PAGE_BLOCKS = KV_PAGE / KV_BLOCK;
constexpr int ST_BAD_BATCH = EVA_STATUS_BAD_BATCH;

// The end of the kernel before this one in the stream (launch_after), and leave for the one behind to be launched.
__device__ __forceinline__ void after_previous()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Launch while the kernel before it in the stream still runs: a kernel launched so begins with after_previous(), which waits for that
// kernel's end and its writes. The four kernels of a decoding layer are a few us each, and their launches overlap this way.
template <typename... A>
inline cudaError_t launch_after(void (*kernel)(A...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Sequence b of a batch: its token rows row0 .. row0 + n - 1 are the positions ctx .. len - 1 (ctx may be
// negative: rows without a token). A sequence whose numbers do not fit the batch has no rows and no tokens.
struct KvSeq {
    int row0, n, len, ctx;
};

__device__ __forceinline__ KvSeq kv_seq(const EvaKvBatch& B, int b, int* status)
{
    const int r0 = B.q_start[b], r1 = B.q_start[b + 1], len = B.seq_lens[b];
    const bool ok = r0 >= 0 && r1 >= r0 && r1 <= B.tokens && r1 - r0 <= B.max_q && len >= 0 &&
                    len <= static_cast<int64_t>(B.max_pages) * KV_PAGE;
    if (!ok) {
        atomicOr(status, ST_BAD_BATCH);
        return {0, 0, 0, 0};
    }
    return {r0, r1 - r0, len, len - (r1 - r0)};
}

// Page that holds tokens 64 i .. 64 i + 63 of sequence b (i < max_pages), -1 where the table names none.
__device__ __forceinline__ int kv_page(const EvaKvCache& C, const EvaKvBatch& B, int b, int i, int* status)
{
    const int p = B.table[static_cast<int64_t>(b) * B.table_stride + i];
    if (p >= 0 && p < C.pages) return p;
    atomicOr(status, ST_BAD_BATCH);
    return -1;
}

// 2^(byte - 127) as a float (byte 0 as 2^-126: the smallest scale an append writes is byte 1)
__device__ __forceinline__ float kv_scale(uint32_t byte) { return __uint_as_float((byte ? byte : 1u) << 23); }

// cos and sin of `pos` steps of `turns` / 2^64 of a turn: the product modulo 2^64 is the exact fraction of a
// turn, whose upper 32 bits (a signed fraction in [-1/2, 1/2)) leave an angle error of 1e-7.
__device__ __forceinline__ float kv_half_turns(int64_t pos, uint64_t turns)
{
    return static_cast<float>(static_cast<int32_t>((static_cast<uint64_t>(pos) * turns) >> 32)) * 0x1p-31f;
}

// Argument checks shared by the entry points (no device work).
bool kv_cache_ok(const EvaKvCache* c);
bool kv_batch_ok(const EvaKvBatch* b);
bool rotary_ok(const EvaRotary* r, int head_dim);

}  // namespace eva
