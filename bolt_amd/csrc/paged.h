// Launchers of the paged key / value cache kernels. Device pointers; the C-ABI layer (api_paged.hip) has checked sizes,
// types and alignment; what stands in device memory (lengths, offsets, page numbers) the kernels check through
// paged_index.h.
#pragma once
#include "kernels.h"
#include "paged_index.h"

namespace bg {

enum PagedType : int { PT_F32 = 0, PT_F16 = 1, PT_BF16 = 2, PT_I8 = 3 };

struct PagedPool {
    void *k = nullptr, *v = nullptr;        // [pages][kv_heads][page_size][dim]
    float *ks = nullptr, *vs = nullptr;     // PT_I8: [pages][kv_heads][page_size], stored = real * scale
    uint32_t pages = 0, shift = 0, kv_heads = 0, dim = 0;  // page_size = 1 << shift
    int type = PT_F16;
};

struct PagedAppendArgs {
    PagedPool pool;
    PagedBatch batch;
    int act = PT_F32;                       // type of k, v, q, qout
    const void *k = nullptr, *v = nullptr, *q = nullptr;
    void *qout = nullptr;
    uint32_t kstride = 0, vstride = 0, qstride = 0, qostride = 0;  // elements between rows
    uint32_t heads = 0;                     // of q; 0: no queries
    const float *cos = nullptr, *sin = nullptr;  // [angles][rot / 2]
    uint32_t rot = 0, angles = 0;
    int interleaved = 0;
};
hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t st);

struct PagedAttentionArgs {
    PagedPool pool;
    PagedBatch batch;
    int act = PT_F32;                       // type of q and out
    const void *q = nullptr;
    void *out = nullptr;
    uint32_t qstride = 0, ostride = 0;      // elements between rows
    uint32_t heads = 0, window = 0;
    PagedDivisor kv_heads, group;           // group: heads that share a key head
    float scale2 = 0;                       // score scale * log2(e)
    void *ws = nullptr;
};
hipError_t launch_paged_decode(const PagedAttentionArgs &a, hipStream_t st);
size_t paged_decode_workspace(const PagedPool &pool, uint32_t heads);  // bytes
hipError_t launch_paged_prompt(const PagedAttentionArgs &a, hipStream_t st);
size_t paged_prompt_workspace(const PagedPool &pool, const PagedBatch &batch, uint32_t heads);  // bytes
bool paged_prompt_fits(const PagedPool &pool, const PagedBatch &batch, uint32_t heads);  // a grid of fewer than 2^32 threads, which is what a launch can have

}  // namespace bg
