// C-ABI entry points of the paged key / value cache: append with position rotation, attention of one new token per
// sequence, attention of prompts (device pointers, asynchronous).
#include <hip/hip_runtime.h>
#include <cstdint>

#include "api_internal.h"
#include "paged.h"

using namespace bg;
using namespace bgapi;

namespace {

EE refuse(const char *why)
{
    return fail(NOT_SUPPORTED, why);
}

EE contradict(const char *why)
{
    return fail(NOT_MATCH, why);
}

bool aligned16(const void *p)
{
    return ((uintptr_t)p & 15) == 0;
}

int paged_type(DataType dt)
{
    return dt == DT_F32 ? PT_F32 : dt == DT_F16 ? PT_F16 : dt == DT_BF16 ? PT_BF16 : dt == DT_I8 ? PT_I8 : -1;
}

EE check_pool(const BoltPagedKvCache *c, PagedPool *pool)
{
    if (!c || !c->k || !c->v) {
        return NULL_POINTER;
    }
    if (c->dt != DT_F16 && c->dt != DT_BF16 && c->dt != DT_I8) {
        return refuse("the cache holds DT_F16, DT_BF16 or DT_I8");
    }
    if (c->dt == DT_I8 && (!c->kScale || !c->vScale)) {
        return NULL_POINTER;
    }
    if (c->headDim != 64 && c->headDim != 128) {
        return refuse("head sizes 64 and 128");
    }
    if (c->pageSize == 0 || c->pageSize > 4096 || (c->pageSize & (c->pageSize - 1))) {
        return refuse("page sizes are powers of two up to 4096");
    }
    if (c->kvHeads == 0 || c->kvHeads > 1024 || c->numPages == 0 || c->numPages > 0x7fffffffu) {
        return refuse("1 to 1024 key heads, 1 to 2^31 - 1 pages");
    }
    if (!aligned16(c->k) || !aligned16(c->v) || ((uintptr_t)c->kScale & 3) || ((uintptr_t)c->vScale & 3)) {
        return refuse("the cache's keys and values start on 16-byte boundaries");
    }
    pool->k = c->k;
    pool->v = c->v;
    pool->ks = c->kScale;
    pool->vs = c->vScale;
    pool->pages = c->numPages;
    pool->shift = (uint32_t)__builtin_ctz(c->pageSize);
    pool->kv_heads = c->kvHeads;
    pool->dim = c->headDim;
    pool->type = paged_type(c->dt);
    return SUCCESS;
}

EE check_batch(const BoltPagedBatch *b, const PagedPool &pool, PagedBatch *batch)
{
    if (!b) {
        return NULL_POINTER;
    }
    if (b->batch && (!b->pageTable || !b->lengths)) {
        return NULL_POINTER;
    }
    if (b->batch > 65535 || b->maxPages == 0 || ((uint64_t)b->maxPages << pool.shift) > 0x7fffffffull || b->numTokens > 0x7fffffffu) {
        return refuse("up to 65535 sequences, 1 to 2^31 - 1 positions in a row of the page table, up to 2^31 - 1 rows");
    }
    if (!b->offsets && b->numTokens != b->batch) {
        return contradict("without offsets every sequence has one row: numTokens == batch");
    }
    if (((uintptr_t)b->pageTable | (uintptr_t)b->lengths | (uintptr_t)b->offsets) & 3) {
        return refuse("lists of 32-bit numbers start on 4-byte boundaries");
    }
    batch->table = b->pageTable;
    batch->lens = b->lengths;
    batch->offsets = b->offsets;
    batch->max_pages = b->maxPages;
    batch->batch = b->batch;
    batch->rows = b->numTokens;
    return SUCCESS;
}

// rows of `heads` head rows each, `stride` elements apart
EE check_rows(const void *p, U32 stride, U32 heads, U32 dim, U32 esize)
{
    if ((uint64_t)heads * dim > stride) {
        return contradict("a stride is at least a row's heads * headDim");
    }
    if (!aligned16(p) || ((uint64_t)stride * esize) % 16) {
        return refuse("rows start on 16-byte boundaries");
    }
    return SUCCESS;
}

EE check_types(DataType dt, const PagedPool &pool, U32 *esize)
{
    const bool wide = dt == DT_F32 || dt == DT_F16;
    if (!(wide && (pool.type == PT_F16 || pool.type == PT_I8)) && !(dt == DT_BF16 && (pool.type == PT_BF16 || pool.type == PT_I8))) {
        return refuse("DT_F32 or DT_F16 over a DT_F16 or DT_I8 cache, DT_BF16 over a DT_BF16 or DT_I8 cache");
    }
    *esize = dt == DT_F32 ? 4 : 2;
    return SUCCESS;
}

EE check_heads(U32 heads, const PagedPool &pool)
{
    if (heads == 0 || heads > 16384) {
        return refuse("1 to 16384 query heads");
    }
    return heads % pool.kv_heads ? contradict("the query heads are a multiple of the key heads") : SUCCESS;
}

EE check_grid(const PagedPool &pool, const PagedBatch &batch, U32 heads)
{
    return !batch.offsets || paged_prompt_fits(pool, batch, heads) ? SUCCESS : refuse("more rows times heads than a launch can have");
}

#define EE_TRY(expr)            \
    do {                        \
        const EE ee__ = (expr); \
        if (ee__ != SUCCESS) {  \
            return ee__;        \
        }                       \
    } while (0)

// zero rows or sequences: nothing is launched
size_t workspace_bytes(const PagedPool &pool, const PagedBatch &batch, U32 heads)
{
    if (batch.batch == 0 || batch.rows == 0) {
        return 256;
    }
    return batch.offsets ? paged_prompt_workspace(pool, batch, heads) : paged_decode_workspace(pool, heads);
}

EE attention(const BoltPagedKvCache *cache, const BoltPagedBatch *batch, DataType dt, U32 heads, const void *q, U32 qStride, void *out,
    U32 outStride, F32 scale, U32 window, void *workspace, size_t workspaceBytes, bool decode)
{
    PagedAttentionArgs a;
    U32 esize = 0;
    EE_TRY(check_pool(cache, &a.pool));
    EE_TRY(check_batch(batch, a.pool, &a.batch));
    EE_TRY(check_types(dt, a.pool, &esize));
    EE_TRY(check_heads(heads, a.pool));
    EE_TRY(check_grid(a.pool, a.batch, heads));
    if (decode && a.batch.offsets) {
        return contradict("decode takes one row per sequence: offsets == NULL");
    }
    if (!decode && a.batch.batch && !a.batch.offsets) {
        return NULL_POINTER;
    }
    if (a.batch.batch == 0 || a.batch.rows == 0) {
        return SUCCESS;
    }
    if (!q || !out || !workspace) {
        return NULL_POINTER;
    }
    EE_TRY(check_rows(q, qStride, heads, a.pool.dim, esize));
    EE_TRY(check_rows(out, outStride, heads, a.pool.dim, esize));
    if (q == out) {
        return refuse("out must not overlap q");
    }
    if ((uintptr_t)workspace & 255) {
        return refuse("the workspace starts on a 256-byte boundary");
    }
    if (workspaceBytes < workspace_bytes(a.pool, a.batch, heads)) {
        return contradict("the workspace is smaller than bolt_gfx950_paged_attention_workspace_bytes asks for");
    }
    EE_TRY(ensure_init());
    a.act = paged_type(dt);
    a.q = q;
    a.out = out;
    a.qstride = qStride;
    a.ostride = outStride;
    a.heads = heads;
    a.window = window;
    a.kv_heads = paged_divisor(a.pool.kv_heads);
    a.group = paged_divisor(heads / a.pool.kv_heads);
    a.scale2 = scale * 1.44269504088896340736f;  // exp(x) = exp2(x log2(e))
    a.ws = workspace;
    HIP_TRY(decode ? launch_paged_decode(a, ctx().stream) : launch_paged_prompt(a, ctx().stream));
    return SUCCESS;
}

}  // namespace

extern "C" {

EE bolt_gfx950_kv_cache_append(const BoltPagedKvCache *cache, const BoltPagedBatch *batch, DataType dt, const void *k,
    U32 kStride, const void *v, U32 vStride, U32 heads, const void *q, U32 qStride, void *qOut, U32 qOutStride,
    const BoltRotary *rotary)
{
    PagedAppendArgs a;
    U32 esize = 0;
    EE_TRY(check_pool(cache, &a.pool));
    EE_TRY(check_batch(batch, a.pool, &a.batch));
    EE_TRY(check_types(dt, a.pool, &esize));
    if (heads) {
        EE_TRY(check_heads(heads, a.pool));
    }
    if (rotary) {
        if (!rotary->cosine || !rotary->sine) {
            return NULL_POINTER;
        }
        if (rotary->dim == 0 || rotary->dim % 16 || rotary->dim > a.pool.dim) {
            return refuse("the rotated part of a head is a multiple of 16 elements, up to headDim");
        }
        if (!aligned16(rotary->cosine) || !aligned16(rotary->sine)) {
            return refuse("tables of angles start on 16-byte boundaries");
        }
        a.cos = rotary->cosine;
        a.sin = rotary->sine;
        a.rot = rotary->dim;
        a.angles = rotary->positions;
        a.interleaved = rotary->interleaved != 0;
    }
    if (a.batch.batch == 0 || a.batch.rows == 0) {
        return SUCCESS;
    }
    if (!k || !v || (heads && (!q || !qOut))) {
        return NULL_POINTER;
    }
    EE_TRY(check_rows(k, kStride, a.pool.kv_heads, a.pool.dim, esize));
    EE_TRY(check_rows(v, vStride, a.pool.kv_heads, a.pool.dim, esize));
    if (heads) {
        EE_TRY(check_rows(q, qStride, heads, a.pool.dim, esize));
        EE_TRY(check_rows(qOut, qOutStride, heads, a.pool.dim, esize));
        if (q == qOut && qStride != qOutStride) {
            return contradict("queries rotated in place keep their stride");
        }
    }
    EE_TRY(ensure_init());
    a.act = paged_type(dt);
    a.k = k;
    a.v = v;
    a.q = q;
    a.qout = qOut;
    a.kstride = kStride;
    a.vstride = vStride;
    a.qstride = qStride;
    a.qostride = qOutStride;
    a.heads = heads;
    HIP_TRY(launch_paged_append(a, ctx().stream));
    return SUCCESS;
}

EE bolt_gfx950_paged_attention_workspace_bytes(const BoltPagedKvCache *cache, const BoltPagedBatch *batch, U32 heads, size_t *bytes)
{
    PagedPool pool;
    PagedBatch b;
    if (!bytes) {
        return NULL_POINTER;
    }
    EE_TRY(check_pool(cache, &pool));
    EE_TRY(check_batch(batch, pool, &b));
    EE_TRY(check_heads(heads, pool));
    EE_TRY(check_grid(pool, b, heads));
    *bytes = workspace_bytes(pool, b, heads);
    return SUCCESS;
}

EE bolt_gfx950_paged_attention_decode(const BoltPagedKvCache *cache, const BoltPagedBatch *batch, DataType dt, U32 heads,
    const void *q, U32 qStride, void *out, U32 outStride, F32 scale, U32 window, void *workspace, size_t workspaceBytes)
{
    return attention(cache, batch, dt, heads, q, qStride, out, outStride, scale, window, workspace, workspaceBytes, true);
}

EE bolt_gfx950_paged_attention_prompt(const BoltPagedKvCache *cache, const BoltPagedBatch *batch, DataType dt, U32 heads,
    const void *q, U32 qStride, void *out, U32 outStride, F32 scale, U32 window, void *workspace, size_t workspaceBytes)
{
    return attention(cache, batch, dt, heads, q, qStride, out, outStride, scale, window, workspace, workspaceBytes, false);
}

}  // extern "C"
