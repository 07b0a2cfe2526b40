// Paged key / value cache: storing the keys and values of new tokens, with the position rotation of keys and queries on the
// way.
#include "paged_device.h"

namespace bg {

// ---- append -----------------------------------------------------------------------------------------
// One workgroup per packed row; DIM / 16 lanes per head row, query heads first, then keys, then values. A lane owns two
// runs of eight elements: the two halves of eight rotated pairs (pairs i, i + rot / 2), or 16 neighbours (pairs 2i, 2i + 1,
// and the elements behind the rotated part). Every step is one fp32 operation in the order the plain formula has it:
//   a' = a * cos - b * sin,  b' = b * cos + a * sin
// rounded once to the stored type. An int8 slot gets s = (1 / max|x|) * 127 (1 for an all-zero row) and q = rne(x * s).
// What bounds it is memory: every element is read once and written once. 16265 rows of 32 query and 2 x 8 key / value heads of
// 128, bf16, are 0.40 GB and take 80 us, 5.0 TB/s, what a copy of 2 GiB reaches (4.9). The rows' elements are asked for before
// anything else, and whose row it is by all lanes at once, so that a row waits twice for memory and not once per step of a
// search: 16 rows take 3.7 us on the GPU, where the host takes 10 for the call. 512 threads to a row, each 16 elements of up to
// two heads: with 256 the 16 rows take 1 us more, with 1024 nothing changes.
constexpr uint32_t kRowsX = 20;  // log2 of the rows along the grid's x extent: a launch has fewer than 2^32 threads there

template <int ACT, int CT, int DIM>
__global__ void paged_append_kernel(PagedAppendArgs a)
{
    constexpr uint32_t kLanes = DIM / 16;
    const uint32_t row = blockIdx.y << kRowsX | blockIdx.x, lane = threadIdx.x & 63;
    if (row >= a.batch.rows) {
        return;
    }
    const uint32_t kvh = a.pool.kv_heads, heads = a.heads + 2 * kvh;
    struct Item {
        uint32_t head, l, h, e0, e1;  // head row among all, run of 16 elements in it, head among its kind, where its halves are
        bool is_q, is_v, turned;
        float x[16];
    };
    auto load = [&](uint32_t item, Item &n) {
        n.head = item / kLanes;
        n.l = item % kLanes;
        n.is_q = n.head < a.heads;
        n.is_v = n.head >= a.heads + kvh;
        n.h = n.is_q ? n.head : n.is_v ? n.head - a.heads - kvh : n.head - a.heads;
        n.turned = !n.is_v && 16 * n.l < a.rot;
        n.e0 = n.turned && !a.interleaved ? 8 * n.l : 16 * n.l;
        n.e1 = n.turned && !a.interleaved ? a.rot / 2 + 8 * n.l : 16 * n.l + 8;
        const void *src = n.is_q ? a.q : n.is_v ? a.v : a.k;
        const size_t base = (size_t)row * (n.is_q ? a.qstride : n.is_v ? a.vstride : a.kstride) + (size_t)n.h * DIM;
        load8<ACT>(src, base + n.e0, n.x);
        load8<ACT>(src, base + n.e1, n.x + 8);
    };
    Item n;
    if (threadIdx.x < heads * kLanes) {
        load(threadIdx.x, n);
    }
    uint32_t b;
    PagedSeq s;
    if (!a.batch.offsets || a.batch.batch > 64) {
        b = paged_owner(a.batch, row);
        s = paged_seq(a.batch, b);
    } else {
        const uint32_t last = a.batch.batch - 1, mine = min(lane, last);
        const int32_t first = a.batch.offsets[mine], next = a.batch.offsets[mine + 1], len = a.batch.lens[mine];
        const unsigned long long reached = __ballot(lane <= last && (int64_t)first <= (int64_t)row);
        b = reached ? 63 - (uint32_t)__builtin_clzll(reached) : 0;
        s = paged_seq_from(__builtin_amdgcn_readlane(first, b), __builtin_amdgcn_readlane(next, b), __builtin_amdgcn_readlane(len, b));
    }
    const int64_t i = (int64_t)row - s.first, pos = s.pos + i;
    if (i < 0 || i >= s.count || pos < 0 || (a.rot && pos >= (int64_t)a.angles)) {
        return;
    }
    // (without a slot nothing is stored; the query is turned all the same)
    const int64_t slot0 = pos >= (int64_t)a.batch.max_pages << a.pool.shift ? -1 : paged_slot(a.batch.table + (size_t)b * a.batch.max_pages, (uint32_t)pos, a.pool.shift, a.pool.pages, kvh, 0);
    for (uint32_t item = threadIdx.x; item < heads * kLanes;) {
        const uint32_t l = n.l, h = n.h, e0 = n.e0, e1 = n.e1;
        const bool is_q = n.is_q, is_v = n.is_v, turned = n.turned;
        float (&x)[16] = n.x;
        if (turned) {
            const size_t at = (size_t)pos * (a.rot / 2) + 8 * l;
            float c[8], sn[8];
            load8<PT_F32>(a.cos, at, c);
            load8<PT_F32>(a.sin, at, sn);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float u = a.interleaved ? x[2 * j] : x[j], w = a.interleaved ? x[2 * j + 1] : x[8 + j];
                const float ra = u * c[j] - w * sn[j], rb = w * c[j] + u * sn[j];
                if (a.interleaved) {
                    x[2 * j] = ra;
                    x[2 * j + 1] = rb;
                } else {
                    x[j] = ra;
                    x[8 + j] = rb;
                }
            }
        }
        if (is_q) {
            const size_t to = (size_t)row * a.qostride + (size_t)h * DIM;
            store8<ACT>(a.qout, to + e0, x);
            store8<ACT>(a.qout, to + e1, x + 8);
        }
        const int64_t slot = slot0 < 0 || is_q ? -1 : slot0 + ((int64_t)h << a.pool.shift);
        void *dst = is_v ? a.pool.v : a.pool.k;
        if (CT == PT_I8) {
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float v = fabsf(x[j]);
                top = v > top || v != v ? v : top;  // a NaN makes the slot's scale NaN, so that what reads it shows it
            }
#pragma unroll
            for (uint32_t off = 1; off < kLanes; off <<= 1) {
                const float v = __shfl_xor(top, off, kLanes);
                top = v > top || v != v ? v : top;
            }
            // (the reciprocal of a subnormal maximum is infinite: the largest number stands in for it)
            float scale = 1.0f / top * 127.0f;
            scale = top == 0.0f ? 1.0f : scale > 3.40282347e38f ? 3.40282347e38f : scale;
            if (slot >= 0) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = 0;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        int v = rne_i32(x[4 * j + t] * scale);
                        v = v < -127 ? -127 : (v > 127 ? 127 : v);
                        w[j] |= ((uint32_t)v & 0xffu) << (8 * t);
                    }
                }
                int8_t *o = (int8_t *)dst + (size_t)slot * DIM;
                *(v2u *)(o + e0) = (v2u){w[0], w[1]};
                *(v2u *)(o + e1) = (v2u){w[2], w[3]};
                if (l == 0) {
                    (is_v ? a.pool.vs : a.pool.ks)[slot] = scale;
                }
            }
        } else if (slot >= 0) {
            store8<CT>(dst, (size_t)slot * DIM + e0, x);
            store8<CT>(dst, (size_t)slot * DIM + e1, x + 8);
        }
        item += blockDim.x;
        if (item < heads * kLanes) {
            load(item, n);
        }
    }
}

namespace {

template <int ACT, int CT, int DIM>
struct Append {
    static hipError_t run(const PagedAppendArgs &a, hipStream_t st)
    {
        const uint32_t items = (a.heads + 2 * a.pool.kv_heads) * (DIM / 16);
        const uint32_t threads = items >= 512 ? 512 : (items + 63) / 64 * 64;
        const uint32_t x = a.batch.rows < 1u << kRowsX ? a.batch.rows : 1u << kRowsX;
        hipLaunchKernelGGL((paged_append_kernel<ACT, CT, DIM>), dim3(x, (a.batch.rows + x - 1) / x), dim3(threads), 0, st, a);
        return hipGetLastError();
    }
};

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t st)
{
    return a.batch.rows && a.batch.batch ? paged_dispatch<Append>(a.act, a.pool.type, a.pool.dim, a, st) : hipSuccess;
}

}  // namespace bg
