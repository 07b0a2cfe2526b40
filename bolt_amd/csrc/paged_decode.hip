// Attention of one new token per sequence over a paged cache. What bounds it is reading the keys and values once; the
// arithmetic is on the matrix cores so that it hides behind that, with the heads of a group (which share keys) as columns.
//
// A wave walks over its keys in steps of 32, all operands in registers (v_mfma_f32_16x16x32):
//   scores^T = K Q^T    lane (c = lane % 16, g = lane / 16) feeds eight d of key c and of query c; the result leaves it
//                       the scores of keys 4g .. 4g + 3 of both 16-key halves, for query c
//   out^T = V^T P^T     contraction over the 32 keys in the order the scores already lie in, so P goes in as it is. Row t of
//                       the lane's V operand is d = (DIM / 16) c + t of its own eight keys: each lane loads DIM / 16
//                       neighbouring d of eight keys (a 16-lane group reads whole rows) and pairs two keys' values per
//                       register with one byte permutation. Which d a result row means is then (DIM / 16) m + t.
// Neither LDS nor a transposed copy of V is needed. Weights are split into two 16-bit parts (their rounding would
// otherwise be as large as the output's); fp32 queries are, too, after a power of two brought their row into fp16's range.
// The running maximum is only raised once a score exceeds it by 2 (base 2). Over an fp16 or int8 cache weights are scaled by 2^13
// and stay below 2^15, inside fp16; a weight of less than 2^-37 of the row's largest is lost. Over a bf16 cache, whose values
// reach as far as fp32's, they are scaled by 2^-2 and stay below 1, so that their products overflow only where the plain formula's
// fp32 sums do. An int8 cache's steps (1 /
// scale) are part of the weights, divided by a power of two that no step seen so far exceeds: nothing leaves fp16 upwards, and a slot
// whose step is 2^k times another's takes k of the other's 37 powers of two.
//
// The tiles (of 128 keys) of all sequences stand in one row that is cut into equal shares, one to a workgroup, which fill the chip once:
// every workgroup reads the same number of bytes, whatever the lengths are. They are read on the device, so a captured launch
// serves any. A share may hold the end of one sequence, whole ones, and the beginning of another; a sequence that lies in one
// share is written out, one that several hold leaves (maximum, sum, output) parts, which a second launch joins.
//
// Two sequences of 104 k and 130 k keys, bf16, 8 key heads of 128 for 32 query heads: 0.96 GB in 142 us, 6.7 TB/s, where reading
// and nothing else reaches 7.0. 32 sequences of up to 4 k keys, fp16: 0.25 GB in 46 us, of which some 8 are the launch, the
// lists' and the first keys' way through memory one behind the other, and the last parts' way out; joining takes 4.5 us more.
#include "paged_device.h"

namespace bg {

namespace {

constexpr uint32_t kCus = 256;
constexpr uint32_t kTileShift = 7;   // keys of one round of a workgroup's four waves: 128

// workgroups of this kernel that a CU can hold (registers)
template <int DIM>
constexpr uint32_t per_cu()
{
    return DIM == 128 ? 2 : 3;
}

constexpr float kLow = -3.40282347e38f;  // running maximum before the first key: no score that is a number lies below
constexpr float kSlack = 2.0f;
template <int CT>
constexpr float kLift = CT == PT_BF16 ? -2.0f : 13.0f;  // see above: 2^(kSlack + kLift) fits fp16

__device__ __forceinline__ PagedSpan span_of(const PagedAttentionArgs &a, uint32_t b)
{
    return paged_span_newest(a.batch.lens[b], a.window, a.batch.max_pages << a.pool.shift);
}

// Tiles of a sequence, counted from its first key rounded down to a step of 32; one where there is nothing to see (somebody
// has to write the zeros). shift: kTileShift, more where sequences are left whole or the launch could have 2^31 tiles.
__device__ __forceinline__ uint32_t tiles_of(const PagedAttentionArgs &a, uint32_t b, uint32_t shift)
{
    const PagedSpan s = span_of(a, b);
    const uint32_t n = (s.hi - (s.lo & ~31u) + (1u << shift) - 1) >> shift;
    return n ? n : 1;
}

// tiles per share, with `shares` of them to a key head's column
__device__ __forceinline__ uint32_t tiles_per_share(uint32_t tiles, uint32_t shares)
{
    return (tiles + shares - 1) / shares;
}

// A part: 16 rows of DIM values, 16 maxima, 16 sums. A share leaves two at most: of the sequence that its first tile belongs to
// (slot 0), and of one that begins inside it and goes on behind it (slot 1).
__device__ __forceinline__ float *part_at(const PagedAttentionArgs &a, uint32_t shares, uint32_t column, uint32_t share, uint32_t slot, uint32_t dim)
{
    return (float *)a.ws + (((size_t)column * shares + share) * 2 + slot) * 16 * (dim + 2);
}

template <int ACT>
__device__ __forceinline__ void store_out4(void *out, size_t at, v4f v)
{
    if (ACT == PT_F32) {
        *(v4f *)((float *)out + at) = v;
    } else if (ACT == PT_F16) {
        typedef _Float16 v4h __attribute__((ext_vector_type(4)));
        *(v4h *)((uint16_t *)out + at) = (v4h){(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
        *(v2u *)((uint16_t *)out + at) = (v2u){pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    }
}

// What a lane holds of a step's keys and values, as they are stored. Bit j of seen: key 16 (j / 4) + 4 g + j % 4 takes part.
template <int CT, int DIM>
struct Step {
    typename CacheOperand<CT>::Raw kr[2][CacheOperand<CT>::kRawK(DIM)];
    typename CacheOperand<CT>::template RawV<DIM> vr[8];
    v4f ksc[2], vsc[2];
    uint32_t seen;
};

// PAGE16: pages of 16 keys and more, so that each 16-key half of a step lies in one page and its address is the wave's (32 requests
// fp16 50.9 us; with an address per lane, as smaller pages need it, 77.3).
// shares == 0: every sequence is one tile and has a workgroup.
// ONCE: up to 16 heads share a key head, so that one workgroup reads a key for all of them, past the caches; more take a
// workgroup per 16, which find it there (head size 128: 32 heads over 8, long bf16, 145 us past them and 166 through them;
// 64 over 2 66.6 and 55.1, 71 over 1 102 and 90).
template <int ACT, int CT, int DIM, bool PAGE16, bool ONCE>
__global__ __launch_bounds__(256, per_cu<DIM>()) void paged_decode_kernel(PagedAttentionArgs a, uint32_t shares, uint32_t shift)
{
    typedef CacheOperand<CT> Op;
    constexpr int kSteps = DIM / 32, kVec = DIM / 16;
    constexpr uint32_t kRowBytes = DIM * (CT == PT_I8 ? 1 : 2), kRow = DIM + 4;
    constexpr bool kSplitQ = ACT == PT_F32, kShiftQ = ACT == PT_F32 || (ACT == PT_BF16 && CT == PT_I8);
    __shared__ __attribute__((aligned(16))) float sO[4][16 * kRow];
    __shared__ float sM[4][16], sL[4][16];

    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c = lane & 15, g = lane >> 4;
    const uint32_t share = blockIdx.x, group = a.group.d, kvh = blockIdx.z, q0 = blockIdx.y * 16, column = kvh * ((group + 15) / 16) + blockIdx.y;
    const uint32_t nq = group - q0 < 16 ? group - q0 : 16;
    uint32_t per = 1, tile = share, before = share, b = share;  // tiles of a share; next tile of the row, those in front of its sequence
    if (shares) {
        auto tiles = [&](uint32_t i) { return tiles_of(a, i, shift); };
        const Places all = places_of(a.batch.batch, lane, tiles);
        per = tiles_per_share(all.sum, shares);
        if ((uint64_t)share * per >= all.sum) {
            return;
        }
        tile = share * per;
        b = entry_at(all, a.batch.batch, lane, tile, tiles, &before);
    }
    const uint32_t end = tile + per;
    for (;;) {
        b = __builtin_amdgcn_readfirstlane(b);
        const PagedSpan span = span_of(a, b);
        const uint32_t first = span.lo & ~31u, behind = before + tiles_of(a, b, shift);
        const uint32_t stop = min(behind, end);
        const uint32_t from = first + ((tile - before) << shift);
        const uint32_t to = min(first + ((stop - before) << shift), span.hi);
        const bool whole_sequence = tile == before && stop == behind;
        const int32_t *table = a.batch.table + (size_t)b * a.batch.max_pages;

        // queries
        typename Op::V qh[kSteps], ql[kSteps];
        float xscale = a.scale2;
        {
            float x[kSteps][8];
            const size_t at = (size_t)b * a.qstride + (size_t)(kvh * group + q0 + min(c, nq - 1)) * DIM;  // (columns behind the group: zeros)
            float top = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                load8<ACT>(a.q, at + Op::d_of(s, g), x[s]);
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[s][j] = c < nq ? x[s][j] : 0.0f;
                    if (kShiftQ) {
                        top = fmaxf(top, fabsf(x[s][j]));
                    }
                }
            }
            float up = 1.0f;
            if (kShiftQ) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                int e = 0;
                up = shift_into_f16(top, &e);
                xscale = ldexpf(a.scale2, e);
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                Op::split(x[s], up, &qh[s], &ql[s]);
            }
        }

        v4f o[kVec];
#pragma unroll
        for (int t = 0; t < kVec; ++t) {
            o[t] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        }
        float m = kLow, l = 0.0f, unit = CT == PT_I8 ? kFirstUnit : 1.0f;  // unit: the power of two that o's int8 steps are divided by

        // One step's 32 keys: list entries of its two halves a step ahead of its loads, those ahead of the arithmetic of the step before
        struct Pages {
            uint32_t p[2];
        };
        const uniform_list list = (uniform_list)table;
        auto look_up = [&](uint32_t k0) -> Pages {
            Pages r = {{0, 0}};
            if (PAGE16) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    r.p[h] = (uint32_t)list[min(k0 + 16 * h, to - 1) >> a.pool.shift];
                }
            }
            return r;
        };
        auto fetch = [&](uint32_t k0, const Pages &pages, Step<CT, DIM> &n) {
            n.seen = 0xff;
            if (PAGE16) {
                const uint8_t *kb[2], *vb[2];
                bool whole = k0 >= span.lo && k0 + 32 <= to;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t key = k0 + 16 * h;
                    const bool there = pages.p[h] < a.pool.pages && key < to;
                    const uint32_t page = there ? pages.p[h] : 0, in = there ? key & ((1u << a.pool.shift) - 1) : 0;
                    n.seen &= there ? 0xff : h ? 0x0f : 0xf0;
                    whole &= there;
                    const size_t slot = ((((size_t)page * a.pool.kv_heads + kvh) << a.pool.shift) | in);
                    kb[h] = (const uint8_t *)a.pool.k + slot * kRowBytes;
                    vb[h] = (const uint8_t *)a.pool.v + slot * kRowBytes;
                    if (CT == PT_I8) {
                        n.ksc[h] = load_scales(a.pool.ks + slot + 4 * g);
                        n.vsc[h] = load_scales(a.pool.vs + slot + 4 * g);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    Op::template load_k<ONCE>(kb[h] + c * kRowBytes, g, n.kr[h]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    n.vr[j] = Op::template load_v<ONCE, DIM>(vb[j >> 2] + (4 * g + (j & 3)) * kRowBytes, c);
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t key = k0 + 16 * (j >> 2) + 4 * g + (j & 3);
                        if (key < span.lo || key >= to) {
                            n.seen &= ~(1u << j);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t key = k0 + 16 * h + c;
                    int64_t slot = key < to ? paged_slot(table, key, a.pool.shift, a.pool.pages, a.pool.kv_heads, kvh) : -1;
                    Op::template load_k<ONCE>((const uint8_t *)a.pool.k + (slot < 0 ? 0 : slot) * kRowBytes, g, n.kr[h]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t key = k0 + 16 * (j >> 2) + 4 * g + (j & 3);
                    int64_t slot = key >= span.lo && key < to ? paged_slot(table, key, a.pool.shift, a.pool.pages, a.pool.kv_heads, kvh) : -1;
                    if (slot < 0) {
                        n.seen &= ~(1u << j);
                        slot = 0;
                    }
                    n.vr[j] = Op::template load_v<ONCE, DIM>((const uint8_t *)a.pool.v + slot * kRowBytes, c);
                    if (CT == PT_I8) {
                        n.ksc[j >> 2][j & 3] = a.pool.ks[slot];
                        n.vsc[j >> 2][j & 3] = a.pool.vs[slot];
                    }
                }
            }
        };
        auto attend = [&](Step<CT, DIM> &n) {
            v4f s[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s[h] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = 0; t < kSteps; ++t) {
                    const typename Op::V kv = Op::k_operand(n.kr[h], t);
                    s[h] = Op::mfma(kv, qh[t], s[h]);
                    if (kSplitQ) {
                        s[h] = Op::mfma(kv, ql[t], s[h]);
                    }
                }
            }
            float x[8], step[8], top = -INFINITY, wide = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float f = xscale;
                if (CT == PT_I8) {
                    f *= __builtin_amdgcn_rcpf(n.ksc[j >> 2][j & 3]);
                    step[j] = __builtin_amdgcn_rcpf(n.vsc[j >> 2][j & 3]);
                }
                x[j] = s[j >> 2][j & 3] * f;
            }
            if (n.seen != 0xff) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (!(n.seen >> j & 1)) {
                        x[j] = -INFINITY;
                        if (CT == PT_I8) {
                            step[j] = 0.0f;
                        } else {
                            n.vr[j] = Op::template zero_v<DIM>();
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                top = fmaxf(top, x[j]);
                if (CT == PT_I8) {
                    wide = fmaxf(wide, fabsf(step[j]));
                }
            }
            if (__any(top - m > kSlack || (CT == PT_I8 && wide > unit))) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float up = fmaxf(top, m);
                float corr = __builtin_amdgcn_exp2f(m - up);
                l *= corr;
                m = up;
                if (CT == PT_I8) {
                    const float was = unit;
                    wide = fmaxf(wide, unit);
#pragma unroll
                    for (int off = 32; off; off >>= 1) {
                        wide = fmaxf(wide, __shfl_xor(wide, off, 64));
                    }
                    unit = power_above(wide);
                    float now_unit = unit;
                    asm volatile("" : "+v"(now_unit));  // (else the reciprocal below is shared with this one, and the way round this block copies the outputs)
                    corr *= was * __builtin_amdgcn_rcpf(now_unit);
                }
#pragma unroll
                for (int t = 0; t < kVec; ++t) {
                    o[t] = o[t] * corr;
                }
            }
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = __builtin_amdgcn_exp2f(x[j] - m + kLift<CT>);
                l += p[j];
            }
            if (CT == PT_I8) {
                const float per_unit = __builtin_amdgcn_rcpf(unit);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] *= step[j] * per_unit;
                }
            }
            typename Op::V ph, pl;
            Op::split(p, 1.0f, &ph, &pl);
#pragma unroll
            for (int t = 0; t < kVec; ++t) {
                const typename Op::V vt = Op::template v_operand<DIM>(n.vr, t);
                o[t] = Op::mfma(vt, ph, o[t]);
                o[t] = Op::mfma(vt, pl, o[t]);
            }
        };
        uint32_t k0 = from + 32 * wave;
        if (k0 < to) {
            Step<CT, DIM> one, two;
            Pages pages = look_up(k0);
            fetch(k0, pages, one);
            pages = look_up(k0 + 128);
            // (behind the last step the first slot of the pool is read: a way round the loads would leave their number open, and what
            // is waited for with it)
            for (;;) {
                fetch(k0 + 128, pages, two);
                pages = look_up(k0 + 256);
                attend(one);
                k0 += 128;
                if (k0 >= to) {
                    break;
                }
                fetch(k0 + 128, pages, one);
                pages = look_up(k0 + 256);
                attend(two);
                k0 += 128;
                if (k0 >= to) {
                    break;
                }
            }
        }

        // the four waves' parts (addresses made anew: kept over the loop they would cost it registers)
        uint32_t me = threadIdx.x;
        asm volatile("" : "+v"(me));
        const uint32_t ec = me & 15, eg = me >> 4 & 3;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        // A sum of zero: the wave has seen no key, which a maximum of -inf says of it, or only scores of -inf
        if (__any(l == 0.0f)) {
            bool any = false;
            for (uint32_t key = from + 32 * wave + (lane & 31); key < to; key += 128) {
                any |= key >= span.lo && (uint32_t)table[key >> a.pool.shift] < a.pool.pages;
            }
            m = l == 0.0f && !__any(any) ? -INFINITY : m;
        }
        if (eg == 0) {
            sM[wave][ec] = m;
            sL[wave][ec] = l * kPartScale<CT>;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int t = 0; t < kVec; t += 4) {
                *(v4f *)(&sO[wave][ec * kRow + kVec * (4 * eg + i) + t]) = (v4f){o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]} * kPartScale<CT> * unit;
            }
        }
        __syncthreads();
        float *part = part_at(a, shares, column, share, tile != share * per, DIM);
        for (uint32_t at = me; at < nq * (DIM / 4); at += 256) {
            const uint32_t r = at / (DIM / 4), d = at % (DIM / 4) * 4;
            const float top = fmaxf(fmaxf(sM[0][r], sM[1][r]), fmaxf(sM[2][r], sM[3][r]));
            float sum = 0.0f;
            v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(sM[w][r] - fmaxf(top, kLow));
                sum += sL[w][r] * f;
                v += *(const v4f *)(&sO[w][r * kRow + d]) * f;
            }
            if (whole_sequence) {
                v = top == -INFINITY ? (v4f){0.0f, 0.0f, 0.0f, 0.0f} : v / sum;
                store_out4<ACT>(a.out, (size_t)b * a.ostride + (size_t)(kvh * group + q0 + r) * DIM + d, v);
            } else {
                *(v4f *)(part + r * DIM + d) = v;
                if (d == 0) {
                    part[16 * DIM + r] = top;
                    part[16 * DIM + 16 + r] = sum;
                }
            }
        }
        tile = stop;
        if (tile >= end || ++b >= a.batch.batch) {
            return;
        }
        before = behind;
        __syncthreads();  // the next sequence's parts go where these were
    }
}

// Joins the parts of split sequences: a workgroup per query head and sequence, DIM / 4 lanes to a part.
template <int ACT, int DIM>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttentionArgs a, uint32_t shares, uint32_t shift)
{
    constexpr uint32_t kLanes = DIM / 4, kWays = 256 / kLanes;
    __shared__ __attribute__((aligned(16))) float sO[kWays][DIM];
    __shared__ float sL[kWays], sM[kWays];
    const uint32_t lane = threadIdx.x & 63, h = blockIdx.x, b = blockIdx.y;
    uint32_t sum_all = 0, before = 0, mine = 0;  // tiles of all sequences, in front of sequence b, its own: every lane's part first
    for (uint32_t i = lane; i < a.batch.batch; i += 64) {
        const uint32_t n = tiles_of(a, i, shift);
        sum_all += n;
        before += i < b ? n : 0;
        mine = i == b ? n : mine;
    }
    sum_all = __builtin_amdgcn_readlane(wave_scan_u32(sum_all), 63);
    before = __builtin_amdgcn_readlane(wave_scan_u32(before), 63);
    mine = __builtin_amdgcn_readlane(mine, b % 64);
    const uint32_t per = tiles_per_share(sum_all, shares);
    const uint32_t first = before / per, count = (before + mine - 1) / per - first + 1;
    if (count == 1) {
        return;
    }
    const uint32_t qtiles = (a.group.d + 15) / 16, kvh = paged_div(h, a.group), in = h - kvh * a.group.d, r = in % 16;
    const float *part = part_at(a, shares, kvh * qtiles + in / 16, first, 0, DIM);
    const uint32_t slot = before % per != 0;  // of the first part; the others are the first of their share
    const uint32_t way = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
    float top = -INFINITY, sum = 0.0f;
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i = way; i < count; i += kWays) {
        const float *p = part + ((size_t)2 * i + (i ? 0 : slot)) * 16 * (DIM + 2);
        const float m = p[16 * DIM + r], up = fmaxf(top, m);
        const float from = fmaxf(up, kLow), f = __builtin_amdgcn_exp2f(top - from), e = __builtin_amdgcn_exp2f(m - from);
        sum = sum * f + p[16 * DIM + 16 + r] * e;
        v = v * f + *(const v4f *)(p + r * DIM + d) * e;
        top = up;
    }
    *(v4f *)(&sO[way][d]) = v;
    if (d == 0) {
        sM[way] = top;
        sL[way] = sum;
    }
    __syncthreads();
    if (way == 0) {
        float up = sM[0];
#pragma unroll
        for (uint32_t w = 1; w < kWays; ++w) {
            up = fmaxf(up, sM[w]);
        }
        sum = 0.0f;
        v = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < kWays; ++w) {
            const float f = __builtin_amdgcn_exp2f(sM[w] - fmaxf(up, kLow));
            sum += sL[w] * f;
            v += *(const v4f *)(&sO[w][d]) * f;
        }
        v = up == -INFINITY ? (v4f){0.0f, 0.0f, 0.0f, 0.0f} : v / sum;
        store_out4<ACT>(a.out, (size_t)b * a.ostride + (size_t)h * DIM + d, v);
    }
}

uint32_t columns(uint32_t heads, uint32_t kv_heads)
{
    return kv_heads * ((heads / kv_heads + 15) / 16);
}

// Shares of n columns with `fit` workgroups at a time: of the numbers that fill the chip once to four times, the first that
// leaves no more than a tenth idle, or else the one that leaves least. (96 key heads of 128, 1 x 20 k keys: 157 us, where the first
// that leaves no more than three tenths idle takes 175 and the one that leaves least 159; 6 ragged requests 114, 129 and 114.)
uint32_t shares_of(uint32_t n, uint32_t fit)
{
    uint32_t best = 1;
    double used = 0.0;
    for (uint32_t r = 1; r <= 4 && used < 0.9; ++r) {
        const uint32_t s = fit * r / n;
        if (s && (double)s * n / (fit * r) > used) {
            used = (double)s * n / (fit * r);
            best = s;
        }
    }
    return best;
}

uint32_t most_per_cu(uint32_t dim)
{
    return dim == 128 ? per_cu<128>() : per_cu<64>();
}

// Workgroups that a CU is given. Where memory is what bounds it, one (head size 64: two, whose loads are half as large) brings
// the bytes as fast as more, and leaves fewer parts to write and join: head size 128, one against two, 32 requests fp16 50.0
// and 50.9 us, 64 int8 106.6 and 109.4, two long ones bf16 145.6 and 150.2, seven heads to a key head 29.3 and 32.6; head
// size 64, two against three, fp32 over fp16 30.6 and 34.6, long bf16 81 and 84, and, the other way, 64 requests fp16 55.9 and 54.7. What an int8
// cache has to be converted for with smaller heads, and for fp32's two parts, takes one more: head size 128, fp32, 36.2
// against 38.9 with one; head size 64 37.8 against 40.2 with two. More waves than that spill or stand idle: head size 128,
// three, 85 us for 32 requests; head size 64, four, 62.
uint32_t wanted_per_cu(int act, int type, uint32_t dim)
{
    return (dim == 128 ? 1 : 2) + (type == PT_I8 && (act == PT_F32 || dim == 64));
}

// Few tiles, as far as the page table's width says, are spread over all that fit: eight requests of up to 2000 keys 14.3 us
// against 15.0.
uint32_t shares_for(const PagedAttentionArgs &a)
{
    const uint32_t n = columns(a.heads, a.pool.kv_heads), all = shares_of(n, kCus * most_per_cu(a.pool.dim));
    const uint64_t tiles = (uint64_t)a.batch.batch * ((((uint64_t)a.batch.max_pages << a.pool.shift) >> kTileShift) + 1);
    return tiles <= 2 * (uint64_t)all ? all : shares_of(n, kCus * wanted_per_cu(a.act, a.pool.type, a.pool.dim));
}

// keys that a sequence sees at most, from its first one rounded down to a step of 32 on
uint64_t most_seen(const PagedAttentionArgs &a)
{
    const uint64_t all = (uint64_t)a.batch.max_pages << a.pool.shift, in_window = (uint64_t)a.window + 31;
    return a.window && in_window < all ? in_window : all;
}

// Sequences of few keys are left whole, a workgroup to each and nothing to join, where they fill the chip all the same: up to 512
// keys (head size 128, 8 key heads, fp16, 32 sequences of up to 300 keys 9.6 us against 14.0 with their keys cut, 64 of up to
// 500 21.4 against 27.1, a window of 300 11.6 against 17.7; head size 64, 12 heads, fp32, 32 of up to 300 9.9 and 12.8), and up to
// 1024 where they also fill what a CU is given (32 of up to 1000 19.5 and 21.6, a window of 1000 23.7 and 30.4; head size 64,
// where they do not, 20.1 and 19.2). Longer ones differ too much in length: 64 of up to 2000 keys 66.7 and 54.8.
bool whole(const PagedAttentionArgs &a)
{
    const uint64_t seen = most_seen(a), groups = (uint64_t)a.batch.batch * columns(a.heads, a.pool.kv_heads);
    return (seen <= 512 + 31 && groups >= kCus) || (seen <= 1024 + 31 && groups >= kCus * wanted_per_cu(a.act, a.pool.type, a.pool.dim));
}

uint32_t tile_shift(const PagedAttentionArgs &a)
{
    const uint64_t seen = most_seen(a), positions = (uint64_t)a.batch.max_pages << a.pool.shift;
    uint32_t shift = kTileShift;
    while ((uint64_t)a.batch.batch * ((positions >> shift) + 2) > 0x7fffffffull || (whole(a) && 1u << shift < seen)) {
        ++shift;
    }
    return shift;
}

template <int ACT, int CT, int DIM>
struct Decode {
    static hipError_t run(const PagedAttentionArgs &a, hipStream_t st)
    {
        const uint32_t shift = tile_shift(a);
        const bool cut = most_seen(a) > 1u << shift;  // sequences of one tile never are
        const uint32_t shares = cut || !whole(a) ? shares_for(a) : 0;
        const dim3 grid(shares ? shares : a.batch.batch, (a.group.d + 15) / 16, a.pool.kv_heads);
        const bool once = a.heads / a.pool.kv_heads <= 16;
        const auto kernel = a.pool.shift >= 4 ? (once ? paged_decode_kernel<ACT, CT, DIM, true, true> : paged_decode_kernel<ACT, CT, DIM, true, false>)
                                              : (once ? paged_decode_kernel<ACT, CT, DIM, false, true> : paged_decode_kernel<ACT, CT, DIM, false, false>);
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a, shares, shift);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || !cut) {
            return e;
        }
        hipLaunchKernelGGL((paged_join_kernel<ACT, DIM>), dim3(a.heads, a.batch.batch), dim3(256), 0, st, a, shares, shift);
        return hipGetLastError();
    }
};

}  // namespace

size_t paged_decode_workspace(const PagedPool &pool, uint32_t heads)
{
    const uint32_t n = columns(heads, pool.kv_heads);
    uint32_t shares = 0;  // the most that a call may take
    for (uint32_t per = 1; per <= most_per_cu(pool.dim); ++per) {
        const uint32_t s = shares_of(n, kCus * per);
        shares = s > shares ? s : shares;
    }
    return (size_t)n * shares * 2 * 16 * (pool.dim + 2) * sizeof(float);
}

hipError_t launch_paged_decode(const PagedAttentionArgs &a, hipStream_t st)
{
    return a.batch.rows && a.batch.batch ? paged_dispatch<Decode>(a.act, a.pool.type, a.pool.dim, a, st) : hipSuccess;
}

}  // namespace bg
