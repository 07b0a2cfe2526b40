// Attention of prompts over a paged cache: many new tokens per sequence, each seeing the keys up to its own. What bounds it
// is the matrix cores.
//
// Rows of a tile are (token, head of a group) pairs, R = token * group + head: the heads of a group share keys, so a short
// prompt of a grouped model still fills a tile. A workgroup owns 128 rows of one (sequence, key head), each of its four waves
// 32, and walks over the keys it needs in tiles of 64 (v_mfma_f32_32x32x16):
//   scores^T = K Q^T   lane (c = lane % 32, h = lane / 32) feeds eight d of key c (from LDS) and of row c (registers); the
//                      result leaves it, for row c, the scores of keys 8 i + 4 h + 0..3, i = 0..3, of each half of the tile
//   out^T = V^T P^T    contraction over the keys in the order the scores lie in: P goes from the accumulators into the
//                      operand with no exchange between lanes; V^T comes from LDS through the transposing read
//                      (ds_read_b64_tr_b16: a lane gets four keys' values of one d)
// Key and value tiles of a 16-bit cache go from memory to LDS without passing registers, one tile ahead, in pieces of 16
// bytes; the pieces of a row are permuted so that 16 lanes of either read pattern touch all banks. An int8 cache's are read
// into registers two tiles ahead and put into LDS as fp16, which holds its values exactly, between the products of the tile
// before theirs (a tile waits for one barrier and no load); its steps multiply scores and weights.
//
// What it costs. A wave issues 32 products of 32x32x16 a tile (head size 128; 36.5 cycles each alone, 44 with real data,
// when the clock falls) and some 200 vector instructions (int8: 400), 32 of them exponentials, and it does not overlap its
// own products with them: two waves on every SIMD, from two workgroups, do. One prompt of 8192 tokens, 32 heads over 8, bf16,
// takes 0.55 ms, 1.0 PFLOP/s, where the library's 8192^3 product of the same type reaches 1.2; 2 x 256 tokens over 27 k
// int8 keys 0.158 ms, 0.71 PFLOP/s. Head size 128 takes 215 to 242 registers of the 256 that two waves leave each; more
// rows to a wave would halve the reads of LDS and do not fit.
// Where few tiles meet many keys, several workgroups share a tile's keys and a second launch joins their parts.
#include <atomic>

#include "paged_device.h"

namespace bg {

namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(1))) void *gptr_t;
typedef __attribute__((address_space(3))) void *lptr_t;
typedef __attribute__((address_space(3))) uint8_t *lds_t;

constexpr uint32_t kRows = 128, kKeys = 64;
// Workgroups (two a CU) below which a tile's keys are shared out, over about so many. 2 x 256 new tokens over 27 k int8 keys, 128 tiles
// of rows: 153 us with 512, 204 with 256 (half the chip idle), 174 with 1024 (more parts written and read). Eight ragged
// prompts of up to 1025 tokens have more tiles than that: 99 us with whole tiles, 153 with their keys cut in two.
constexpr uint32_t kSpread = 512;
// Fewest key tiles per share. 20 tokens over 2000 keys, fp16, 32 heads over 8: 15.1 us with 4, 14.9 with 2, 22.2 with 1 (more parts to
// write and join than keys to share), 19.2 with 8; 100 over 700: 17.1, 16.5, 21.5, 19.6.
constexpr uint32_t kLeast = 4;
constexpr float kLow = -3.40282347e38f;  // running maximum before the first key: no score that is a number lies below
// A row's running maximum is raised once a score exceeds it by kSlack (base 2; the difference is exact where it counts, m + kSlack need
// not be), and by nothing but what the row sees, whatever
// the wave's others do: what they see must not change how it is rounded. Weights are scaled by 2^kLift and stay below 2^15.75,
// inside fp16; in bf16, whose values reach as far as fp32's, below 1. (Raising outputs costs, so that bf16 takes as much slack as is
// of use: 8192 tokens 543 us, with 2 560.)
template <int CT>
constexpr float kSlack = CT == PT_BF16 ? 8.0f : 2.75f;
template <int CT>
constexpr float kLift = CT == PT_BF16 ? -8.0f : 13.0f;

// rows (token, head) of a sequence in tiles of kRows; no more tokens than the buffers have rows, so that it all fits 31 bits
__device__ __forceinline__ uint32_t rows_of(const PagedAttentionArgs &a, const PagedSeq &s)
{
    return (s.count < (int64_t)a.batch.rows ? (uint32_t)s.count : a.batch.rows) * a.group.d;
}

// Row tile number x of the launch: its sequence and its number there. What takes longest starts first: the longest sequence
// (of up to 64, of more the last one), and of a sequence the last tile, which sees the most keys.
__device__ __forceinline__ bool find_tile(const PagedAttentionArgs &a, uint32_t x, uint32_t lane, uint32_t *b_out, uint32_t *tile, PagedSeq *seq)
{
    const uint32_t n = a.batch.batch;
    if (n <= 64) {  // everything that is needed is asked for at once
        const uint32_t mine = lane < n ? lane : n - 1;
        const int32_t first = a.batch.offsets[mine], next = a.batch.offsets[mine + 1], keys = lane < n ? a.batch.lens[mine] : -0x7fffffff - 1;
        const uint32_t tiles = lane < n ? (rows_of(a, paged_seq_from(first, next, keys)) + kRows - 1) / kRows : 0;
        uint32_t before = 0;  // tiles of longer sequences, and of those in front that are as long
        for (uint32_t i = 0; i < n; ++i) {
            const int32_t other = __builtin_amdgcn_readlane(keys, i);
            before += other > keys || (other == keys && i < lane) ? (uint32_t)__builtin_amdgcn_readlane(tiles, i) : 0;
        }
        const unsigned long long here = __ballot(x >= before && x - before < tiles);
        const uint32_t at = here ? (uint32_t)__builtin_ctzll(here) : 0;
        *b_out = at;
        *tile = __builtin_amdgcn_readlane(tiles, at) - 1 - (x - __builtin_amdgcn_readlane(before, at));
        *seq = paged_seq_from(__builtin_amdgcn_readlane(first, at), __builtin_amdgcn_readlane(next, at), __builtin_amdgcn_readlane(keys, at));
        return here != 0;
    }
    auto count = [&](uint32_t i) { return (rows_of(a, paged_seq(a.batch, i)) + kRows - 1) / kRows; };
    const Places all = places_of(n, lane, count);
    if (x >= all.sum) {
        return false;
    }
    uint32_t before;
    const uint32_t b = __builtin_amdgcn_readfirstlane(entry_at(all, n, lane, all.sum - 1 - x, count, &before));
    *b_out = b;
    *tile = __builtin_amdgcn_readfirstlane(all.sum - 1 - x - before);
    *seq = paged_seq(a.batch, b);
    return true;
}

// What a tile's rows see: positions of the first and last row, keys [lo, hi) with lo rounded down to a tile
struct Reach {
    int64_t first, last;
    uint32_t lo, hi, tiles;
};

__device__ __forceinline__ Reach reach_of(const PagedAttentionArgs &a, const PagedSeq &s, uint32_t rows, uint32_t tile)
{
    Reach r;
    const uint32_t r0 = tile * kRows, r1 = min(r0 + kRows, rows);
    r.first = s.pos + paged_div(r0, a.group);
    r.last = s.pos + paged_div(r1 - 1, a.group);
    const uint32_t capacity = a.batch.max_pages << a.pool.shift;
    r.hi = paged_span(r.last, a.window, capacity).hi;
    r.lo = paged_span(r.first > 0 ? r.first : 0, a.window, capacity).lo & ~(kKeys - 1);
    r.tiles = r.hi > r.lo ? (r.hi - r.lo + kKeys - 1) / kKeys : 0;
    return r;
}

__device__ __forceinline__ uint32_t tiles_per_share(uint32_t tiles, const PagedDivisor &shares)
{
    const uint32_t n = paged_div(tiles + shares.d - 1, shares);
    return n < kLeast ? kLeast : n;
}

// A share's part: 128 rows of DIM values, 128 maxima, 128 sums
__device__ __forceinline__ float *part_at(const PagedAttentionArgs &a, uint32_t x, uint32_t kvh, uint32_t share, uint32_t shares, uint32_t dim)
{
    return (float *)a.ws + (((size_t)x * a.pool.kv_heads + kvh) * shares + share) * kRows * (dim + 2);
}

// place of 16-byte piece `piece` of row `row` in a tile's LDS image (units of 16 bytes)
template <int DIM>
__device__ __forceinline__ uint32_t swizzle_k(uint32_t row)
{
    return DIM == 128 ? row & 15 : (row >> 1) & 7;
}

template <int DIM>
__device__ __forceinline__ uint32_t swizzle_v(uint32_t row)
{
    return DIM == 128 ? (row & 3) << 2 | ((row >> 2) & 3) : ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
}

// no instruction is moved across
__device__ __forceinline__ void in_order()
{
    __builtin_amdgcn_sched_barrier(0);
}

// One instruction; a NaN wins, and makes its row's weights NaN anyway (fmaxf has the operands quieted first, one more each)
__device__ __forceinline__ float max_of(float a, float b, float c)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

constexpr float kLargeScore = 262144.0f;  // 2^18: half an fp32 step of it is 2^-6

// int8: the steps of a tile's keys (times the score scale) and values, values whose step is not finite, and the power of two above
// the largest step. Values' steps three times: over `unit`, for rows that see the whole tile; as they are and times 2^-80, for
// rows that do not, whose own largest step may be any number of powers of two below `unit`.
enum { kStepK, kStepV, kStepOwn, kStepOwnLow };
constexpr float kLowStep = 8.27180613e-25f;  // 2^-80
struct StepsOfTile {
    float step[4][kKeys];
    unsigned long long bad;
    float unit, unused;
};

// the workgroup's barrier behind its LDS accesses, without a wait for loads from memory, which __syncthreads() has
__device__ __forceinline__ void barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int CT>
struct Product {
    typedef v8h V;
    static __device__ __forceinline__ v16f mfma(V a, V b, v16f c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    // l + both values of a pair
    static __device__ __forceinline__ float add_pair(uint32_t w, float l)
    {
        typedef _Float16 v2h __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, w), (v2h){(_Float16)1.0f, (_Float16)1.0f}, l, false);
    }
    // two values rounded to nearest
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        typedef _Float16 v2h __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, v2h));
    }
};
template <>
struct Product<PT_BF16> {
    typedef v8b V;
    static __device__ __forceinline__ v16f mfma(V a, V b, v16f c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float add_pair(uint32_t w, float l)
    {
        typedef __bf16 v2b __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, w), (v2b){(__bf16)1.0f, (__bf16)1.0f}, l, false);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        typedef __bf16 v2b __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, v2b));
    }
};

template <int ACT>
__device__ __forceinline__ void store_out4(void *out, size_t at, float a, float b, float c, float d)
{
    if (ACT == PT_F32) {
        *(v4f *)((float *)out + at) = (v4f){a, b, c, d};
    } else if (ACT == PT_F16) {
        *(v2u *)((uint16_t *)out + at) = (v2u){Product<PT_F16>::pack(a, b), Product<PT_F16>::pack(c, d)};
    } else {
        *(v2u *)((uint16_t *)out + at) = (v2u){Product<PT_BF16>::pack(a, b), Product<PT_BF16>::pack(c, d)};
    }
}

template <int CT, int DIM>
constexpr uint32_t prompt_lds()
{
    return 4 * kKeys * DIM * 2 + (CT == PT_I8 ? 2 * sizeof(StepsOfTile) : DIM * 16 + 4 * 4 + 4);
}

// rows of a tile that one load of a wave brings
template <int CT, int DIM>
constexpr uint32_t rows_at()
{
    return 64 / (DIM * (CT == PT_I8 ? 1 : 2) / 16);
}

template <int ACT, int CT, int DIM, bool PAGED>
__global__ __launch_bounds__(256, 2) void paged_prompt_kernel(PagedAttentionArgs a, PagedDivisor shares)
{
    typedef Product<CT> Op;
    typedef typename Op::V V;
    constexpr bool kWide = ACT == PT_F32;                                            // two parts per operand
    constexpr bool kShiftQ = kWide || (ACT == PT_BF16 && CT == PT_I8);
    constexpr uint32_t kTileBytes = kKeys * DIM * 2, kRowBytes = DIM * (CT == PT_I8 ? 1 : 2), kPieces = DIM / 8;
    constexpr int kSteps = DIM / 16, kOut = DIM / 32, kLoads = kKeys * kRowBytes / 16 / 256;
    // LDS: two buffers, each a tile of keys and one of values in 16 bits; behind them
    //   16-bit caches: [DIM][128 rows as bits] rows that see a value which is not finite, [4] whether a wave found one, whether there is any
    //   int8: two buffers of steps
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    lds_t const sTiles = (lds_t)0;  // smem's own address: the kernel has no other LDS. As a constant it goes into the reads' offsets.
    constexpr uint32_t kBehind = 4 * kTileBytes;
    StepsOfTile *const sSteps = (StepsOfTile *)(smem + kBehind);
    uint32_t *const sPoison = (uint32_t *)(smem + kBehind), *const sHit = sPoison + 4 * DIM, *const sAny = sHit + 4;

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t c = lane & 31, h = lane >> 5;
    const uint32_t column = paged_div(blockIdx.x, a.kv_heads), kvh = blockIdx.x - column * a.kv_heads.d;
    const uint32_t x = paged_div(column, shares), share = column - x * shares.d, group = a.group.d;
    uint32_t b, tile_index;
    PagedSeq seq;
    if (!find_tile(a, x, lane, &b, &tile_index, &seq)) {
        return;
    }
    const uint32_t rows = rows_of(a, seq);
    const Reach all = reach_of(a, seq, rows, tile_index);
    const uint32_t per = tiles_per_share(all.tiles, shares);
    const uint32_t t0 = share * per, t1 = min(t0 + per, all.tiles);
    if (share && t0 >= all.tiles) {
        return;
    }
    const bool alone = per >= all.tiles;
    const int32_t *table = a.batch.table + (size_t)b * a.batch.max_pages;

    // this lane's row
    const uint32_t r = tile_index * kRows + 32 * wave + c, token = paged_div(r, a.group);
    const int64_t row = seq.first + token, pos = seq.pos + token;
    const bool idle = tile_index * kRows + 32 * wave >= rows;  // (the wave's)
    const bool mine = r < rows && row >= 0 && row < (int64_t)a.batch.rows;
    const uint32_t head = kvh * group + (r - token * group);
    const PagedSpan span = paged_span(mine ? pos : -1, a.window, all.hi);

    const uint32_t all_hi = paged_span(all.first, 0, all.hi).hi, all_lo = paged_span(all.last, a.window, all.hi).lo;  // seen by every row

    V qh[kSteps], ql[kWide ? kSteps : 1];
    const float score_scale = a.scale2 == 0.0f ? 1.0f : fabsf(a.scale2);  // (int8: part of the keys' steps)
    float xscale = CT == PT_I8 ? 1.0f : score_scale;                      // the factor of the scores, positive

    v16f o[kOut];
#pragma unroll
    for (int t = 0; t < kOut; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            o[t][i] = 0.0f;
        }
    }
    if (CT != PT_I8) {  // (visible to all behind the first tile's barrier)
        for (uint32_t at = tid; at < 4 * DIM + 5; at += 256) {
            sPoison[at] = 0;
        }
    }
    bool poisoned = false;  // int8: this row sees a slot whose step is not finite
    float m = kLow, l = 0.0f, unit = CT == PT_I8 ? kFirstUnit : 1.0f;

    // Page of key k0 + lane, none: -1. In two halves: the list is read a tile ahead of its use.
    auto look_up = [&](uint32_t k0) -> int32_t { return table[min(k0 + lane, all.hi - 1) >> a.pool.shift]; };
    auto page_of = [&](uint32_t k0, int32_t found) -> int32_t { return k0 + lane < all.hi && (uint32_t)found < a.pool.pages ? found : -1; };
    // A wave's load n covers kRowsAt rows of the tile, from row (4n + wave) kRowsAt on. In pages of so many keys and more (PAGED) they
    // lie side by side, so that their address is the wave's and what a lane adds to it is the same for every load (8192 tokens bf16
    // 536 us; with an address per lane, as smaller pages need it, 568). A key without
    // a page is read from page 0: what it brings is masked, and taken out of the tile where it is not finite.
    constexpr uint32_t kRowsAt = rows_at<CT, DIM>(), kChunks = kRowBytes / 16;
    const uint32_t in_row = lane / kChunks, chunk = lane % kChunks;
    // byte offset of key k0 + lane in the pool
    auto offset_of = [&](uint32_t k0, int32_t page) -> size_t {
        const size_t first = (size_t)(uint32_t)max(page, 0) * a.pool.kv_heads + kvh;
        return ((first << a.pool.shift) | ((k0 + lane) & ((1u << a.pool.shift) - 1))) * kRowBytes;
    };
    // of load n: the wave's part in *base, the lane's as the answer
    auto row_at = [&](size_t offset, int n, size_t *base) -> uint32_t {
        if (PAGED) {
            const uint32_t from = n * 4 * kRowsAt + wave * kRowsAt;
            *base = (size_t)__builtin_amdgcn_readlane((uint32_t)(offset >> 32), from) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)offset, from);
            return in_row * kRowBytes;
        }
        const uint32_t from = n * 4 * kRowsAt + wave * kRowsAt + in_row;
        *base = (size_t)(uint32_t)__shfl((uint32_t)(offset >> 32), from, 64) << 32 | (uint32_t)__shfl((uint32_t)offset, from, 64);
        return 0;
    };
    // 16-bit caches: straight into LDS, the rows' pieces permuted
    const uint32_t first_row = wave * kRowsAt + in_row;  // of load 0; the others' rows are 4 kRowsAt apart, which changes no permutation
    auto fetch = [&](uint32_t k0, int32_t pages, lds_t to) {
        const size_t offset = offset_of(k0, pages);
        const uint32_t pk = 16 * (chunk ^ swizzle_k<DIM>(first_row)), pv = 16 * (chunk ^ swizzle_v<DIM>(first_row));
        lds_t const mine_to = to + wave * 1024;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            size_t base;
            const uint32_t add = row_at(offset, n, &base);
            const uint8_t *const kp = (const uint8_t *)a.pool.k + base, *const vp = (const uint8_t *)a.pool.v + base;
            __builtin_amdgcn_global_load_lds((gptr_t)(kp + (add + pk)), (lptr_t)(mine_to + n * 4096), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((gptr_t)(vp + (add + pv)), (lptr_t)(mine_to + kTileBytes + n * 4096), 16, 0, 0);
        }
    };
    // int8: into registers as it is stored, from where it goes to LDS as fp16 while the tile before is worked on (by way of LDS, and
    // converted there between two barriers, 2 x 256 new tokens over 27 k keys took 176 us against 167; between the products, but
    // with a barrier for keys and one for values, 182)
    v4u raw[CT == PT_I8 ? kLoads : 1][2];
    float scale = 0.0f;  // of key lane (wave 0: key, the others: value)
    auto fetch_raw = [&](uint32_t k0, int32_t pages) {
        const size_t offset = offset_of(k0, pages);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            size_t base;
            const uint32_t add = row_at(offset, n, &base) + 16 * chunk;
            raw[n][0] = *(const v4u *)((const uint8_t *)a.pool.k + base + add);
            raw[n][1] = *(const v4u *)((const uint8_t *)a.pool.v + base + add);
        }
        scale = (wave ? a.pool.vs : a.pool.ks)[offset / kRowBytes];
        scale = pages < 0 ? INFINITY : scale;
    };
    // eight elements in each lane: piece p of 4 kLoads
    uint32_t at_put_k = (first_row * kPieces + (2 * chunk ^ swizzle_k<DIM>(first_row))) * 16;
    uint32_t at_put_v = (first_row * kPieces + (2 * chunk ^ swizzle_v<DIM>(first_row))) * 16;
    auto convert = [&](int p, lds_t to) {
        const int n = p / 4, kv = p / 2 % 2, half = p % 2;
        const v4u w = raw[n][kv];
        v4u f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = biased_to_f16(__builtin_amdgcn_perm(0x64646464u, w[2 * half + i / 2] ^ 0x80808080u, i & 1 ? 0x04030402 : 0x04010400));
        }
        *(__attribute__((address_space(3))) v4u *)(to + kv * kTileBytes + n * 4 * kRowsAt * DIM * 2 + ((kv ? at_put_v : at_put_k) ^ (16 * half))) = f;
    };
    // The steps. One of a value that is not finite is taken out.
    auto put_steps = [&](StepsOfTile *to) {
        if (wave < 2) {
            float step = __builtin_amdgcn_rcpf(scale);
            if (wave == 1) {
                const bool fine = step - step == 0.0f;  // neither infinite nor NaN
                const unsigned long long not_fine = __ballot(!fine);
                step = fine ? step : 0.0f;
                const float unit_of_tile = power_above(wave_max_abs(step));
                if (lane == 0) {
                    to->bad = not_fine;
                    to->unit = unit_of_tile;
                }
                to->step[kStepOwn][lane] = step;
                to->step[kStepOwnLow][lane] = step * kLowStep;
                step *= __builtin_amdgcn_rcpf(unit_of_tile);
            } else {
                step *= score_scale;
            }
            to->step[wave ? kStepV : kStepK][lane] = step;
        }
    };

    // where this lane reads in a tile: K pieces of row c, and for V (16 lanes read four keys of 16 d, lane e of them the d
    // 4 (e % 4) .. + 3 of key e / 4, and get d e of all four); of the first step, the others' differ in two or three bits
    static_assert(CT != PT_I8 || 4 * kLoads == kSteps, "a piece is converted at every step of the scores");
    uint32_t at_k = (c * kPieces + (h ^ swizzle_k<DIM>(c))) * 16, at_v[2];
    {
        const uint32_t e = lane & 15, sub = (lane >> 4) & 1, from = 2 * sub + e % 4 / 2;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t rowk = 4 * h + e / 4 + 8 * w;
            at_v[w] = (rowk * kPieces + (from ^ swizzle_v<DIM>(rowk))) * 16 + 8 * (e % 2);
        }
    }

    int32_t pages = -1, next = -1;
    unsigned long long stored = 0;  // (bit i) key i of the tile has a page
    if (t0 < t1) {
        const uint32_t k0 = all.lo + t0 * kKeys;
        pages = page_of(k0, look_up(k0));
        next = look_up(k0 + kKeys);
        if (CT == PT_I8) {
            fetch_raw(k0, pages);
            stored = __ballot(pages >= 0);
            pages = page_of(k0 + kKeys, next);
            next = look_up(k0 + 2 * kKeys);
#pragma unroll
            for (int p = 0; p < 4 * kLoads; ++p) {
                convert(p, sTiles);
            }
            put_steps(sSteps);
            fetch_raw(k0 + kKeys, pages);
        } else {
            fetch(k0, pages, sTiles);
        }
    }
    // queries (while the first tile is on its way)
    {
        const float sign = a.scale2 == 0.0f ? 0.0f : a.scale2 < 0.0f ? -1.0f : 1.0f;
        const size_t at = (size_t)(mine ? row : 0) * a.qstride + (size_t)(mine ? head : 0) * DIM + 8 * h;
        float top = 0.0f, up = 1.0f;
        if (kShiftQ) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                float v[8];
                load8<ACT>(a.q, at + 16 * s, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    top = fmaxf(top, fabsf(v[j]));
                }
            }
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            int e = 0;
            up = shift_into_f16(top, &e);
            xscale = ldexpf(xscale, e);
            xscale = xscale < 1.17549435e-38f ? 1.17549435e-38f : xscale;  // not zero: it meets scores of -inf
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            float v[8];
            load8<ACT>(a.q, at + 16 * s, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] *= sign;
            }
            V lo;
            Operand<CT>::split(v, up, &qh[s], &lo);
            if (kWide) {
                ql[s] = lo;
            }
        }
    }

    // One tile: `now` holds it, `ahead` is where the next one goes. (16-bit caches: the compiler has to know that the two are apart,
    // else it waits for the next tile's arrival before it reads this one.)
    auto step_over = [&](uint32_t t, __attribute__((address_space(3))) uint8_t *__restrict now,
                         __attribute__((address_space(3))) uint8_t *__restrict ahead, const StepsOfTile *steps, StepsOfTile *steps_ahead) {
        const uint32_t k0 = all.lo + t * kKeys;
        if (CT == PT_I8) {
            barrier();  // the tile is there; and everyone is done with the tile before
        } else {
            stored = __ballot(pages >= 0);
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the tile is there
            __syncthreads();                     // everyone's; and everyone is done with the tile before
            pages = page_of(k0 + kKeys, next);
            next = look_up(k0 + 2 * kKeys);
            if (t + 1 < t1) {
                fetch(k0 + kKeys, pages, ahead);
            }
        }
        // does every row of the workgroup see every key of the tile?
        const bool whole = stored == ~0ull && k0 + kKeys <= all_hi && k0 >= all_lo;
        // A value that is infinite or NaN must not reach the rows that do not see its key (0 * inf): it is taken out of the tile, and
        // the rows that do see it become NaN in the end. An int8 cache has it in the slot's step, which put_steps has taken out.
        if (CT != PT_I8 && !whole) {
            constexpr uint32_t kExp = CT == PT_BF16 ? 0x7f80u : 0x7c00u;
            lds_t const base = now + kTileBytes;
            v4u w[kTileBytes / 16 / 256];
#pragma unroll
            for (uint32_t n = 0; n < kTileBytes / 16 / 256; ++n) {
                w[n] = *(const __attribute__((address_space(3))) v4u *)(base + (n * 256 + tid) * 16);
            }
            bool hit = false;
#pragma unroll
            for (uint32_t n = 0; n < kTileBytes / 16 / 256; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    hit |= (w[n][i] & kExp) == kExp || (w[n][i] >> 16 & kExp) == kExp;
                }
            }
            hit = __any(hit);
            if (lane == 0) {
                sHit[wave] = hit;
            }
            __syncthreads();
            if (sHit[0] | sHit[1] | sHit[2] | sHit[3]) {
                for (uint32_t at = tid; at < kKeys * DIM; at += 256) {
                    const uint32_t rowk = at / DIM, d = at % DIM;
                    auto *const p = (__attribute__((address_space(3))) uint16_t *)(base + (rowk * kPieces + (d / 8 ^ swizzle_v<DIM>(rowk))) * 16) + d % 8;
                    if ((*p & kExp) == kExp) {
                        *p = 0;
                        if (stored >> rowk & 1) {
                            // rows from the key's own position on, as far as the window reaches
                            const int64_t key = k0 + rowk, r0 = (int64_t)tile_index * kRows;
                            const int64_t from = (key - seq.pos) * group - r0, upto = a.window ? (key + a.window - seq.pos) * group - r0 : kRows;
                            for (uint32_t w = 0; w < 4; ++w) {
                                const int64_t x = from - 32 * w, y = upto - 32 * w;
                                const uint32_t bits = (y >= 32 ? ~0u : y <= 0 ? 0u : (1u << y) - 1) & (x <= 0 ? ~0u : x >= 32 ? 0u : ~0u << x);
                                if (bits) {
                                    atomicOr(&sPoison[4 * d + w], bits);
                                    *sAny = 1;
                                }
                            }
                        }
                    }
                }
                __syncthreads();
            }
        }
        // int8: the next tile's steps into LDS, the one's behind it on their way
        auto further = [&] {
            put_steps(steps_ahead);
            stored = __ballot(pages >= 0);
            pages = page_of(k0 + 2 * kKeys, next);
            next = look_up(k0 + 3 * kKeys);
            fetch_raw(k0 + 2 * kKeys, pages);
        };
        // a wave without rows only brings its part of the tiles (32 sequences of up to 4 new tokens over up to 2000 keys 53 us, with
        // all four at work on nothing 59)
        if (idle) {
            if (CT == PT_I8) {
#pragma unroll
                for (int p = 0; p < 4 * kLoads; ++p) {
                    convert(p, ahead);
                }
                further();
            }
            return;
        }
        // Scores. The order is written out (the compiler would wait for every read right behind it): six or eight reads ahead of the
        // products that use them.
        v16f s[2];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            s[0][j] = s[1][j] = 0.0f;
        }
        constexpr int kRing = CT == PT_I8 || kWide ? 3 : 4;  // pairs of reads under way
        V kf[kRing][2];
        uint32_t from = at_k;
        if (CT == PT_I8) {
            asm volatile("" : "+v"(from));  // addresses are made anew: kept from tile to tile they would cost registers that the tile needs
        }
        auto keys = [&](int st) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                kf[st % kRing][i] = *(const __attribute__((address_space(3))) V *)(now + i * 32 * DIM * 2 + (from ^ 32 * st));
            }
        };
#pragma unroll
        for (int st = 0; st < kRing; ++st) {
            keys(st);
        }
        in_order();
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[i] = Op::mfma(kf[st % kRing][i], qh[st], s[i]);
                if (kWide) {
                    s[i] = Op::mfma(kf[st % kRing][i], ql[st], s[i]);
                }
            }
            in_order();
            if (st + kRing < kSteps) {
                keys(st + kRing);
                in_order();
            }
            if (CT == PT_I8) {
                convert(st, ahead);
                in_order();
            }
        }
        const unsigned long long stored_here = stored;
        if (CT == PT_I8) {
            further();
        }
        V vv[2][kOut], ph[2], pl[2];
        Words<4> pw[2];
        auto value = [&](int u, int i) {
            lds_t const base = now + kTileBytes + u * 16 * DIM * 2;
            struct {
                v4s a, b;
            } w;
            w.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)(base + (at_v[0] ^ 64 * i)));
            w.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)(base + (at_v[1] ^ 64 * i)));
            vv[u & 1][i] = __builtin_bit_cast(V, w);
        };
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            value(0, i);
        }
        in_order();
        if (CT == PT_I8) {
            v4f ks[3];
            auto read = [&](int x) { ks[x % 3] = *(const v4f *)(steps->step[kStepK] + 32 * (x / 4) + 8 * (x % 4) + 4 * h); };
            read(0);
            read(1);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                if (x + 2 < 8) {
                    read(x + 2);
                }
                in_order();
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[x / 4][4 * (x % 4) + e] *= ks[x % 3][e];
                }
                in_order();
            }
        }
        unsigned long long seen = ~0ull;
        float tile_unit = CT == PT_I8 ? steps->unit : 1.0f;  // no step of a value that the row sees exceeds it
        if (!whole) {
            const uint32_t from = span.lo > k0 ? span.lo - k0 : 0, upto = span.hi > k0 ? span.hi - k0 : 0;  // keys of the tile this row sees
            seen = from >= kKeys || upto <= from ? 0 : (upto >= kKeys ? ~0ull : (1ull << upto) - 1) & (~0ull << from);
            seen &= stored_here;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t half = (uint32_t)(seen >> (32 * i)) >> (4 * h);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const bool sees = half >> (8 * (j / 4) + j % 4) & 1;
                    s[i][j] = sees ? s[i][j] : -INFINITY;
                }
            }
            if (CT == PT_I8) {
                float wide = 0.0f;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const uint32_t some = (uint32_t)(seen >> (32 * (x / 4))) >> (8 * (x % 4) + 4 * h);
                    const v4f step = *(const v4f *)(steps->step[kStepOwn] + 32 * (x / 4) + 8 * (x % 4) + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        wide = fmaxf(wide, some >> e & 1 ? fabsf(step[e]) : 0.0f);
                    }
                }
                tile_unit = power_above(fmaxf(wide, __shfl_xor(wide, 32, 64)));
            }
        }
        if (CT == PT_I8) {
            poisoned |= (steps->bad & seen) != 0;
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            top = max_of(top, s[0][j], s[1][j]);
        }
        top *= xscale;
        if (__any(top - m > kSlack<CT> || (CT == PT_I8 && tile_unit > unit))) {
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float up = top - m > kSlack<CT> ? top : m;
            float corr = __builtin_amdgcn_exp2f(m - up);
            l *= corr;
            m = up;
            if (CT == PT_I8) {
                const float was = unit;
                unit = fmaxf(tile_unit, unit);
                float now_unit = unit;
                asm volatile("" : "+v"(now_unit));  // (else the reciprocal below is shared with this one, and the way round this block copies the outputs)
                corr *= was * __builtin_amdgcn_rcpf(now_unit);
            }
#pragma unroll
            for (int i = 0; i < kOut; ++i) {
                o[i] = o[i] * corr;
            }
        }
        // A weight's exponent is s * factor + shift in one instruction. Its product is not rounded as that in the maximum m was, and in
        // the shift m meets small numbers: above 2^23 either is off by a whole and more, weights leave fp16 and differ from tile to
        // tile. Of scores that large (a row's own: others keep their bytes) the maximum is taken away first (of
        // -inf, where a row sees nothing of the tile, too).
        float factor = xscale, off = m;
        if (fabsf(top) > kLargeScore) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    s[i][j] = s[i][j] * xscale - m;
                }
            }
            factor = 1.0f;
            off = 0.0f;
        }
        // Weights times values, 16 keys a step: behind every product stand the next step's reads and a share of its weights
        // (int8: the steps that weights are multiplied by are over `unit` in the end. What is left of that beside the way they are stored
        // goes into the exponent, and out of the sum again: the tile's power of two over `unit`, down to 2^-64, where a tile's values
        // are far below what the output can hold of others; or, of steps as they are, 1 / unit, which fp32 holds a weight times
        // where unit < 1, and of those times 2^-80 2^80 / unit. What a row does not see has a weight of zero.)
        const float *steps_v = nullptr;
        float part = 1.0f;
        if (CT == PT_I8) {
            part = __builtin_amdgcn_rcpf(unit);
            const bool low = unit >= 1.0f;
            const float own = low ? part * (1.0f / kLowStep) : part;
            part = whole ? fmaxf(tile_unit * part, 5.42101086e-20f) : own;
            steps_v = steps->step[kStepV] + (whole ? 0 : (low ? kStepOwnLow - kStepV : kStepOwn - kStepV) * kKeys);
        }
        const float shift = (CT == PT_I8 ? kLift<CT> + __builtin_amdgcn_logf(part) : kLift<CT>) - off;
        float sum = 0.0f;
        float p[8];
        v4f vs[2][2];  // int8: steps of this group's and the next one's values
        auto steps_of = [&](int u) {
            vs[u & 1][0] = *(const v4f *)(steps_v + 16 * u + 4 * h);
            vs[u & 1][1] = *(const v4f *)(steps_v + 16 * u + 8 + 4 * h);
        };
        if (CT == PT_I8) {
            steps_of(0);
            steps_of(1);
        }
        // Weights of 16-bit activations are rounded once, which leaves an error of the order of the output's own rounding. Two parts, as
        // fp32 activations have, would double these products: 8192 tokens bf16 717 us against 540, ragged prompts fp16 120 and 97,
        // 2 x 256 tokens over 27 k int8 keys 195 and 158. Over a 16-bit cache the sum takes the rounded ones, so that they add up to one.
        auto weight = [&](int u, int j) {  // j and j + 1
#pragma unroll
            for (int e = j; e < j + 2; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u % 2) + e], factor, shift));
                if (CT == PT_I8) {
                    sum += p[e];
                    p[e] *= vs[u & 1][e / 4][e % 4];
                } else if (kWide) {
                    l += p[e];
                }
            }
            if (!kWide) {
                const uint32_t w = Op::pack(p[j], p[j + 1]);
                pw[u & 1].w[j / 2] = w;
                if (CT != PT_I8) {
                    l = Op::add_pair(w, l);
                }
            }
        };
        auto ready = [&](int u) {
            if (kWide) {
                Operand<CT>::split(p, 1.0f, &ph[u & 1], &pl[u & 1]);
            } else {
                ph[u & 1] = __builtin_bit_cast(V, pw[u & 1]);
            }
        };
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            weight(0, j);
        }
        ready(0);
        in_order();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int i = 0; i < kOut; ++i) {
                o[i] = Op::mfma(vv[u & 1][i], ph[u & 1], o[i]);
                if (kWide) {
                    o[i] = Op::mfma(vv[u & 1][i], pl[u & 1], o[i]);
                }
                in_order();
                if (u < 3) {
                    value(u + 1, i);
#pragma unroll
                    for (int j = i * (8 / kOut); j < (i + 1) * (8 / kOut); j += 2) {
                        weight(u + 1, j);
                    }
                    if (i == kOut - 1) {
                        ready(u + 1);
                        if (CT == PT_I8 && u < 2) {
                            steps_of(u + 2);
                        }
                    }
                    in_order();
                }
            }
        }
        if (CT == PT_I8) {
            l += sum * __builtin_amdgcn_rcpf(part);
        }
    };
    if (CT == PT_I8) {
        // (One body, the buffers told apart by a bit of the addresses. Two, as below, take more registers than there are: 177 us
        // against 157 for 2 x 256 new tokens over 27 k keys.)
        auto other = [&] {
            at_put_k ^= 2 * kTileBytes;
            at_put_v ^= 2 * kTileBytes;
        };
        other();
        for (uint32_t t = t0, at = 0; t < t1; ++t, at ^= 1) {
            step_over(t, sTiles, sTiles, sSteps + at, sSteps + (at ^ 1));
            other();
            at_k ^= 2 * kTileBytes;
            at_v[0] ^= 2 * kTileBytes;
            at_v[1] ^= 2 * kTileBytes;
        }
    } else {
        for (uint32_t t = t0; t < t1; t += 2) {
            step_over(t, sTiles, sTiles + 2 * kTileBytes, nullptr, nullptr);
            if (t + 1 < t1) {
                step_over(t + 1, sTiles + 2 * kTileBytes, sTiles, nullptr, nullptr);
            }
        }
    }

    l += __shfl_xor(l, 32, 64);
    if (CT == PT_I8) {
        l = poisoned ? NAN : l;
    } else {
        __syncthreads();
        if (*sAny) {
#pragma unroll
            for (int i = 0; i < kOut; ++i) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    o[i][j] = sPoison[4 * (32 * i + 8 * (j / 4) + 4 * h + j % 4) + wave] >> c & 1 ? NAN : o[i][j];
                }
            }
        }
    }
    // A sum of zero: the row has seen no key here, which a maximum of -inf says of it, or only scores of -inf
    if (l == 0.0f) {
        const uint32_t upto = min(span.hi, all.lo + t1 * kKeys), mask = (1u << a.pool.shift) - 1;
        bool any = false;
        for (uint32_t key = max(span.lo, all.lo + t0 * kKeys); key < upto && !any; key = (key | mask) + 1) {
            any = (uint32_t)table[key >> a.pool.shift] < a.pool.pages;
        }
        m = any ? m : -INFINITY;
    }
    if (alone) {
        if (!mine) {
            return;
        }
        uint32_t again = r;
        asm volatile("" : "+v"(again));  // the row's place is worked out anew: kept over the loop it would cost registers
        const uint32_t token_again = paged_div(again, a.group);
        const float inv = m == -INFINITY ? 0.0f : l == 0.0f ? NAN : unit / l;
        const size_t at = (size_t)(seq.first + token_again) * a.ostride + (size_t)(kvh * group + (again - token_again * group)) * DIM + 4 * h;
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                store_out4<ACT>(a.out, at + 32 * i + 2 * j, o[i][j] * inv, o[i][j + 1] * inv, o[i][j + 2] * inv, o[i][j + 3] * inv);
            }
        }
        return;
    }
    if (idle) {
        return;
    }
    float *const part = part_at(a, x, kvh, share, shares.d, DIM);
    constexpr float down = kPartScale<CT>;
    const uint32_t pr = 32 * wave + c;
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            *(v4f *)(part + (size_t)pr * DIM + 32 * i + 2 * j + 4 * h) =
                (v4f){o[i][j] * down * unit, o[i][j + 1] * down * unit, o[i][j + 2] * down * unit, o[i][j + 3] * down * unit};
        }
    }
    if (h == 0) {
        part[kRows * DIM + pr] = m;
        part[kRows * DIM + kRows + pr] = l * down;
    }
}

// Joins the shares of a tile's keys: a workgroup per eight rows of a tile, DIM / 4 lanes to a row
template <int ACT, int DIM>
__global__ __launch_bounds__(8 * DIM / 4) void paged_prompt_join_kernel(PagedAttentionArgs a, PagedDivisor shares)
{
    const uint32_t lane = threadIdx.x & 63, x = paged_div(blockIdx.x, a.kv_heads), kvh = blockIdx.x - x * a.kv_heads.d;
    const uint32_t group = a.group.d;
    uint32_t b, tile_index;
    PagedSeq seq;
    if (!find_tile(a, x, lane, &b, &tile_index, &seq)) {
        return;
    }
    const uint32_t rows = rows_of(a, seq);
    const Reach all = reach_of(a, seq, rows, tile_index);
    const uint32_t per = tiles_per_share(all.tiles, shares);
    if (per >= all.tiles) {
        return;
    }
    const uint32_t count = (all.tiles + per - 1) / per;
    const uint32_t pr = blockIdx.y * 8 + threadIdx.x / (DIM / 4), d = threadIdx.x % (DIM / 4) * 4;
    const uint32_t r = tile_index * kRows + pr;
    const uint32_t token = paged_div(r, a.group);
    const int64_t row = seq.first + token;
    if (r >= rows || row < 0 || row >= (int64_t)a.batch.rows) {
        return;
    }
    float top = -INFINITY, sum = 0.0f;
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i = 0; i < count; ++i) {
        const float *const p = part_at(a, x, kvh, i, shares.d, DIM);
        const float m = p[kRows * DIM + pr], up = fmaxf(top, m);
        const float from = fmaxf(up, kLow), f = __builtin_amdgcn_exp2f(top - from), e = __builtin_amdgcn_exp2f(m - from);
        sum = sum * f + p[kRows * DIM + kRows + pr] * e;
        v = v * f + *(const v4f *)(p + (size_t)pr * DIM + d) * e;
        top = up;
    }
    const float inv = top == -INFINITY ? 0.0f : sum == 0.0f ? NAN : 1.0f / sum;
    store_out4<ACT>(a.out, (size_t)row * a.ostride + (size_t)(kvh * group + r - token * group) * DIM + d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
}

// row tiles that a launch may have, and how many workgroups share a tile's keys
uint64_t most_tiles(const PagedBatch &b, uint32_t group)
{
    return (uint64_t)b.rows * group / kRows + b.batch;
}

uint32_t shares_of(const PagedPool &pool, const PagedBatch &b, uint32_t heads)
{
    const uint64_t grid = most_tiles(b, heads / pool.kv_heads) * pool.kv_heads;
    const uint64_t keys = (((uint64_t)b.max_pages << pool.shift) + kKeys * kLeast - 1) / (kKeys * kLeast);
    const uint64_t n = grid >= kSpread ? 1 : (kSpread + grid / 2) / grid;
    return (uint32_t)(n < keys ? n : keys);
}

// Before a kernel's first launch on a device (one bit each in `done`; a second time does no harm): it may ask for its LDS, and has
// none besides, for the tiles are taken to start at LDS address 0
hipError_t prepare(const void *kernel, uint32_t lds, std::atomic<uint64_t> &done)
{
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if (e != hipSuccess || (device < 64 && done.load(std::memory_order_relaxed) & bit)) {
        return e;
    }
    hipFuncAttributes have;
    e = hipFuncGetAttributes(&have, kernel);
    if (e == hipSuccess && have.sharedSizeBytes != 0) {
        e = hipErrorInvalidImage;
    }
    e = e != hipSuccess ? e : hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e == hipSuccess) {
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    return e;
}

template <int ACT, int CT, int DIM>
struct Prompt {
    static hipError_t run(const PagedAttentionArgs &a, hipStream_t st)
    {
        const uint32_t shares = shares_of(a.pool, a.batch, a.heads);
        const uint64_t tiles = most_tiles(a.batch, a.heads / a.pool.kv_heads);
        constexpr uint32_t lds = prompt_lds<CT, DIM>();
        const bool paged = 1u << a.pool.shift >= rows_at<CT, DIM>();
        const auto kernel = paged ? paged_prompt_kernel<ACT, CT, DIM, true> : paged_prompt_kernel<ACT, CT, DIM, false>;
        static std::atomic<uint64_t> ready[2];
        hipError_t e = prepare((const void *)kernel, lds, ready[paged]);
        if (e != hipSuccess) {
            return e;
        }
        const uint64_t blocks = tiles * a.pool.kv_heads;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)(blocks * shares)), dim3(256), lds, st, a, paged_divisor(shares));
        e = hipGetLastError();
        if (e != hipSuccess || shares == 1) {
            return e;
        }
        hipLaunchKernelGGL((paged_prompt_join_kernel<ACT, DIM>), dim3((uint32_t)blocks, kRows / 8), dim3(8 * DIM / 4), 0, st, a, paged_divisor(shares));
        return hipGetLastError();
    }
};

}  // namespace

bool paged_prompt_fits(const PagedPool &pool, const PagedBatch &batch, uint32_t heads)
{
    const uint32_t group = heads / pool.kv_heads;
    return (uint64_t)batch.rows * group <= 0x7fffffffull && most_tiles(batch, group) * pool.kv_heads < 1u << 24;
}

size_t paged_prompt_workspace(const PagedPool &pool, const PagedBatch &batch, uint32_t heads)
{
    const uint32_t shares = shares_of(pool, batch, heads);
    const uint64_t parts = shares == 1 ? 0 : most_tiles(batch, heads / pool.kv_heads) * pool.kv_heads * shares;
    return parts * kRows * (pool.dim + 2) * sizeof(float) + 256;
}

hipError_t launch_paged_prompt(const PagedAttentionArgs &a, hipStream_t st)
{
    return a.batch.rows && a.batch.batch ? paged_dispatch<Prompt>(a.act, a.pool.type, a.pool.dim, a, st) : hipSuccess;
}

}  // namespace bg
