// The blocks of packed keys that a query attends to, chosen by a bound on its scores.
//
// A group of packed keys lies in channel c between zero_c and zero_c + L scale_c (L the top code), so no key of it has a product
// with a query above  sum_c max(q_c zero_c, q_c (zero_c + L scale_c)).  A block's score is the largest such bound over its groups, over
// the query heads of the kv head and over the queries of a tile, which choose together; the bounds are what the store keeps anyway.
//
// Which blocks are chosen must not hang on the order of a sum, so scores are formed in 64 bits: the sum of a head's channels is good to
// 1e-15 of its terms.  Equal scores: the lower block first.
//
// The chosen ones come out in ascending order, -1 behind them where fewer are visible: the first `first` and the last `recent` visible
// blocks always, the others by score.
#include "attend_span_mfma.hpp"

namespace vq {

namespace {

struct SelectCall {
    vq_block_select_args a;
    int64_t tiles, total;   // tiles of queries a sequence, blocks of the store
    int64_t items;          // B Hkv tiles
    uint64_t *exact;        // [items][total], room for the keys of scores of 64 bits (block_pick_kernel)
    uint64_t *stored;       // [items][groups], those of every group where the filter does not take the call
    // the filter on the matrix units:
    int mma;                // 1: it takes the call
    int one;                // 1: in one launch, a block an item
    int64_t query_block;    // (at most Sq)
    int row_tiles;          // of 32 rows an item
    int64_t groups, stride; // of the packed slots, of the store
    int runs, run_units;    // waves a row tile, units of 32 groups of each
    float *approx;          // [items][row_tiles][groups]
    float *bounds;          // [items][row_tiles][runs]
    // float32 scales and zeros, which it takes rounded to fp16: a's are the copies
    int narrow;
    u16 *copies;            // [zeros, scales][B][Hkv][groups][D]
    const float *wide_zero, *wide_scale;
    int64_t wide_stride;
};

// Live slots of a sequence, and of the packed ones those [0, end) that its query i sees (slots and queries: below 2^30).
__device__ __forceinline__ int sel_live(const vq_block_select_args &a, int b) {
    const int room = (int)a.n_packed + (int)a.n_tail;
    if (a.seq_lens == nullptr) return room;
    const int64_t n = a.seq_lens[b];
    return n < 0 ? 0 : n < room ? (int)n : room;
}
__device__ __forceinline__ int sel_end(const vq_block_select_args &a, int live, int i) {
    const int packed = (int)a.n_packed;
    int end = a.causal ? live - (int)a.Sq + i + 1 : live;
    end = end < live ? end : live;
    return end < 0 ? 0 : end < packed ? end : packed;
}
__device__ __forceinline__ int sel_last(const vq_block_select_args &a, int tile) {
    const int64_t last = (tile + INT64_C(1)) * a.query_block;
    return (int)(last < a.Sq ? last : a.Sq) - 1;
}

// Scores of 64 bits as whole numbers in their order.
__device__ __forceinline__ uint64_t pick_key(double s) {   // ascending with the score, NaN above all
    if (s != s) return ~UINT64_C(0);
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.);
    return u >> 63 ? ~u : u | (UINT64_C(1) << 63);
}
__device__ __forceinline__ uint64_t max_key(uint64_t x, uint64_t y) { return x > y ? x : y; }
__device__ __forceinline__ double key_score(uint64_t k) { return __longlong_as_double((int64_t)(k >> 63 ? k & ~(UINT64_C(1) << 63) : ~k)); }   // (NaN for NaN's)

// Over a wave by moves within rows of sixteen lanes and from row to row, not through the LDS unit: the largest (of op's) in every lane; the sum up to and with a lane.
template <int CTRL, int ROWS> __device__ __forceinline__ u32 moved(u32 old, u32 x) { return (u32)__builtin_amdgcn_update_dpp((int)old, (int)x, CTRL, ROWS, 0xF, false); }
template <typename Op> __device__ __forceinline__ u32 wave_all(u32 x, Op op) {
    x = op(x, moved<0x111, 0xF>(x, x));   // row_shr 1, 2, 4, 8: a lane without a source meets itself
    x = op(x, moved<0x112, 0xF>(x, x));
    x = op(x, moved<0x114, 0xF>(x, x));
    x = op(x, moved<0x118, 0xF>(x, x));
    x = op(x, moved<0x142, 0xA>(x, x));   // row_bcast 15, 31
    x = op(x, moved<0x143, 0xC>(x, x));
    return (u32)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ u32 wave_max_bits(u32 x) { return wave_all(x, [](u32 y, u32 z) { return y > z ? y : z; }); }
__device__ __forceinline__ float wave_max(float x) {
    return __uint_as_float(wave_all(__float_as_uint(x), [](u32 y, u32 z) { return __float_as_uint(fmaxf(__uint_as_float(y), __uint_as_float(z))); }));
}
__device__ __forceinline__ float wave_min(float x) {
    return __uint_as_float(wave_all(__float_as_uint(x), [](u32 y, u32 z) { return __float_as_uint(fminf(__uint_as_float(y), __uint_as_float(z))); }));
}
__device__ __forceinline__ u32 wave_sum_up(u32 x) {
    x += moved<0x111, 0xF>(0, x);
    x += moved<0x112, 0xF>(0, x);
    x += moved<0x114, 0xF>(0, x);
    x += moved<0x118, 0xF>(0, x);
    x += moved<0x142, 0xA>(0, x);
    x += moved<0x143, 0xC>(0, x);
    return x;
}

// The sum over `parts` neighbouring lanes (a power of two), in each of them: within sixteen by moves (as above), then through the LDS unit.
template <int CTRL> __device__ __forceinline__ double add_moved(double s) {
    const uint64_t x = (uint64_t)__double_as_longlong(s);
    const u32 low = moved<CTRL, 0xF>(0, (u32)x), high = moved<CTRL, 0xF>(0, (u32)(x >> 32));
    return s + __longlong_as_double((int64_t)((uint64_t)high << 32 | low));
}
__device__ __forceinline__ double sum_parts(double s, int parts) {
    if (parts > 1) s = add_moved<0xB1>(s);    // quad_perm [1,0,3,2]
    if (parts > 2) s = add_moved<0x4E>(s);    // quad_perm [2,3,0,1]
    if (parts > 4) s = add_moved<0x141>(s);   // row_half_mirror
    if (parts > 8) s = add_moved<0x140>(s);   // row_mirror
    if (parts > 16) s += __shfl_xor(s, 16);
    if (parts > 32) s += __shfl_xor(s, 32);
    return s;
}

// Float32 queries, head sizes that the matrix units do not take, few products over float32 scales and zeros: every group's score in 64 bits, on the vector units.
//
// Eight lanes a group, each with four channels of every 32, all of them asked for ahead of the queries, of which RW rows at a time lie in LDS as
// doubles.  With a group's middle and half width in a channel, m = z + L s / 2 and w = L |s| / 2, the bound is sum y m + |y| w: two
// multiply-adds a channel and row, where the larger of two products takes six instructions (a ninth less time).  What is not finite leaves no finite sum, and is done
// again by the products.  WIDE: four channels a load.
constexpr int SCORE_GROUPS = 32;   // a block of threads
template <typename T, bool WIDE, int RW> __global__ __launch_bounds__(256) void group_score_kernel(SelectCall c) {
    constexpr int STEPS = 4;   // of 32 channels, at once
    extern __shared__ double qs[];   // [RW][D, up to whole 32s]
    const vq_block_select_args &a = c.a;
    const int tid = threadIdx.x, part = tid & 7;
    // (tiles outermost, so that those of a head, which read the same groups, share a cache: 5 sequences of 4 kv heads, three queries a tile
    // of their own, 12 MB of float32: a tenth less than head by head)
    const u32 many = (u32)((c.groups + SCORE_GROUPS - 1) / SCORE_GROUPS), heads = (u32)a.B * (u32)a.Hkv, id = blockIdx.x / many, bh = id % heads;
    const int u0 = (int)(blockIdx.x % many) * SCORE_GROUPS, tile = (int)(id / heads), hkv = (int)(bh % (u32)a.Hkv), b = (int)(bh / (u32)a.Hkv);
    const int64_t item = (int64_t)bh * c.tiles + tile;
    const int live = sel_live(a, b), G = (int)a.Hq / (int)a.Hkv, D = (int)a.D, room = (D + 31) / 32 * 32, g = a.group, pos0 = tile * (int)c.query_block,
              last = sel_last(a, tile), groups = (sel_end(a, live, last) + g - 1) / g;   // that some row sees
    if (u0 >= groups) return;
    const int rows = (last - pos0 + 1) * G, u = u0 + (tid >> 3);
    const int64_t at = ((int64_t)bh * c.stride + (u < groups ? u : groups - 1)) * D;   // (past the last group: it again)
    const T *const zero = (const T *)a.k_zero + at, *const scale = (const T *)a.k_scale + at;
    struct alignas(4 * sizeof(T)) Four { T v[4]; };
    const double levels = (double)a.levels, half = 0.5 * levels;
    // (of every 32 channels the lanes' first two lie side by side, then their second two: as they come, half of the reads' cycles were bank conflicts,
    // 12.4 us for the call above and 9.7 so)
    auto place = [](int d) __attribute__((always_inline)) { return (d & ~31) | (d & 2) << 3 | (d >> 2 & 7) << 1 | (d & 1); };
    uint64_t best = 0;   // (no score's key)
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += RW) {
        if (r0 > 0) __syncthreads();
        Four z[STEPS], t[STEPS];
        auto load = [&](int from) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const int d = from + part * 4 + 32 * k;
                if (WIDE && d < D) {
                    z[k] = *(const Four *)(zero + d);
                    t[k] = *(const Four *)(scale + d);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        z[k].v[e] = d + e < D ? zero[d + e] : (T)0.f;
                        t[k].v[e] = d + e < D ? scale[d + e] : (T)0.f;
                    }
                }
            }
        };
        load(0);
        auto fill = [&](auto value) __attribute__((always_inline)) {
            float y[RW];
#pragma unroll
            for (int r = 0; r < RW; ++r) {
                const int x = r0 + r < rows ? r0 + r : rows - 1;
                y[r] = tid < D ? value((((int64_t)b * a.Hq + hkv * G + x % G) * a.Sq + pos0 + x / G) * D + tid) : 0.f;
            }
            if (tid < room)
#pragma unroll
                for (int r = 0; r < RW; ++r) qs[r * room + place(tid)] = (double)y[r];
        };
        if (a.dtype == VQ_F16) fill([&](int64_t i) { return (float)((const f16 *)a.q)[i]; });
        else if (a.dtype == VQ_BF16) fill([&](int64_t i) { return bf16_to_f32(((const u16 *)a.q)[i]); });
        else fill([&](int64_t i) { return ((const float *)a.q)[i]; });
        __syncthreads();
        double sum[RW];
#pragma unroll
        for (int r = 0; r < RW; ++r) sum[r] = 0.;
#pragma unroll 1
        for (int d0 = 0; d0 < D; d0 += 32 * STEPS) {
            if (d0 > 0) load(d0);
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const int d = d0 + 32 * k;
                if (d >= D) break;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double td = (double)(float)t[k].v[e], m = __builtin_fma(half, td, (double)(float)z[k].v[e]), w = half * __builtin_fabs(td);
#pragma unroll
                    for (int r = 0; r < RW; ++r) {
                        const double y = qs[r * room + d + place(part * 4 + e)];
                        sum[r] = __builtin_fma(y, m, sum[r]);
                        sum[r] = __builtin_fma(__builtin_fabs(y), w, sum[r]);
                    }
                }
            }
        }
        auto take = [&](int r, double x) __attribute__((always_inline)) {   // (the row's score, in each of the group's lanes)
            const int row = r0 + r;
            if (row < rows && u < groups && u * g < sel_end(a, live, pos0 + row / G)) best = max_key(best, pick_key(x));
        };
        // A group's score hangs on its own numbers alone: of equal groups none may be rounded another way because its neighbour in the wave is not finite.
        u32 odd = 0;   // rows whose score is not finite
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            const double x = sum_parts(sum[r], 8);
            if (__builtin_fabs(x) < (double)INFINITY) take(r, x);
            else odd |= 1u << r;
        }
        if (__any(odd != 0)) {
#pragma unroll 1
            for (int r = 0; r < RW; ++r) {
                double s = 0., p = 0.;
                for (int d0 = part * 4; d0 < D; d0 += 32)
                    for (int d = d0; d < d0 + 4 && d < D; ++d) {
                        const double y = qs[r * room + place(d)], x = y * (double)(float)scale[d];
                        s = __builtin_fma(y, (double)(float)zero[d], s);
                        p += x <= 0. ? 0. : x;
                    }
                const double x = sum_parts(__builtin_fma(levels, p, s), 8);
                if (odd >> r & 1) take(r, x);
            }
        }
    }
    if (part == 0 && u < groups) c.stored[item * c.groups + u] = best;
}

// ---- the matrix units as a filter

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef u32 u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u32 positive(u32 x) { return __builtin_bit_cast(u32, __builtin_elementwise_max(as_h2(x), f16x2{(f16)0.f, (f16)0.f})); }
__device__ __forceinline__ u32 max_bits(u32 x, u32 y) {   // of two magnitudes each
    return __builtin_bit_cast(u32, __builtin_elementwise_max(__builtin_bit_cast(u16x2, x), __builtin_bit_cast(u16x2, y)));
}
// of two magnitudes each, of the second its bits less one: zeros are the largest
__device__ __forceinline__ u32 min_bits(u32 x, u32 y) {
    return __builtin_bit_cast(u32, __builtin_elementwise_min(__builtin_bit_cast(u16x2, x), (u16x2)(__builtin_bit_cast(u16x2, y) - (u16x2){1, 1})));
}
// the smallest of three halves each, NaN where one is (none the result of a matrix product)
__device__ __forceinline__ u32 low3(u32 x, u32 y, u32 z) {
    u32 r;
    asm("v_pk_minimum3_f16 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}

// Bounds of 32 rows (the query heads of a kv head at the queries of a tile) and 32 groups a step, in float32:
//
//   sum_c max(q z, q (z + L s)) = q . z + L (q+ . s+ + q- . s-),   x+ = max(x, 0), x- = max(-x, 0)
//
// products of fp16 numbers with v_mfma_f32_32x32x16 (the last one only where a scale is negative; lane n = lane % 32, h = lane / 32: row or group n,
// channels 16 ks + 8 h ..).  A wave keeps its rows' queries, walks a run of units of 32 groups and writes each group's largest bound over its rows.
// bf16 queries become fp16 numbers by a power of two that puts a row tile's largest near 2^15.  A float32 sum of D terms, each cut to 24 bits of the
// largest, is off by less than D 2^-23 of the magnitudes' sum: the scores by (D + 16) 2^-23 A, A = sum |q| (|z| + L |s|), which the wave forms too, by a third product: the choice knows how far to trust the scores (with A
// bounded by the largest sum of |q| times the largest |z| + L |s| it asked 64 bits for 3 to 5 blocks a tile).  Bound by the bytes of the scales and zeros for one query a sequence.
// Zeros and scales come asynchronously, in whole stretches of 1 KB, into the wave's ring, the next unit's ahead (as loads of a lane's own operands they touch a
// cache line in four instructions: 16 sequences at 32k 27 us, and 21.5 so); pieces of a row lie rotated by the row, so that the lanes that read them
// spread over the banks.
template <int D> struct BoundRing { static constexpr int HALF = 64 * D, BYTES = 2 * HALF, COPIES = HALF / 1024; };   // a wave's: zeros, scales of 32 groups

// One wave's run: units u0, u0 + stride, .. of 32 groups below u1 (in groups; u0 < u1), each group's score to out; returns the largest
// A (the same in every lane; not finite where a query, scale or zero is not).
template <int D, bool BF16>
__device__ __forceinline__ float bound_units(const SelectCall &c, int b, int hkv, int tile, int rt, int live, int u0, int u1, int stride, float *out, char *ring) {
    constexpr int KS = D / 16, CH = D / 8, N = BoundRing<D>::COPIES;
    const vq_block_select_args &a = c.a;
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5, G = (int)a.Hq / (int)a.Hkv, g = a.group;
    const int pos0 = tile * (int)c.query_block, rows = (sel_last(a, tile) - pos0 + 1) * G;
    const int64_t first = ((int64_t)b * a.Hkv + hkv) * c.stride * D;
    const u16 *const zeros = (const u16 *)a.k_zero + first, *const scales = (const u16 *)a.k_scale + first;
    constexpr int TURN = D >= 128 ? CH / 4 : 1;   // copies until the pieces lie as in the first one
    u32 place[TURN];
#pragma unroll
    for (int x = 0; x < TURN; ++x) {
        const int t = x * (64 / CH) + lane / CH;
        place[x] = (u32)(t * D * 2 + sp_kpiece<D>(t, lane % CH) * 16);
    }
    auto copy = [&](const u16 *from, int u, u32 to) __attribute__((always_inline)) {
        const u16 *base = from + (int64_t)u * D;
        if (u1 - u >= 32) {
#pragma unroll
            for (int x = 0; x < N; ++x) lds_copy16<0>(base + x / TURN * (TURN * 512), place[x % TURN], to + x * 1024);
        } else {   // (a group past the run's repeats the last)
#pragma unroll 1
            for (int x = 0; x < N; ++x) {
                const int t = x * (64 / CH) + lane / CH, row = t < u1 - u ? t : u1 - u - 1;
                lds_copy16<0>(base, (u32)(row * D * 2 + sp_kpiece<D>(t, lane % CH) * 16), to + x * 1024);
            }
        }
    };
    auto read = [&](const char *from, u32x4 (&x)[KS]) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < KS; ++k) x[k] = *(const u32x4 *)(from + n * D * 2 + sp_kpiece<D>(n, 2 * k + h) * 16);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (before a copy may land there)
    };
    const u32 zeros_at = lds_addr(ring), scales_at = zeros_at + BoundRing<D>::HALF;
    copy(zeros, u0, zeros_at);
    copy(scales, u0, scales_at);
    auto row_at = [&](int x) __attribute__((always_inline)) { x += rt * 32; return x < rows ? x : rows - 1; };
    u32x4 q[KS];
    {
        const int x = row_at(n);
        const u16 *src = (const u16 *)a.q + (((int64_t)b * a.Hq + hkv * G + x % G) * a.Sq + pos0 + x / G) * D + 8 * h;
#pragma unroll
        for (int k = 0; k < KS; ++k) q[k] = *(const u32x4 *)(src + 16 * k);
    }
    float unscale = 1.f;
    if constexpr (BF16) {
        u32 top = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max_bits(top, q[k][i] & 0x7FFF7FFFu);
        top = top >> 16 > (top & 0xFFFFu) ? top >> 16 : top & 0xFFFFu;
        top = wave_max_bits(top);
        // 2^(141 - e) with e the largest's exponent field: below 2^15; what is not finite stays so
        const int e = (int)(top >> 7), up = e == 0 || e == 255 ? 0 : 141 - e;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                q[k][i] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_pkrtz(__builtin_amdgcn_ldexpf(__uint_as_float(q[k][i] << 16), up),
                                                                             __builtin_amdgcn_ldexpf(__uint_as_float(q[k][i] & 0xFFFF0000u), up)));
        unscale = __builtin_amdgcn_ldexpf(1.f, -up);
    }
    const float levels = (float)a.levels;
    float small = 0.f;   // what rounded zeros and scales below the normal numbers are off by, (1 + L) 2^-25 sum |q|, as a part of A (see pick_error), twice
    if (c.narrow) {
        small = 0x1p-6f;   // (queries below the normal numbers, which may count as zero here)
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) small = __builtin_amdgcn_fdot2(as_h2(q[k][i] & 0x7FFF7FFFu), f16x2{(f16)1.f, (f16)1.f}, small, false);
        small = wave_max(small + __shfl_xor(small, 32));
        small *= (1.f + levels) * 0x1p-13f;
#pragma unroll
        for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(q[k]));   // (the magnitudes are not kept)
    }
    const u32 levels2 = __builtin_bit_cast(u32, f16x2{(f16)levels, (f16)levels});
    const int seen = sel_end(a, live, pos0);   // by every query
    u32 most = 0;   // bits of the largest sum of |q| (|z| + L |s|), NaN above infinity above all else
#pragma unroll 1
    for (int u = u0; u < u1; u += stride) {
        const bool more = u + stride < u1;
        if constexpr (D == 256) {   // (what is formed of the queries is held across the steps elsewhere)
#pragma unroll
            for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(q[k]));
        }
        f32x16 S, W, A;
#pragma unroll
        for (int r = 0; r < 16; ++r) S[r] = W[r] = A[r] = 0.f;
        u32x4 x[KS], y[KS];
        wait_copies<N>();   // the scales' copies may be under way
        read(ring, x);
        if (more) copy(zeros, u + stride, zeros_at);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            S = SpanMma<f16>::mma(q[k], x[k], S);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[k][i] = x[k][i] & 0x7FFF7FFFu;
        }
        if (more) wait_copies<N>();
        else wait_copies<0>();
        read(ring + BoundRing<D>::HALF, x);
        if (more) copy(scales, u + stride, scales_at);
        u32 low = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; i += 2) low = low3(low, x[k][i], x[k][i + 1]);
        const bool negative = __any(low != 0);   // a scale below zero, or NaN
        // A over |z| + L |s| as fp16 numbers, off by 2^-11 of themselves
        auto sum = [&](int k, u32 mask) __attribute__((always_inline)) {
            u32x4 p, size;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                size[i] = as_u(__builtin_elementwise_fma(as_h2(x[k][i] & mask), as_h2(levels2), as_h2(y[k][i])));
                p[i] = q[k][i] & 0x7FFF7FFFu;
                // (a bf16 query far below its tile's largest is cut to a multiple of 2^-24: as magnitudes of 2^-7 or more cover that too)
                if (BF16) p[i] = max_bits(p[i], 0x20002000u);
            }
            A = SpanMma<f16>::mma(p, size, A);
        };
        if (!negative) {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                sum(k, ~0u);
                u32x4 p;
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = positive(q[k][i]);
                W = SpanMma<f16>::mma(p, x[k], W);
            }
        } else {
#pragma unroll
            for (int k = 0; k < KS; ++k) sum(k, 0x7FFF7FFFu);
#pragma unroll 1
            for (int m = 0; m < 2; ++m) {
                const u32 flip = m ? 0x80008000u : 0u;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    u32x4 p, t;
#pragma unroll
                    for (int i = 0; i < 4; ++i) { p[i] = positive(q[k][i] ^ flip); t[i] = positive(x[k][i] ^ flip); }
                    W = SpanMma<f16>::mma(p, t, W);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) { const u32 bits = __float_as_uint(A[r]); most = bits > most ? bits : most; }
#pragma unroll
        for (int r = 0; r < 16; ++r) S[r] = __builtin_fmaf(levels, W[r], S[r]);
        if ((u + 31) * (int64_t)g >= seen) {   // groups that some queries do not see (in 64 bits: the last ones may lie past the store)
            const int at = u + n < u1 ? u + n : u1 - 1;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int x2 = row_at(8 * (r / 4) + 4 * h + r % 4);
                if (at * g >= sel_end(a, live, pos0 + x2 / G)) S[r] = -INFINITY;
            }
        }
        float best = S[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) best = fmaxf(best, S[r]);
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(best), __float_as_uint(best), false, false);
        best = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * unscale;
        if (h == 0 && u + n < u1) out[u + n] = best;
    }
    return (__uint_as_float(wave_max_bits(most)) + small) * unscale;
}

// Items of many rows, and few of many groups: a wave a run of units, scores and bounds to memory.
template <int D, bool BF16> __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) void block_bound_kernel(SelectCall c) {
    extern __shared__ __align__(16) char rings[];
    const vq_block_select_args &a = c.a;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u32 id = blockIdx.x * 4 + (u32)wave;
    if (id >= (u32)c.items * (u32)c.row_tiles * (u32)c.runs) return;
    const int run = (int)(id % (u32)c.runs);
    const u32 tile_row = id / (u32)c.runs;   // (item, row tile)
    const u32 item = tile_row / (u32)c.row_tiles, bh = item / (u32)c.tiles;
    const int tile = (int)(item % (u32)c.tiles), hkv = (int)(bh % (u32)a.Hkv), b = (int)(bh / (u32)a.Hkv), live = sel_live(a, b);
    const int groups = (sel_end(a, live, sel_last(a, tile)) + a.group - 1) / a.group;   // that some row sees
    const int u0 = run * c.run_units * 32, u1 = u0 + c.run_units * 32 < groups ? u0 + c.run_units * 32 : groups;
    float bound = 0.f;
    if (u0 < u1) bound = bound_units<D, BF16>(c, b, hkv, tile, (int)(tile_row % (u32)c.row_tiles), live, u0, u1, 32, c.approx + (int64_t)tile_row * c.groups,
                                                   rings + wave * BoundRing<D>::BYTES);
    if ((threadIdx.x & 63) == 0) c.bounds[id] = bound;
}

// Float32 zeros and scales of the groups that a sequence sees, rounded to fp16: eight channels a thread.
__global__ __launch_bounds__(256) void narrow_kernel(SelectCall c) {
    const vq_block_select_args &a = c.a;
    const u32 pieces = (u32)(c.groups * a.D / 8), id = blockIdx.x * 256 + threadIdx.x, bh = id / pieces, at = id % pieces;
    if (bh >= (u32)(a.B * a.Hkv)) return;
    const int64_t u = at * 8 / (u32)a.D;
    if (u * a.group >= sel_live(a, (int)(bh / (u32)a.Hkv))) return;
    const int64_t from = (int64_t)bh * c.wide_stride * a.D + (int64_t)at * 8;
    u16 *const to = c.copies + (int64_t)id * 8;
    const f32x4 z0 = *(const f32x4 *)(c.wide_zero + from), z1 = *(const f32x4 *)(c.wide_zero + from + 4), s0 = *(const f32x4 *)(c.wide_scale + from), s1 = *(const f32x4 *)(c.wide_scale + from + 4);
    f16x8 z, s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        z[i] = (f16)z0[i]; z[4 + i] = (f16)z1[i];
        s[i] = (f16)s0[i]; s[4 + i] = (f16)s1[i];
    }
    *(f16x8 *)to = z;
    *(f16x8 *)(to + a.B * a.Hkv * c.groups * a.D) = s;
}

// ---- the choice

// The key of group u's score in 64 bits, the largest over the tile's rows, by a wave: 64 / R lanes a row (R the rows, up to the next power of two),
// eight channels at a time.
__device__ __forceinline__ uint64_t exact_key(const SelectCall &c, int b, int hkv, int tile, int live, int u) {
    constexpr int AHEAD = 8;   // steps of the channels whose loads are under way at once
    const vq_block_select_args &a = c.a;
    const int lane = threadIdx.x & 63, G = (int)a.Hq / (int)a.Hkv, D = (int)a.D, g = a.group;
    const int pos0 = tile * (int)c.query_block, rows = (sel_last(a, tile) - pos0 + 1) * G;
    int many = 1;
    while (many < rows && many < 64) many <<= 1;
    const int parts = 64 / many, part = lane % parts;
    const int64_t at = (((int64_t)b * a.Hkv + hkv) * c.stride + u) * D;
    const u16 *const zero = (const u16 *)a.k_zero + at, *const scale = (const u16 *)a.k_scale + at;
    const bool bf16 = a.dtype == VQ_BF16;
    uint64_t best = 0;
    for (int r0 = 0; r0 < rows; r0 += many) {
        const int r = r0 + lane / parts, x = r < rows ? r : rows - 1, end = sel_end(a, live, pos0 + x / G);
        const u16 *q = (const u16 *)a.q + (((int64_t)b * a.Hq + hkv * G + x % G) * a.Sq + pos0 + x / G) * D;
        double s = 0., w = 0.;
        for (int d0 = part * 8; d0 < D; d0 += AHEAD * parts * 8) {
            u32x4 x4[AHEAD], z4[AHEAD], s4[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int d = d0 + k * parts * 8;
                if (k > 0 && d >= D) { x4[k] = z4[k] = s4[k] = u32x4{0, 0, 0, 0}; continue; }
                x4[k] = *(const u32x4 *)(q + d);
                z4[k] = *(const u32x4 *)(zero + d);
                s4[k] = *(const u32x4 *)(scale + d);
            }
            // Products are exact in float32 (22 bits), where no bf16 query lies outside 2^-63 .. 2^64
            u32 top = 0, low = ~0u;   // of the magnitudes' bits, the lower end less one, so that zeros are not it
            if (bf16) {
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const u32 size = x4[k][i] & 0x7FFF7FFFu;
                        top = max_bits(top, size);
                        low = min_bits(low, size);
                    }
            }
            const bool narrow = !bf16 || ((top >> 16) < 0x5F80u && (top & 0xFFFFu) < 0x5F80u && (low >> 16) >= 0x2000u && (low & 0xFFFFu) >= 0x2000u);
            auto add = [&](auto product) __attribute__((always_inline)) {
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    if (k > 0 && d0 + k * parts * 8 >= D) break;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const u16 xb = (u16)(x4[k][i / 2] >> (16 * (i & 1)));
                        product(bf16 ? bf16_to_f32(xb) : (float)__builtin_bit_cast(f16, xb), (float)as_h2(z4[k][i / 2])[i & 1], (float)as_h2(s4[k][i / 2])[i & 1]);
                    }
                }
            };
            if (__all(narrow))
                add([&](float y, float z, float t) __attribute__((always_inline)) {
                    const float p = y * t;
                    s += (double)(y * z);
                    w += (double)(p <= 0.f ? 0.f : p);
                });
            else
                add([&](double y, double z, double t) __attribute__((always_inline)) {
                    const double p = y * t;
                    s += y * z;
                    w += p <= 0. ? 0. : p;
                });
        }
        s += (double)a.levels * w;
        s = sum_parts(s, parts);
        if (u * g < end) best = max_key(best, pick_key(s));
    }
    for (int off = 32; off >= parts; off >>= 1) best = max_key(best, __shfl_xor((unsigned long long)best, off));
    return best;
}

// The same from float32 scales and zeros.
__device__ __forceinline__ uint64_t exact_key_wide(const SelectCall &c, int b, int hkv, int tile, int live, int u) {
    constexpr int AHEAD = 4;
    const vq_block_select_args &a = c.a;
    const int lane = threadIdx.x & 63, G = (int)a.Hq / (int)a.Hkv, D = (int)a.D, g = a.group;
    const int pos0 = tile * (int)c.query_block, rows = (sel_last(a, tile) - pos0 + 1) * G;
    int many = 1;
    while (many < rows && many < 64) many <<= 1;
    const int parts = 64 / many, part = lane % parts;
    const int64_t at = (((int64_t)b * a.Hkv + hkv) * c.wide_stride + u) * D;
    const float *const zero = c.wide_zero + at, *const scale = c.wide_scale + at;
    const bool bf16 = a.dtype == VQ_BF16;
    uint64_t best = 0;
    for (int r0 = 0; r0 < rows; r0 += many) {
        const int r = r0 + lane / parts, x = r < rows ? r : rows - 1, end = sel_end(a, live, pos0 + x / G);
        const u16 *q = (const u16 *)a.q + (((int64_t)b * a.Hq + hkv * G + x % G) * a.Sq + pos0 + x / G) * D;
        double s = 0., w = 0.;
        for (int d0 = part * 4; d0 < D; d0 += AHEAD * parts * 4) {
            u32x2 x2[AHEAD];
            f32x4 z4[AHEAD], s4[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int d = d0 + k * parts * 4;
                if (k > 0 && d >= D) { x2[k] = u32x2{0, 0}; z4[k] = s4[k] = f32x4{0.f, 0.f, 0.f, 0.f}; continue; }
                x2[k] = *(const u32x2 *)(q + d);
                z4[k] = *(const f32x4 *)(zero + d);
                s4[k] = *(const f32x4 *)(scale + d);
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u16 xb = (u16)(x2[k][i / 2] >> (16 * (i & 1)));
                    const double y = bf16 ? bf16_to_f32(xb) : (float)__builtin_bit_cast(f16, xb), p = y * (double)s4[k][i];
                    s = __builtin_fma(y, (double)z4[k][i], s);
                    w += p <= 0. ? 0. : p;
                }
        }
        s = __builtin_fma((double)a.levels, w, s);
        s = sum_parts(s, parts);
        if (u * g < end) best = max_key(best, pick_key(s));
    }
    for (int off = 32; off >= parts; off >>= 1) best = max_key(best, __shfl_xor((unsigned long long)best, off));
    return best;
}

constexpr int PICK_MOST = 16384;   // blocks whose scores are held in LDS
constexpr int ONE_SCORES = 20 * 1024;   // bytes of scores beside the rings of eight waves
constexpr int PICK_LIST = 512;     // blocks that are told apart in 64 bits there

template <int THREADS> struct PickRoom {
    static constexpr int WAVES = THREADS / 64;
    u32 hist[THREADS], waves[WAVES], found[2];
    float low[WAVES], high[WAVES], off_by[WAVES];
    int list[PICK_LIST];
    uint64_t exact[PICK_LIST];
};

// How many threads below this one say `one` (lower half) and `two` (upper half; counts below 2^16), and in `total` how many in all.  (Two barriers
// around each use of `waves`.)
template <int WAVES> __device__ __forceinline__ u32 block_before(bool one, bool two, u32 &total, u32 *waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t m1 = __ballot(one), m2 = __ballot(two), below = (UINT64_C(1) << lane) - 1;
    __syncthreads();
    if (lane == 0) waves[wave] = (u32)__popcll(m1) | (u32)__popcll(m2) << 16;
    __syncthreads();
    u32 before = (u32)__popcll(m1 & below) | (u32)__popcll(m2 & below) << 16;
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const u32 x = waves[w];
        before += w < wave ? x : 0;
        total += x;
    }
    return before;
}

// The bin that holds the `left`-th from the highest bin down (a thread each, the highest bin's first); `left` becomes how many of that bin are
// wanted.  (A barrier lies between the last count and the call.)
template <int WAVES> __device__ __forceinline__ int pick_bin(const u32 *hist, u32 &left, u32 *waves, u32 *found) {
    const int tid = threadIdx.x, wave = tid >> 6, bin = WAVES * 64 - 1 - tid;
    const u32 mine = hist[bin], sum = wave_sum_up(mine);
    if ((tid & 63) == 63) waves[wave] = sum;
    __syncthreads();
    u32 above = sum - mine;
#pragma unroll
    for (int w = 0; w < WAVES - 1; ++w) above += w < wave ? waves[w] : 0;
    if (above < left && above + mine >= left) { found[0] = (u32)bin; found[1] = left - above; }
    __syncthreads();
    left = found[1];
    return (int)found[0];
}

// A tile's place, what it sees, and the choices that need no score: all of at most `count` visible blocks, and else the first and the recent ones.
// False: nothing is left to choose.
struct PickTile {
    int b, hkv, tile, live, lo, n;   // (blocks lo .. lo + n - 1 to choose from)
    int per, seen;                   // groups of a block, groups that some row sees
    u32 want;
};
__device__ __forceinline__ bool pick_begin(const SelectCall &c, PickTile &t) {
    const vq_block_select_args &a = c.a;
    const u32 bh = blockIdx.x / (u32)c.tiles;
    t.tile = (int)(blockIdx.x % (u32)c.tiles);
    t.hkv = (int)(bh % (u32)a.Hkv);
    t.b = (int)(bh / (u32)a.Hkv);
    t.live = sel_live(a, t.b);
    const int end = sel_end(a, t.live, sel_last(a, t.tile));
    t.per = (int)a.block_tokens / a.group;
    t.seen = (end + a.group - 1) / a.group;
    const int V = (int)((u32)(end + (int)a.block_tokens - 1) / (u32)a.block_tokens), count = (int)a.count;
    int32_t *out = a.out + (int64_t)blockIdx.x * count;
    if (V <= count) {
        for (int i = threadIdx.x; i < count; i += blockDim.x) out[i] = i < V ? i : -1;
        return false;
    }
    t.lo = (int)a.first;
    t.n = V - (int)a.recent - t.lo;
    t.want = (u32)(count - (int)a.first - (int)a.recent);   // of n, which are more
    for (int i = threadIdx.x; i < t.lo; i += blockDim.x) out[i] = i;
    for (int i = threadIdx.x; i < (int)a.recent; i += blockDim.x) out[count - (int)a.recent + i] = t.lo + t.n + i;
    return t.want > 0;
}

// The choice of a tile, by a block of threads.  keys: the approximate scores of the blocks [lo, hi) from this thread's blocks on, in LDS; `least`, `most`, `e`: of this
// thread's, the last one how far a score may be off, infinite where something is not finite.
//
// The kth best is looked for among the approximate scores by bins between the smallest and the largest, again inside its bin while
// that holds many, then in the bin's order.  With scores off by e at most, those more than 2 e above it are among the chosen, those more than 2 e
// below are not; if not all of the few between are wanted, these are told apart by their scores in 64 bits, a wave a group.  Where these are more than
// PICK_LIST (equal scores, values that are not finite, which make e so) they are by a radix select over the bits.
// STORED: the scores of 64 bits lie in memory; else they are formed here.
template <bool STORED, int THREADS>
__device__ __forceinline__ void pick(const SelectCall &c, PickRoom<THREADS> &room, float *keys, const PickTile &t, float least, float most, float e) {
    constexpr int WAVES = THREADS / 64;
    const vq_block_select_args &a = c.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int32_t *out = a.out + (int64_t)blockIdx.x * a.count;
    uint64_t *const score = c.exact + (int64_t)blockIdx.x * c.total;
    const int b = t.b, hkv = t.hkv, tile = t.tile, live = t.live, lo = t.lo, n = t.n, per = t.per, seen = t.seen;
    const u32 want = t.want;
    // the key of group i of block j, by a wave; 0 behind the last group that some row sees
    auto key_of = [&](int j, int i) __attribute__((always_inline)) -> uint64_t {
        const int u = (lo + j) * per + i;
        if (u >= seen) return 0;
        if (STORED) return c.stored[(int64_t)blockIdx.x * c.groups + u];
        return c.narrow ? exact_key_wide(c, b, hkv, tile, live, u) : exact_key(c, b, hkv, tile, live, u);
    };
    least = wave_min(least);
    most = wave_max(most);
    e = wave_max(e);
    if (lane == 0) { room.low[wave] = least; room.high[wave] = most; room.off_by[wave] = e; }
    room.hist[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) { least = fminf(least, room.low[w]); most = fmaxf(most, room.high[w]); e = fmaxf(e, room.off_by[w]); }
    e = 2.f * e + 0x1p-100f;   // of two scores' difference, also where products are too small for float32

    // ---- the bin of the kth best
    u32 left = want, among = (u32)n;
    float from = least, to = most;
    if (e < INFINITY) {
#pragma unroll 1
        for (int pass = 0; pass < 4 && among > 32 && to - from > e; ++pass) {
            const float by = (float)(THREADS - 1) / (to - from);   // (the last bin: the largest alone)
            if (pass > 0) {
                room.hist[tid] = 0;
                __syncthreads();
            }
            for (int j = tid; j < n; j += THREADS) {
                const float x = keys[j];
                if (x >= from && x <= to) atomicAdd(&room.hist[(u32)((x - from) * by) % THREADS], 1u);
            }
            __syncthreads();
            const u32 bin = (u32)pick_bin<WAVES>(room.hist, left, room.waves, room.found);
            among = room.hist[bin];
            if (among <= 32 || pass == 3) {   // (by its edges, and what rounding may put beside them)
                const float width = (to - from) / (float)(THREADS - 1), edge = from + ((float)bin + 1.001f) * width;
                from += ((float)bin - 0.001f) * width;
                to = edge < to ? edge : to;
                break;
            }
            float l = INFINITY, m = -INFINITY;
            for (int j = tid; j < n; j += THREADS) {
                const float x = keys[j];
                if (x >= from && x <= to && (u32)((x - from) * by) % THREADS == bin) { l = fminf(l, x); m = fmaxf(m, x); }
            }
            l = wave_min(l);
            m = wave_max(m);
            if (lane == 0) { room.low[wave] = l; room.high[wave] = m; }
            __syncthreads();
            from = room.low[0]; to = room.high[0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) { from = fminf(from, room.low[w]); to = fmaxf(to, room.high[w]); }
        }
    }
    // ---- the list of those that may be the kth best, or are within e of it; t: the kth best's score, where the list is short
    float over = e < INFINITY ? to + e : INFINITY, under = e < INFINITY ? from - e : -INFINITY;
    u32 sure = 0, listed = 0;
    u32 at_of[2] = {0, 0};   // of this thread's first two: how many are listed before it, how many sure ones (upper half)
    bool sure_of[2] = {false, false}, listed_of[2] = {false, false};
    for (int j0 = 0, turn = 0; j0 < n; j0 += THREADS, ++turn) {
        const float x = j0 + tid < n ? keys[j0 + tid] : -INFINITY;
        const bool here = j0 + tid < n, in = here && x > over, maybe = here && !in && !(x < under);
        u32 some;
        const u32 before = block_before<WAVES>(maybe, in, some, room.waves), at = listed + (before & 0xFFFFu);
        if (maybe && at < PICK_LIST) room.list[at] = j0 + tid;
        if (turn == 0) { at_of[0] = before; sure_of[0] = in; listed_of[0] = maybe; }
        if (turn == 1) { at_of[1] = before + (listed | sure << 16); sure_of[1] = in; listed_of[1] = maybe; }
        listed += some & 0xFFFFu;
        sure += some >> 16;
    }
    const u32 need = want - sure;   // of the list
    __syncthreads();
    if (listed <= 64) {   // every wave the same
        const int j = room.list[lane < (int)listed ? lane : 0];
        const float x = lane < (int)listed ? keys[j] : -INFINITY;
        u32 rank = 0;   // (equal ones in the list's order)
        for (int o = 0; o < (int)listed; ++o) { const float y = __uint_as_float((u32)__builtin_amdgcn_readlane(__float_as_uint(x), o)); rank += y > x || (y == x && o < lane) ? 1 : 0; }
        const uint64_t kth = __ballot(lane < (int)listed && rank == need - 1);
        const float t = __uint_as_float((u32)__builtin_amdgcn_readlane(__float_as_uint(x), kth != 0 ? __builtin_ctzll(kth) : 0));   // (none among values that are not finite: e is not either)
        const bool in = lane < (int)listed && x > t + e, maybe = lane < (int)listed && !in && !(x < t - e);
        const uint64_t m = __ballot(maybe);
        const u32 doubt = (u32)__popcll(m), wanted = need - (u32)__popcll(__ballot(in));
        const bool all = doubt == wanted;
        if (all && n <= 2 * THREADS) {   // (every wave knows the taken ones of the list: the places of all follow)
            const uint64_t taken = __ballot(in || maybe);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const u32 at = at_of[k] & 0xFFFFu, before = at < 64 ? (u32)__popcll(taken & ((UINT64_C(1) << at) - 1)) : (u32)__popcll(taken);
                if (sure_of[k] || (listed_of[k] && (taken >> (at & 63) & 1))) out[lo + (int)(before + (at_of[k] >> 16))] = lo + k * THREADS + tid;
            }
            return;
        }
        const u32 mine = (u32)__popcll(m & ((UINT64_C(1) << lane) - 1));   // this lane's place among the doubtful
        if (wave == 0 && maybe) { room.list[64 + mine] = j; room.exact[mine] = 0; }
        __syncthreads();   // (every wave has read the list's scores, which the first one replaces)
        if (!all) {
            for (u32 i = wave; i < doubt * per; i += WAVES) {
                const uint64_t k = key_of(room.list[64 + i / per], i % per);
                if (lane == 0) atomicMax((unsigned long long *)&room.exact[i / per], (unsigned long long)k);
            }
            __syncthreads();
        }
        if (wave == 0 && lane < (int)listed) {
            bool take = in || (maybe && all);
            if (maybe && !all) {
                const uint64_t k = room.exact[mine];
                u32 better = 0;   // (the list ascends: of equal scores the lower block comes first)
                for (u32 o = 0; o < doubt; ++o) better += room.exact[o] > k || (room.exact[o] == k && o < mine) ? 1 : 0;
                take = better < wanted;
            }
            keys[j] = take ? INFINITY : -INFINITY;
        }
    } else if (listed <= PICK_LIST) {
        for (u32 i = tid; i < listed; i += THREADS) room.exact[i] = 0;
        __syncthreads();
        for (u32 i = wave; i < listed * per; i += WAVES) {
            const uint64_t k = key_of(room.list[i / per], i % per);
            if (lane == 0) atomicMax((unsigned long long *)&room.exact[i / per], (unsigned long long)k);
        }
        __syncthreads();
        for (u32 i = tid; i < listed; i += THREADS) {
            const uint64_t k = room.exact[i];
            u32 better = 0;
            for (u32 o = 0; o < listed; ++o) better += room.exact[o] > k || (room.exact[o] == k && o < i) ? 1 : 0;
            keys[room.list[i]] = better < need ? INFINITY : -INFINITY;
        }
    } else {
        // all of the list by their bits; the sure ones as the highest
        for (int j = wave; j < n; j += WAVES) {
            const float x = keys[j];
            uint64_t k = x > over ? ~UINT64_C(0) : 0;
            if (!(x > over) && !(x < under))
                for (int i = 0; i < per; ++i) k = max_key(k, key_of(j, i));
            if (lane == 0) score[lo + j] = k;
        }
        __threadfence_block();
        __syncthreads();
        const uint64_t *all = score + lo;
        uint64_t key = 0;
        left = want;
        for (int shift = 56; shift >= 0; shift -= 8) {
            room.hist[tid] = 0;
            __syncthreads();
            for (int j = tid; j < n; j += THREADS)
                if (shift == 56 || (all[j] ^ key) >> (shift + 8) == 0) atomicAdd(&room.hist[all[j] >> shift & 255], 1u);
            __syncthreads();
            key |= (uint64_t)pick_bin<WAVES>(room.hist, left, room.waves, room.found) << shift;
            __syncthreads();
        }
        u32 equal = 0;
        for (int j0 = 0; j0 < n; j0 += THREADS) {
            const int j = j0 + tid;
            u32 some;
            const u32 rank = equal + block_before<WAVES>(j < n && all[j] == key, false, some, room.waves);
            equal += some;
            if (j < n) keys[j] = all[j] > key || (all[j] == key && rank < left) ? INFINITY : -INFINITY;
        }
    }
    __syncthreads();
    // ---- in order
    u32 done = 0;
    for (int j0 = 0; j0 < n; j0 += THREADS) {
        const bool take = j0 + tid < n && (keys[j0 + tid] == INFINITY || keys[j0 + tid] > over);
        u32 some;
        const u32 at = done + block_before<WAVES>(take, false, some, room.waves);
        if (take) out[lo + at] = lo + j0 + tid;
        done += some;
    }
}

// A thread's blocks' approximate scores from those of their groups (row tile rt's at approx + rt * groups).
template <int THREADS> __device__ __forceinline__ void pick_blocks(const SelectCall &c, const PickTile &t, const float *approx, int row_tiles, int groups, float *keys, float &least, float &most, float &e) {
    for (int j = threadIdx.x; j < t.n; j += THREADS) {
        const int u0 = (t.lo + j) * t.per, u1 = u0 + t.per < t.seen ? u0 + t.per : t.seen;
        float x = -INFINITY;
        for (int rt = 0; rt < row_tiles; ++rt)
            for (int u = u0; u < u1; ++u) x = fmaxf(x, approx[(int64_t)rt * groups + u]);
        keys[j] = x;
        if (!(__builtin_fabsf(x) < INFINITY)) e = INFINITY;
        least = fminf(least, x);
        most = fmaxf(most, x);
    }
}
// How far a score may be off, A the bound's; scales and zeros rounded to fp16 are off by 2^-11 of themselves.
__device__ __forceinline__ float pick_error(const SelectCall &c, float bound) {
    return bound < INFINITY ? bound * ((float)(c.a.D + 16) * 0x1p-23f + (c.narrow ? 0x1.02p-11f : 0.f)) : INFINITY;
}

template <bool STORED, int THREADS> __global__ __launch_bounds__(THREADS) void block_pick_kernel(SelectCall c) {
    extern __shared__ float keys[];
    __shared__ PickRoom<THREADS> room;
    PickTile t;
    if (!pick_begin(c, t)) return;
    float least = INFINITY, most = -INFINITY, e = 0.f;
    if (STORED) {
        const uint64_t *stored = c.stored + (int64_t)blockIdx.x * c.groups;
        for (int j = threadIdx.x; j < t.n; j += THREADS) {
            uint64_t k = 0;
            for (int u = (t.lo + j) * t.per; u < (t.lo + j + 1) * t.per && u < t.seen; ++u) k = max_key(k, stored[u]);
            const float x = (float)key_score(k);
            keys[j] = x;
            e = __builtin_fabsf(x) < INFINITY ? fmaxf(e, __builtin_fabsf(x) * 0x1p-23f) : INFINITY;
            least = fminf(least, x);
            most = fmaxf(most, x);
        }
    } else {
        const int many = c.row_tiles * c.runs;
        for (int i = threadIdx.x; i < many; i += THREADS) e = fmaxf(e, pick_error(c, c.bounds[(int64_t)blockIdx.x * many + i]));
        pick_blocks<THREADS>(c, t, c.approx + (int64_t)blockIdx.x * c.row_tiles * c.groups, c.row_tiles, (int)c.groups, keys, least, most, e);
    }
    pick<STORED, THREADS>(c, room, keys, t, least, most, e);
}

// Scores and choice of a tile of up to 32 rows in one block, the scores in LDS.
template <int D, bool BF16, int THREADS>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) void block_choose_kernel(SelectCall c) {
    constexpr int WAVES = THREADS / 64;
    extern __shared__ __align__(16) char rings[];   // of the waves, then the scores of the blocks and of the groups
    float *const keys = (float *)(rings + WAVES * BoundRing<D>::BYTES);
    __shared__ PickRoom<THREADS> room;
    PickTile t;
    if (!pick_begin(c, t)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), u0 = t.lo * t.per,
              u1 = (t.lo + t.n) * t.per < t.seen ? (t.lo + t.n) * t.per : t.seen;   // the groups of those to choose from
    float *const approx = keys + c.total;
    float least = INFINITY, most = -INFINITY, e = 0.f;
    if (u0 + wave * 32 < u1) e = pick_error(c, bound_units<D, BF16>(c, t.b, t.hkv, t.tile, 0, t.live, u0 + wave * 32, u1, WAVES * 32, approx,
                                                                       rings + wave * BoundRing<D>::BYTES));
    __syncthreads();
    pick_blocks<THREADS>(c, t, approx, 1, 0, keys, least, most, e);
    pick<false, THREADS>(c, room, keys, t, least, most, e);
}

// The same over any number of blocks, their scores of 64 bits in memory throughout.
__global__ __launch_bounds__(256) void block_pick_any_kernel(SelectCall c) {
    constexpr int THREADS = 256, WAVES = THREADS / 64;
    __shared__ u32 hist[THREADS], waves[WAVES], found[2];
    PickTile t;
    if (!pick_begin(c, t)) return;
    const int tid = threadIdx.x;
    const uint64_t *stored = c.stored + (int64_t)blockIdx.x * c.groups;
    auto key_of = [&](int j) __attribute__((always_inline)) {
        uint64_t k = 0;
        for (int u = (t.lo + j) * t.per; u < (t.lo + j + 1) * t.per && u < t.seen; ++u) k = max_key(k, stored[u]);
        return k;
    };
    int32_t *out = c.a.out + (int64_t)blockIdx.x * c.a.count + t.lo;
    u32 left = t.want;
    uint64_t key = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < t.n; j += THREADS) {
            const uint64_t k = key_of(j);
            if (shift == 56 || (k ^ key) >> (shift + 8) == 0) atomicAdd(&hist[k >> shift & 255], 1u);
        }
        __syncthreads();
        key |= (uint64_t)pick_bin<WAVES>(hist, left, waves, found) << shift;
        __syncthreads();
    }
    u32 done = 0, equal = 0;
    for (int j0 = 0; j0 < t.n; j0 += THREADS) {
        const int j = j0 + tid;
        const uint64_t k = j < t.n ? key_of(j) : 0;
        u32 some;
        const u32 rank = equal + block_before<WAVES>(j < t.n && k == key, false, some, waves);
        equal += some;
        const bool take = j < t.n && (k > key || (k == key && rank < left));
        const u32 at = done + block_before<WAVES>(take, false, some, waves);
        if (take) out[at] = t.lo + j;
        done += some;
    }
}

int check_select(const char *fn, const vq_block_select_args *args) {
    VQ_REQUIRE(args != nullptr, VQ_ERR_INVALID, "%s: null argument block", fn);
    const vq_block_select_args &a = *args;
    VQ_REQUIRE(a.B >= 1 && a.Hq >= 1 && a.Hkv >= 1 && a.Sq >= 1 && a.D >= 1 && a.D <= 256, VQ_ERR_INVALID, "%s: bad sizes (heads of at most 256 channels)", fn);
    VQ_REQUIRE(a.Hq % a.Hkv == 0, VQ_ERR_INVALID, "%s: H_q=%lld must be a multiple of H_kv=%lld", fn, (long long)a.Hq, (long long)a.Hkv);
    VQ_REQUIRE(is_float_tag(a.dtype), VQ_ERR_INVALID, "%s: unsupported q dtype", fn);
    VQ_REQUIRE(a.meta_dtype == VQ_F32 || a.meta_dtype == VQ_F16, VQ_ERR_INVALID, "%s: scale and zero must be float32 or float16", fn);
    VQ_REQUIRE(a.n_packed >= 0 && a.n_tail >= 0 && a.cap_tokens >= a.n_packed, VQ_ERR_INVALID, "%s: bad token counts", fn);
    VQ_REQUIRE(a.group >= 1 && a.levels >= 1 && a.levels <= 255, VQ_ERR_INVALID, "%s: bad group size or levels", fn);
    VQ_REQUIRE(a.block_tokens >= 1 && a.block_tokens % a.group == 0, VQ_ERR_INVALID, "%s: blocks of %lld tokens are no multiple of groups of %d", fn,
               (long long)a.block_tokens, a.group);
    VQ_REQUIRE(a.query_block >= 1, VQ_ERR_INVALID, "%s: query_block must be at least 1", fn);
    VQ_REQUIRE(a.first >= 0 && a.recent >= 0 && a.count >= 1 && a.first + a.recent <= a.count, VQ_ERR_INVALID,
               "%s: %lld first and %lld recent blocks of %lld", fn, (long long)a.first, (long long)a.recent, (long long)a.count);
    VQ_REQUIRE(a.n_packed + a.n_tail < (INT64_C(1) << 30) && a.cap_tokens < (INT64_C(1) << 31) && a.block_tokens < (INT64_C(1) << 30) &&
                   a.Sq < (INT64_C(1) << 30) && a.query_block < (INT64_C(1) << 30) && a.count < (INT64_C(1) << 30),
               VQ_ERR_UNSUPPORTED, "%s: 2^30 or more slots, queries or blocks", fn);
    VQ_REQUIRE(!a.causal || a.Sq <= a.n_packed + a.n_tail, VQ_ERR_INVALID, "%s: S_q=%lld exceeds the %lld slots; queries align to their end", fn,
               (long long)a.Sq, (long long)(a.n_packed + a.n_tail));
    const double tiles = (double)cdiv(a.Sq, a.query_block), rows = (double)a.B * (double)a.Hkv * tiles;
    VQ_REQUIRE((double)a.B * (double)a.Hq * (double)a.Sq < 16777216., VQ_ERR_UNSUPPORTED, "%s: 2^24 or more query rows", fn);
    VQ_REQUIRE(rows * (double)cdiv(a.n_packed, a.group) < 67108864. && rows < 8388608., VQ_ERR_UNSUPPORTED, "%s: 2^26 or more scores", fn);
    VQ_REQUIRE(a.q != nullptr && a.out != nullptr && (a.n_packed == 0 || (a.k_scale != nullptr && a.k_zero != nullptr)), VQ_ERR_INVALID,
               "%s: null q, out, scale or zero", fn);
    return VQ_OK;
}

SelectCall cut_select(const vq_block_select_args &a) {
    SelectCall c = {};
    c.a = a;
    c.tiles = cdiv(a.Sq, a.query_block);
    c.total = cdiv(a.n_packed, a.block_tokens);
    c.items = a.B * a.Hkv * c.tiles;
    c.query_block = a.query_block < a.Sq ? a.query_block : a.Sq;
    c.groups = cdiv(a.n_packed, a.group);
    c.stride = cdiv(a.cap_tokens, a.group);
    c.row_tiles = (int)cdiv(a.Hq / a.Hkv * c.query_block, 32);
    if (c.total <= a.count) return c;   // every visible block is chosen: no scores
    // (what it costs to round them and to tell more blocks apart is earned back from some 10^8 products on: 8 kv heads of 128 channels over 524 groups, 128 rows a kv
    // head 34.5 us and 33.2 in 64 bits throughout, 256 rows 37.4 and 47.8, 2048 rows 74 and 308; 16 sequences at 32k, 4 rows a head 56 and 38, 16 rows 84 and 117)
    c.narrow = a.meta_dtype == VQ_F32 && (double)a.B * (double)a.Hq * (double)a.Sq * (double)c.groups * (double)a.D >= 1e8;
    c.mma = (a.D == 64 || a.D == 128 || a.D == 256) && a.dtype != VQ_F32 && (a.meta_dtype == VQ_F16 || c.narrow) && c.total <= PICK_MOST &&
            (((uintptr_t)a.q | (uintptr_t)a.k_scale | (uintptr_t)a.k_zero) & 15) == 0;
    if (c.mma) {
        // a unit a wave until the eight waves that a CU holds have work
        const int64_t units = cdiv(c.groups, 32), waves = c.items * c.row_tiles * units;
        c.run_units = (int)cdiv(waves, 2048);
        if (c.run_units > units) c.run_units = (int)units;
        c.runs = (int)cdiv(units, c.run_units);
        // (the products and the grid of a call of this size are left to the vector units)
        if ((double)c.items * c.row_tiles * (double)c.groups >= 67108864.) c.mma = 0;
        // One block a tile where its waves walk two units each at most, or tiles fill the chip: one sequence of 8 kv heads over 8k tokens in groups of
        // 32 11.9 us, in two launches 13.1; over 16k 13.6 and 13.4, 32k 16.1 and 13.2; four sequences of 32k 17.5 and 16.1, eight 17.9 and 19.0.
        c.one = c.mma && c.row_tiles == 1 && (c.total + c.groups) * 4 <= ONE_SCORES && (c.items >= 64 || units <= (a.D == 256 ? 8 : 16));
    }
    if (!c.mma) c.narrow = 0;
    return c;
}
struct SelectRoom { size_t stored, approx, bounds, copies, all; };
SelectRoom select_room(const SelectCall &c) {
    SelectRoom r = {};
    if (c.total <= c.a.count) return r;
    auto whole = [](size_t n) { return (n + 15) / 16 * 16; };
    r.stored = whole((size_t)(c.items * c.total) * 8);
    r.approx = r.stored + (c.mma ? 0 : whole((size_t)(c.items * c.groups) * 8));
    r.bounds = r.copies = r.approx;
    if (c.mma && !c.one) {
        r.bounds = r.approx + whole((size_t)(c.items * c.row_tiles * c.groups) * 4);
        r.copies = r.bounds + whole((size_t)(c.items * c.row_tiles * c.runs) * 4);
    }
    r.all = r.copies + (c.narrow ? (size_t)(c.a.B * c.a.Hkv * c.groups * c.a.D) * 4 : 0);
    return r;
}

// `bytes` of block-shared memory, of `most` for other calls
template <typename Kernel> int launch_of(const char *fn, Kernel kernel, int64_t blocks, int threads, size_t bytes, size_t most, std::atomic<bool> *allowed, const SelectCall &c) {
    if (bytes > 48 * 1024) {   // (with the tables beside it more than a block has unasked)
        int dev = 0;
        (void)hipGetDevice(&dev);
        if (dev < 0 || dev >= 64 || !allowed[dev].load(std::memory_order_acquire)) {
            const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)most);
            VQ_REQUIRE(e == hipSuccess, VQ_ERR_HIP, "%s: %zu bytes of block-shared memory: %s", fn, most, hipGetErrorString(e));
            if (dev >= 0 && dev < 64) allowed[dev].store(true, std::memory_order_release);
        }
    }
    kernel<<<(unsigned)blocks, threads, bytes, (hipStream_t)c.a.stream>>>(c);
    VQ_HIP_CHECK_LAUNCH(fn);
    return VQ_OK;
}
template <bool STORED> int launch_pick(const char *fn, const SelectCall &c, size_t bytes) {
    static std::atomic<bool> allowed[64] = {};
    return launch_of(fn, block_pick_kernel<STORED, 512>, c.items, 512, bytes, PICK_MOST * 4, allowed, c);
}
template <int D, bool BF16, int THREADS> int launch_one(const char *fn, const SelectCall &c) {
    constexpr size_t rings = THREADS / 64 * BoundRing<D>::BYTES;
    static std::atomic<bool> allowed[64] = {};
    return launch_of(fn, block_choose_kernel<D, BF16, THREADS>, c.items, THREADS, rings + (size_t)(c.total + c.groups) * 4, rings + ONE_SCORES, allowed, c);
}
template <int D, bool BF16> int launch_choice(const char *fn, const SelectCall &c) {
    if (c.one) {
        if constexpr (D < 256) {
            if (c.items <= 256) return launch_one<D, BF16, 512>(fn, c);
        }
        return launch_one<D, BF16, 256>(fn, c);
    }
    constexpr size_t rings = 4 * BoundRing<D>::BYTES;
    static std::atomic<bool> allowed[64] = {};
    if (int rc = launch_of(fn, block_bound_kernel<D, BF16>, cdiv(c.items * c.row_tiles * c.runs, 4), 256, rings, rings, allowed, c)) return rc;
    return launch_pick<false>(fn, c, (size_t)c.total * 4);
}
template <typename T, bool WIDE, int RW> void launch_scores_of(const SelectCall &c) {
    group_score_kernel<T, WIDE, RW><<<(unsigned)(c.items * cdiv(c.groups, SCORE_GROUPS)), 256, (size_t)RW * cdiv(c.a.D, 32) * 32 * 8, (hipStream_t)c.a.stream>>>(c);
}
template <typename T, bool WIDE> void launch_scores(const SelectCall &c) {
    const int64_t rows = c.a.Hq / c.a.Hkv * c.query_block;
    if (rows == 1) launch_scores_of<T, WIDE, 1>(c);
    else if (rows == 2) launch_scores_of<T, WIDE, 2>(c);
    else if (rows <= 4) launch_scores_of<T, WIDE, 4>(c);
    else launch_scores_of<T, WIDE, 8>(c);
}

template <int D> int launch_choice(const char *fn, const SelectCall &c) { return c.a.dtype == VQ_BF16 ? launch_choice<D, true>(fn, c) : launch_choice<D, false>(fn, c); }

}  // namespace

}  // namespace vq

extern "C" size_t vq_block_select_workspace(const vq_block_select_args *args) {
    using namespace vq;
    if (check_select("vq_block_select", args) != VQ_OK) return 0;
    return select_room(cut_select(*args)).all;
}

extern "C" int vq_block_select(const vq_block_select_args *args) {
    using namespace vq;
    const char *fn = "vq_block_select";
    if (int rc = check_select(fn, args)) return rc;
    SelectCall c = cut_select(*args);
    const vq_block_select_args &a = c.a;
    const SelectRoom room = select_room(c);
    VQ_REQUIRE(room.all == 0 || (a.workspace != nullptr && a.workspace_bytes >= room.all && ((uintptr_t)a.workspace & 15) == 0), VQ_ERR_WORKSPACE,
               "%s: workspace of %zu bytes required, 16-byte aligned", fn, room.all);
    hipStream_t st = (hipStream_t)a.stream;
    if (room.all > 0) {
        c.exact = (uint64_t *)a.workspace;
        c.stored = (uint64_t *)((char *)a.workspace + room.stored);
        c.approx = (float *)((char *)a.workspace + room.approx);
        c.bounds = (float *)((char *)a.workspace + room.bounds);
        if (c.narrow) {
            c.copies = (u16 *)((char *)a.workspace + room.copies);
            c.wide_zero = (const float *)a.k_zero;
            c.wide_scale = (const float *)a.k_scale;
            c.wide_stride = c.stride;
            c.stride = c.groups;
            c.a.k_zero = c.copies;
            c.a.k_scale = c.copies + a.B * a.Hkv * c.groups * a.D;
            narrow_kernel<<<(unsigned)cdiv(a.B * a.Hkv * c.groups * a.D / 8, 256), 256, 0, st>>>(c);
            VQ_HIP_CHECK_LAUNCH(fn);
        }
        if (c.mma) return a.D == 64 ? launch_choice<64>(fn, c) : a.D == 128 ? launch_choice<128>(fn, c) : launch_choice<256>(fn, c);
        const bool wide = a.D % 4 == 0 && (((uintptr_t)a.k_scale | (uintptr_t)a.k_zero) & 15) == 0;
        if (a.meta_dtype == VQ_F32) wide ? launch_scores<float, true>(c) : launch_scores<float, false>(c);
        else wide ? launch_scores<f16, true>(c) : launch_scores<f16, false>(c);
        VQ_HIP_CHECK_LAUNCH(fn);
        if (c.total > PICK_MOST) {
            block_pick_any_kernel<<<(unsigned)c.items, 256, 0, st>>>(c);
            VQ_HIP_CHECK_LAUNCH(fn);
            return VQ_OK;
        }
    }
    // (without a workspace: every visible block is chosen)
    return launch_pick<true>(fn, c, room.all > 0 ? (size_t)c.total * 4 : 0);
}
