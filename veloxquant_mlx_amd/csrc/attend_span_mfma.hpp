// Attention over spans of slots on the matrix units (gfx950, wave64): one kernel for the shared prefix, for a sequence's own slots
// and for both maps of differential attention.
//
// A block of four waves walks units of 64 slots (32 with heads of 256 channels) of one kv head, two blocks a CU.  A unit's keys and
// values are staged in LDS once for the block.  Plain rows are copied there asynchronously, a unit or more ahead.  Packed slots come as
// words, scales and zeros into a ring of such units, copied ahead, and are reconstructed to fp16 between the products (one packed fused
// multiply-add for two codes: exactly fp16(code * scale + zero)).  A wave holds 32 query rows of one map.  The rows of a block are those of
// all sequences that share the kv head (prefix), or of one sequence (own slots); where they fill half of the waves or less, two waves
// share rows, each with its half of every unit, and add up in LDS at the end.
//
// Bound by what a SIMD's two waves do one after the other.  For a unit of 64 slots and 32 rows, two maps of 128 channels, a wave spends 770
// cycles in 24 products and ~900 in the softmax (32 exponentials of 16 cycles, ~110 other instructions); measured: 2550 cycles a unit while
// the other wave takes 3100, 1.87 GHz, 225 to 233 us for 32 heads over 4096 tokens (900 TFLOP/s of products).  Two blocks a CU, which no barrier
// ties together, overlap one's vector work, copies, start (5000 cycles, integer divisions) and end with the other's products.  What was
// slower: eight waves in one block, 3700 cycles a unit in step at every barrier, 2700 with half of the waves a phase behind the other half, as
// every block then starts and ends alone on its CU; 64 rows a wave, which halves the LDS reads, 268 us to 261; a causal order
// that pairs long tiles with short ones on a CU, 99 us to 96 for heads of 256 channels.
//
// v_mfma_f32_32x32x16 with n = lane % 32, h = lane / 32: A[i = n][k = 8 h + j], B[k = 8 h + j][n], j = 0..7, and
// D[i = 8 (r / 4) + 4 h + r % 4][n] in register r = 0..15.  Scores are formed transposed, S^T = K Q^T: a lane then holds sixteen slots of
// ONE query row, n, so the softmax is lane-local up to the other half's lane, and its registers 8 s .. 8 s + 7 -- slots 16 s +
// {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3} -- are already the B operand of the second product O^T = V^T P^T.  Its A operand takes the
// values of the same slots: from row-major values by transposing LDS reads (ds_read_b64_tr_b16: of each sixteen lanes' four rows of
// sixteen columns, lane i gets column i), from packed ones by storing them transposed in that very order.  Sums, maxima
// and accumulators stay in the lane of their row.
//
// The softmax keeps a reference maximum that follows the true one only where a lane's sum of weights passes 2^15, so accumulators are rescaled
// a few times a run and most units look for no maximum; weights are rounded to the operand type, and their sum is that of the rounded ones.
#pragma once
#include <atomic>
#include <type_traits>

#include "attend_span.hpp"

namespace vq {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int SP_WAVES = 4, SP_THREADS = 64 * SP_WAVES;

// Weights of fp16 are formed as 2^SP_LIFT exp2(s - m), at most SP_MOST: fp16 then tells a weight of 2^-32 of the
// largest from zero (2^-25 without), of which a long context may hold as many as count.  Sums and the weights' sum carry the factor alike.
constexpr float SP_LIFT = 7.f, SP_MOST = 32768.f;

template <typename T> struct SpanMma;
template <> struct SpanMma<f16> {
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ u32 pack(float x, float y) { return as_u(f16x2{(f16)x, (f16)y}); }
    static __device__ __forceinline__ float add_pair(u32 p, float l) {
        return __builtin_amdgcn_fdot2(as_h2(p), f16x2{(f16)1.f, (f16)1.f}, l, false);
    }
};
template <> struct SpanMma<bf16_t> {
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ u32 pack(float x, float y) { return __builtin_bit_cast(u32, bf16x2v{(__bf16)x, (__bf16)y}); }
    static __device__ __forceinline__ float add_pair(u32 p, float l) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, p), bf16x2v{(__bf16)1.f, (__bf16)1.f}, l, false);
    }
};

// 16-byte piece of a row where the tiles keep piece `c` of row `t`: keys so that the 32 rows one score step reads spread over the
// banks, values so that four consecutive rows' 64-byte stretches do
template <int D> __device__ __forceinline__ int sp_kpiece(int t, int c) { return c ^ (t & (D >= 128 ? 15 : 7)); }
template <int D> __device__ __forceinline__ int sp_vpiece(int t, int c) { return c ^ (D >= 128 ? (t & 3) << 2 : (t >> 1 & 1) << 2); }

// Eight codes of a packed word (4 bits: the word; 2 bits: its bytes `first` and `first` + 1) as fp16, in order.  A byte is set in both
// halves of a register and the codes are taken where they stand, adjacent ones one in each half, as the low mantissa bits of a number
// whose unit is the place: bits 0 and up of 1024, bits 2 and up of 256, bits 4 and up of 64, bits 6 and up of 16.
template <int BITS> struct SpanMagic {
    u32 even = vreg_const(BITS == 4 ? 0x54006400u : 0x5C006400u), odd = vreg_const(0x4C005400u);
};
template <int BITS> __device__ __forceinline__ void sp_codes8(u32 w, const SpanMagic<BITS> &magic, u32 (&c)[4], int first = 0) {
    if constexpr (BITS == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32 x = __builtin_amdgcn_perm(0u, w, 0x00010001u * i);
            c[i] = as_u(as_h2((x & 0x00F0000Fu) | magic.even) + f16x2{(f16)-1024.f, (f16)-64.f});
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32 x = __builtin_amdgcn_perm(0u, w, 0x00010001u * (first + i));
            c[2 * i] = as_u(as_h2((x & 0x000C0003u) | magic.even) + f16x2{(f16)-1024.f, (f16)-256.f});
            c[2 * i + 1] = as_u(as_h2((x & 0x00C00030u) | magic.odd) + f16x2{(f16)-64.f, (f16)-16.f});
        }
    }
}
__device__ __forceinline__ u32x4 sp_values8(const u32 (&c)[4], uint4 scale, uint4 zero) {
    const u32 s[4] = {scale.x, scale.y, scale.z, scale.w}, z[4] = {zero.x, zero.y, zero.z, zero.w};
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = as_u(__builtin_elementwise_fma(as_h2(c[i]), as_h2(s[i]), as_h2(z[i])));
    return o;
}

// sixteen bytes a lane from any addresses into LDS at lds + 16 * lane (lds_copy16 with 64-bit addresses)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void span_copy16(const void *from, u32 lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(from), "s"(uniform(lds)) : "memory", "m0");
}
#pragma clang diagnostic pop

// bare three-way maximum (fmaxf canonicalises its operands first); not the first reader of a matrix product, whose result the
// compiler does not wait for on behalf of inline assembly
__device__ __forceinline__ float sp_max3(float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
// a choice between two values (between two places, as `c ? x : y` may become, it would move both to scratch memory)
template <typename T> __device__ __forceinline__ T sp_pick(bool c, T x, T y) { return c ? x : y; }

// bf16 as fp16, two at a time, rounded towards zero: exact in fp16's normal range, magnitudes above 65504 as 65504, below 2^-14 cut to multiples of
// 2^-24 (a product of such a channel is off by 2^-24 of the other factor, where a score's bf16 operands are by 2^-9 of themselves); what is not
// finite stays so.  (Rounded to nearest and clamped it takes twice the instructions, which made the kernel of tiles and few rows 2 % slower.)
__device__ __forceinline__ u32 sp_bf16_to_f16(u32 x) {
    return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u)));
}
__device__ __forceinline__ u32x4 sp_bf16_to_f16(u32x4 x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = sp_bf16_to_f16(x[i]);
    return x;
}
// N adjacent words
template <int N> __device__ __forceinline__ void sp_load_words(const char *p, u32 (&w)[N]) {
    if constexpr (N == 1) {
        w[0] = *(const u32 *)p;
    } else if constexpr (N == 2) {
        const uint2 x = *(const uint2 *)p;
        w[0] = x.x; w[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *(const uint4 *)(p + 4 * i);
            w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
        }
    }
}

template <int BITS, int D> struct SpanTile {
    static constexpr int UNIT = D == 256 ? 32 : 64;      // slots a unit
    static constexpr int HALVES = UNIT / 32;
    static constexpr int VROW = 2 * UNIT + 16;           // bytes of a channel's row of transposed values (144, 80: b128 reads free of conflicts)
    static constexpr int KEYS = UNIT * D * 2;
    static constexpr int VALUES = BITS && D * VROW > KEYS ? D * VROW : KEYS;
    static constexpr int BUF = KEYS + VALUES;
    static constexpr int MOST = 80 * 1024;   // block-shared memory of a block
    static constexpr int ROW_BUF = 2 * KEYS, ROW_BUFS = MOST / ROW_BUF < 4 ? MOST / ROW_BUF : 4;   // tiles of plain rows: one at work, the others under way
    // a packed unit as it lies in memory: key words, value words, key scales and zeros a piece of 32 slots, value scales and
    // zeros a piece of 32 channels
    static constexpr int KWORDS = UNIT * D * BITS / 8, META = UNIT * D / 8;
    static constexpr int RAW = 2 * KWORDS + 2 * META;
    static constexpr int RAWS = BITS ? (MOST - BUF) / RAW < 6 ? (MOST - BUF) / RAW : 6 : 0;   // beside the one tile
    static constexpr int PIECES = RAW / 1024;            // copies of 1 KB, dealt to the waves
    static constexpr int COPIES = (PIECES + SP_WAVES - 1) / SP_WAVES;
    static constexpr int max(int x, int y) { return x > y ? x : y; }
    static constexpr int EXCHANGE = max(SP_WAVES / 2 * (D / 8 * 64 + 64) * 16, SP_WAVES * 32 * (D < 128 ? 4 * D + 16 : 528));   // rows at the end, of half of the waves or by 128 channels
    static constexpr int LDS = max(max(BITS ? BUF + RAWS * RAW : 0, ROW_BUFS * ROW_BUF), EXCHANGE);
    static_assert(LDS <= MOST && ROW_BUFS >= 2 && (BITS == 0 || RAWS >= 3) && RAW % 1024 == 0 && KEYS % (1024 * SP_WAVES) == 0, "tile sizes");
};

// blocks of the prefix, in front of those of the sequences' own slots
__host__ __device__ __forceinline__ int span_shared_blocks(const SpanCall &c) { return c.apart && !c.pfew ? c.psplits * c.ptiles * (int)c.a.Hkv : 0; }

// One block.  WT = 2: two waves share rows, each with its half of every unit.
template <int BITS, typename T, int D, int MAPS, int WT> __device__ __forceinline__ void span_mfma_block(const SpanCall &c, int id) {
    extern __shared__ __align__(16) char lds[];
    using M = SpanMma<T>;
    using Tile = SpanTile<BITS, D>;
    constexpr int UNIT = Tile::UNIT, KS = D / MAPS / 16, DT = D / 32, CH = D / 8;   // channel steps of a score, channel tiles, 16-byte pieces a row
    const vq_store_attend_args &a = c.a;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int Hkv = (int)a.Hkv, G = (int)(a.Hq / a.Hkv), Sq = (int)a.Sq, B = (int)a.B, r1 = G * Sq;
    const int before = (int)span_prefix_slots(a);

    // ---- the block: kv head fastest (blocks of one kv head and run, which read the same slots, lie a multiple of the head count
    // apart), under a causal mask the row tiles that see most first
    const int shared_blocks = span_shared_blocks(c);
    const bool shared = id < shared_blocks;
    int b = 0, split, tile, splits, rows, part;
    const int hkv = shared ? id % Hkv : (id - shared_blocks) % Hkv;
    if (shared) {
        id /= Hkv;
        splits = c.psplits; split = id % splits; tile = id / splits;
        rows = B * r1; part = split;
    } else {
        id = (id - shared_blocks) / Hkv;
        b = id % B; id /= B;
        splits = c.osplits; split = id % splits; tile = c.otiles - 1 - id / splits;
        rows = r1; part = (c.apart ? c.psplits : 0) + split;
    }
    // the waves: one map and 32 rows each
    constexpr int groups = SP_WAVES / MAPS / WT, rt = 32 * groups, X = WT == 2 ? 1 : Tile::HALVES;   // ... and X stretches of 32 slots of a unit
    const int map = MAPS == 2 ? wave & 1 : 0, rest = wave / MAPS, rg = WT == 2 ? rest >> 1 : rest, th = WT == 2 ? rest & 1 : 0;

    // ---- this lane's query row: positions outermost, so that a tile covers few of them
    const int j0 = tile * rt, j = j0 + 32 * rg + n, jc = j < rows ? j : rows - 1;
    const int64_t jb = shared ? jc / r1 : b;
    const int rem = shared ? jc % r1 : jc;
    const int pos = rem / G;
    const int64_t qrow = (jb * a.Hq + hkv * G + rem % G) * Sq + pos;
    const bool wave_works = j0 + 32 * rg < rows;
    int64_t lo64, hi64;
    span_visible(a, before + span_own_live(a, jb), pos, lo64, hi64);
    const int lane_lo = (int)lo64, lane_hi = (int)hi64;
    // slots that every row of the wave sees, that some row of it sees, that some row of the block sees
    int all_lo = lane_lo, all_hi = lane_hi, any_lo = lane_lo, any_hi = lane_hi, blk_lo, blk_hi;
    if (a.seq_lens != nullptr || a.sliding_window > 0 || (a.causal && Sq > 1)) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            const int x = __shfl_xor(all_lo, off), y = __shfl_xor(all_hi, off), u = __shfl_xor(any_lo, off), v = __shfl_xor(any_hi, off);
            all_lo = x > all_lo ? x : all_lo; all_hi = y < all_hi ? y : all_hi;
            any_lo = u < any_lo ? u : any_lo; any_hi = v > any_hi ? v : any_hi;
        }
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo); all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    any_lo = __builtin_amdgcn_readfirstlane(any_lo); any_hi = __builtin_amdgcn_readfirstlane(any_hi);
    const int own_live = (int)span_own_live(a, b);
    if (shared && a.seq_lens != nullptr) { blk_lo = 0; blk_hi = before; }
    else {
        const int last = shared ? rows - 1 : j0 + rt < rows ? j0 + rt - 1 : rows - 1;
        int64_t l, u, x;
        span_visible(a, before + own_live, shared ? 0 : j0 / G, l, x);
        span_visible(a, before + own_live, shared ? Sq - 1 : last / G, x, u);
        blk_lo = (int)l; blk_hi = (int)u;
    }
    blk_lo = __builtin_amdgcn_readfirstlane(blk_lo); blk_hi = __builtin_amdgcn_readfirstlane(blk_hi);

    // ---- the walk: prefix packed, prefix plain, own packed, own plain slots, in units that the block's rows see; this block's run of them
    auto units_seen = [&](int place, int live) __attribute__((always_inline)) {
        const int hi = blk_hi - place, seen = hi < live ? hi : live;
        const int units = (seen + UNIT - 1) / UNIT - (blk_lo > place ? (blk_lo - place) / UNIT : 0);
        return seen > 0 && units > 0 ? units : 0;
    };
    const int np0 = shared || !c.apart ? (int)a.prefix.n_packed : 0, nt0 = shared || !c.apart ? (int)a.prefix.n_tail : 0;
    const int own = shared ? 0 : own_live, np1 = own < (int)a.own.n_packed ? own : (int)a.own.n_packed, nt1 = own - np1;
    const int tail0 = (int)a.prefix.n_packed, tail1 = before + (int)a.own.n_packed;   // places of the plain slots
    const int total = units_seen(0, np0) + units_seen(tail0, nt0) + units_seen(before, np1) + units_seen(tail1, nt1);
    const int run = total / splits, longer = total % splits;   // (the first runs a unit longer)
    const int w0 = split * run + (split < longer ? split : longer), w1 = w0 + run + (split < longer ? 1 : 0);
    if (w0 == w1 && c.nparts > 1) {   // (uniform) nothing: sums are not written
        if (th == 0 && h == 0 && j < rows) *(float2 *)(c.ml + ((qrow * c.nparts + part) * MAPS + map) * 2) = make_float2(-INFINITY, 0.f);
        return;
    }

    // ---- queries as the B operand: row n, channels 16 ks + 8 h .. + 7
    const float c2 = __builtin_fabsf(a.scale) * LOG2E;
    u32x4 q[KS];
    {
        const u16 *src = (const u16 *)a.q + qrow * D + map * (D / MAPS) + 8 * h;
        const u32 sign = a.scale < 0.f ? 0x80008000u : 0u;   // the softmax takes the maximum of the scores themselves
        const bool q_bf16 = a.dtype == VQ_BF16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) q[ks] = *(const u32x4 *)(src + 16 * ks);
        if (BITS != 0 && q_bf16) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) q[ks] = sp_bf16_to_f16(q[ks]);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) q[ks][i] = a.scale == 0.f ? 0u : q[ks][i] ^ sign;
    }
    const float cc = a.scale == 0.f ? 1.f : c2;

    // ---- state of the lane's row
    f32x16 O[DT];
    float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] = 0.f;

    // Where the lane's pieces of the operands lie in a tile: keys of slot n, its piece for channel step ks at key0 ^ 32 ks; row-major values
    // for the transposing reads, channel tile dt at val0 ^ 64 dt; transposed values of channel n.
    const u32 lds0 = lds_addr(lds);
    const u32 key0 = n * D * 2 + sp_kpiece<D>(n, 2 * map * KS + h) * 16;
    u32 val0;
    {
        const int i = lane & 15, t = 4 * h + (i >> 2);
        val0 = t * D * 2 + sp_vpiece<D>(t, 2 * (lane >> 4 & 1) + ((i & 3) >> 1)) * 16 + (i & 1) * 8;
    }
    const u32 col0 = n * Tile::VROW + 16 * h;
    using L4 = __attribute__((address_space(3))) const u32x4;
    using LT = __attribute__((address_space(3))) s16x4;

    f32x16 S[X];
    u32x4 P[X][2];
    // Operands are asked for four products ahead, as written: left to itself the scheduler reads each right before its product and waits.
    constexpr int AHEAD = 4;
    struct Nothing {
        __device__ __forceinline__ void keys(int) {}
        __device__ __forceinline__ void values(int) {}
        __device__ __forceinline__ void all() {}
    };
    // (`aside`: copies of a later unit that are asked for in between, keys' beside the products, values' beside the exponentials)
    auto scores = [&](u32 tile, auto &aside) __attribute__((always_inline)) {
        constexpr int N = X * KS;
        // (the stretches in turn: a product waits 52 cycles for the one it adds to, and takes 32)
        auto key = [&](int i) __attribute__((always_inline)) { return *(L4 *)(uintptr_t)((key0 ^ (32 * (i / X))) + tile + i % X * (32 * D * 2)); };
        u32x4 k[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD && i < N; ++i) k[i] = key(i);
#pragma unroll
        for (int x = 0; x < X; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) S[x][r] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            S[i % X] = M::mma(k[i % AHEAD], q[i / X], S[i % X]);
            if (i + AHEAD < N) k[i % AHEAD] = key(i + AHEAD);
            aside.keys(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto weights = [&](int place, int live, auto &aside) __attribute__((always_inline)) {
        const int end = place + live;
        if (place + 32 * X > (all_hi < end ? all_hi : end) || place < all_lo) {
            const int hi = (lane_hi < end ? lane_hi : end) - place - 4 * h, lo = lane_lo - place - 4 * h;
#pragma unroll
            for (int x = 0; x < X; ++x)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int t = 32 * x + 8 * (r / 4) + r % 4;
                    if (t >= hi || t < lo) S[x][r] = -INFINITY;
                }
        }
        // The weights at the reference maximum as it is.  Only where a lane's sum of them passes what fp16 holds, or a row has no reference yet,
        // the maximum is looked for and they are formed again: a few times a run.
        // (the first reader of the products is the compiler's own, which waits for them: it does not on behalf of inline assembly)
        float l2[2], nm;   // (short chains)
        auto form = [&](auto &aside) __attribute__((always_inline)) {
            nm = m_run == -INFINITY ? 0.f : std::is_same_v<T, f16> ? SP_LIFT - m_run : -m_run;
            l2[0] = l2[1] = 0.f;
#pragma unroll
            for (int x = 0; x < X; ++x)
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const u32 p = M::pack(__builtin_amdgcn_exp2f(__builtin_fmaf(S[x][2 * r], cc, nm)), __builtin_amdgcn_exp2f(__builtin_fmaf(S[x][2 * r + 1], cc, nm)));
                    P[x][r / 4][r % 4] = p;
                    l2[r & 1] = M::add_pair(p, l2[r & 1]);
                    if (r & 1) aside.values(4 * x + r / 2);
                }
        };
        form(aside);
        const bool late = l2[0] + l2[1] > SP_MOST || m_run == -INFINITY;
        if (__any(late)) {   // (for the rows that need it: a row's bits do not depend on the wave's others)
            const int other = __shfl_xor(late ? 1 : 0, 32);   // (by all lanes)
            const bool needed = late || other != 0;
            float mx[X];
#pragma unroll
            for (int x = 0; x < X; ++x) {
                const float m0 = fmaxf(S[x][0], S[x][1]);
                mx[x] = sp_max3(sp_max3(sp_max3(m0, S[x][2], S[x][3]), sp_max3(m0, S[x][4], S[x][5]), sp_max3(m0, S[x][6], S[x][7])), sp_max3(m0, S[x][8], S[x][9]),
                                sp_max3(sp_max3(m0, S[x][10], S[x][11]), sp_max3(m0, S[x][12], S[x][13]), sp_max3(m0, S[x][14], S[x][15])));
            }
            const float most = X == 2 ? fmaxf(mx[0], mx[X - 1]) : mx[0];
            const float top = fmaxf(most, __shfl_xor(most, 32)) * cc, m = needed ? fmaxf(m_run, top) : m_run;
            const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m);
            m_run = m;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) O[dt][r] *= alpha;
            Nothing nothing;
            form(nothing);
        }
        l_run += l2[0] + l2[1];
    };
    auto sums = [&](auto transposed, u32 tile) __attribute__((always_inline)) {
        constexpr int N = 2 * X * DT;
        const u32 values = tile + Tile::KEYS + (transposed.value ? col0 : 0u);
        auto value = [&](int i) __attribute__((always_inline)) {   // of channel tile i % DT, the step's slots 16 (i / DT) .. + 15
            const int s = i / DT, dt = i % DT;
            if constexpr (transposed.value) {
                return *(L4 *)(uintptr_t)(values + dt * (32 * Tile::VROW) + s * 32);
            } else {
                LT *row = (LT *)(uintptr_t)((val0 ^ (64 * dt)) + values);
                const uint2 v0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(row + s * 16 * D / 4));
                const uint2 v1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(row + (s * 16 + 8) * D / 4));
                return u32x4{v0.x, v0.y, v1.x, v1.y};
            }
        };
        u32x4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD && i < N; ++i) v[i] = value(i);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            O[i % DT] = M::mma(v[i % AHEAD], P[i / DT / 2][i / DT % 2], O[i % DT]);
            if (i + AHEAD < N) v[i % AHEAD] = value(i + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // (units that none of the wave's rows sees are left out whole: a unit's stretches are not tested one by one)
    auto compute = [&](auto transposed, u32 tile, int place, int live, auto &&aside) __attribute__((always_inline)) {
        if (!wave_works || place >= any_hi || place + UNIT <= any_lo) {
            aside.all();
            return;
        }
        // (a wave at its products goes before one at its softmax: 1 to 2 % but for few units a block)
        __builtin_amdgcn_s_setprio(1);
        scores(tile + th * (32 * D * 2), aside);
        __builtin_amdgcn_s_setprio(0);
        weights(place + 32 * th, live - 32 * th, aside);
        __builtin_amdgcn_s_setprio(1);
        sums(transposed, tile + (transposed.value ? th * 64 : th * (32 * D * 2)));
        __builtin_amdgcn_s_setprio(0);
    };

    // ---- one span after the other.  A store's fields are read from the argument block where a span begins (`fresh` hides the block's
    // address from the compiler, which would hold all of them in scalar registers from the start and spill those).
    using Args = const __attribute__((address_space(4))) SpanCall;
    using Store = const __attribute__((address_space(4))) vq_kv_store;
    auto fresh = []() __attribute__((always_inline)) {
        Args *p = (Args *)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(p));
        return p;
    };
    // `count` units of plain rows from row t0 on
    auto walk_rows = [&](int which, int t0, int count, int place, int live) __attribute__((always_inline)) {
        Args *args = fresh();
        Store *s = &args->a.prefix + which;
        const int64_t sb = which ? b : 0;
        const int64_t ks = s->k_strides[2] * 2, vs = s->v_strides[2] * 2;
        const char *kb = (const char *)s->k_tail + (sb * s->k_strides[0] + hkv * s->k_strides[1]) * 2 + t0 * ks;
        const char *vb = (const char *)s->v_tail + (sb * s->v_strides[0] + hkv * s->v_strides[1]) * 2 + t0 * vs;
        const bool convert = BITS != 0 && args->a.tail_dtype == VQ_BF16;   // (a unit at a time, not copied ahead)
        constexpr int R = Tile::ROW_BUFS, N = Tile::KEYS / 1024 / SP_WAVES;   // copies a wave for the keys of a unit
        u32 koff[N], voff[N];   // of the lane's pieces, in a whole unit
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int slot = (wave * N + i) * 64 + lane, t = slot / CH, p = slot % CH;
            koff[i] = (u32)t * (u32)ks + sp_kpiece<D>(t, p) * 16;
            voff[i] = (u32)t * (u32)vs + sp_vpiece<D>(t, p) * 16;
        }
        const u32 past = lds0 + R * Tile::ROW_BUF;
        static_assert(X * KS >= N && 4 * X >= N, "as many copies as places to ask for them");
        u32 fill = lds0 + wave * N * 1024;   // where the next unit's copies go
        int asked = 0, asked_live = live;    // that unit
        auto cut_short = [&]() __attribute__((always_inline)) {   // a row past the live ones repeats the last (the pieces' order goes by the tile's row)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                int slot = (wave * N + i) * 64 + lane;
                asm volatile("" : "+v"(slot));   // (not to be worked out ahead, and held, for all units)
                const int t = slot / CH, p = slot % CH;
                const u32 r = (u32)(t < asked_live ? t : asked_live - 1);
                koff[i] = r * (u32)ks + sp_kpiece<D>(t, p) * 16;
                voff[i] = r * (u32)vs + sp_vpiece<D>(t, p) * 16;
            }
        };
        if (asked_live < UNIT) cut_short();
        auto next = [&]() __attribute__((always_inline)) {   // (behind the last unit: that one again, which nobody reads)
            if (asked + 1 < count) {
                kb += UNIT * ks;
                vb += UNIT * vs;
                ++asked;
                asked_live -= UNIT;
                if (asked_live < UNIT) cut_short();
            }
            fill += Tile::ROW_BUF;
            if (fill >= past) fill -= R * Tile::ROW_BUF;
        };
        struct Copies {
            const char *kb, *vb;
            const u32 (&koff)[N], (&voff)[N];
            u32 to;
            __device__ __forceinline__ void keys(int i) const { if (i < N) lds_copy16<0>(kb, koff[i < N ? i : 0], to + i * 1024); }
            __device__ __forceinline__ void values(int i) const { if (i < N) lds_copy16<0>(vb, voff[i < N ? i : 0], to + i * 1024 + Tile::KEYS); }
            __device__ __forceinline__ void all() const {
#pragma unroll
                for (int i = 0; i < N; ++i) { keys(i); values(i); }
            }
        };
#pragma unroll 1
        for (int i = 0; i < R - 1 && !convert; ++i) {
            Copies{kb, vb, koff, voff, fill}.all();
            next();
        }
        u32 tile = lds0;
#pragma unroll 1
        for (int i = 0; i < count; ++i, place += UNIT, live -= UNIT) {
            // the unit is here once the copies of at most R - 2 later ones are under way; past the barrier every wave has left the tile
            // before it, the next to be filled
            wait_copies<(R - 2) * 2 * N>();
            lds_barrier();
            if constexpr (BITS == 0) {
                // (asked for at once behind the barrier, the waves' copies hold each other up for 500 cycles)
                const Copies copies{kb, vb, koff, voff, fill};
                compute(std::false_type{}, tile, place, live, copies);
                next();
            } else {
                if (convert) {   // (a unit at a time)
#pragma unroll 1
                    for (int x = tid; x < UNIT * CH; x += SP_THREADS) {
                        const int t = x / CH, p = x % CH, r = t < live ? t : live - 1;
                        *(u32x4 *)(lds + t * D * 2 + sp_kpiece<D>(t, p) * 16) = sp_bf16_to_f16(*(const u32x4 *)(kb + r * ks + 16 * p));
                        *(u32x4 *)(lds + Tile::KEYS + t * D * 2 + sp_vpiece<D>(t, p) * 16) = sp_bf16_to_f16(*(const u32x4 *)(vb + r * vs + 16 * p));
                    }
                    kb += UNIT * ks;
                    vb += UNIT * vs;
                    lds_barrier();
                } else {
                    Copies{kb, vb, koff, voff, fill}.all();
                    next();
                }
                compute(std::false_type{}, tile, place, live, Nothing{});
            }
            if (!convert) tile += Tile::ROW_BUF;
            if (tile == past) tile = lds0;
        }
        wait_copies<0>();
        lds_barrier();   // the tiles are free
    };
    // `count` units of packed slots from slot t0 on
    auto walk_packed = [&](auto which, int t0, int count, int place, int live) __attribute__((always_inline)) {   // (a template: plain rows have none)
        constexpr int BB = BITS ? BITS : 4, PER = 32 / BB, KW = D / PER, RAWS = Tile::RAWS, N = Tile::COPIES;
        Args *args = fresh();
        Store *s = &args->a.prefix + which;
        const int gshift = __builtin_ctz(args->a.group);
        const int64_t bh = (which ? (int64_t)b : 0) * Hkv + hkv, cap = s->cap_tokens;
        const char *kw = (const char *)s->k_packed + bh * cap * KW * 4, *vw = (const char *)s->v_packed + bh * (cap / PER) * D * 4;
        const char *ks = (const char *)s->k_scale + bh * (cap >> gshift) * D * 2, *kz = (const char *)s->k_zero + bh * (cap >> gshift) * D * 2;
        const char *vs = (const char *)s->v_scale + bh * (D >> gshift) * cap * 2, *vz = (const char *)s->v_zero + bh * (D >> gshift) * cap * 2;
        // The unit as it lies in memory: a piece of 1 KB a copy, the pieces dealt to the waves (as many copies a wave: spare ones repeat the
        // last piece).  What lies past the live slots is not read: a lane whose sixteen bytes would start there repeats the last ones before.
        constexpr int MP = Tile::META / 16, TP = UNIT / 8;   // scales and zeros: [32 slots][which][pieces of channels], then [32 channels][which][pieces of slots]
        auto piece_of = [&](int i) __attribute__((always_inline)) {
            const int p = i * SP_WAVES + wave;
            return p < Tile::PIECES ? p : Tile::PIECES - 1;
        };
        auto lane_at = [&](int i, int n_live) __attribute__((always_inline)) -> const char * {   // in the span's first unit
            const int p = piece_of(i);
            int off = p * 1024 + lane * 16;
            asm volatile("" : "+v"(off));   // (not to be worked out ahead, and held, for all units)
            if (p < Tile::KWORDS / 1024) {
                const int last = n_live * KW * 4 - 16;
                return kw + (off < last ? off : last);
            }
            off -= Tile::KWORDS;
            if (p < 2 * Tile::KWORDS / 1024) {
                const int last = (n_live + PER - 1) / PER * D * 4 - 16;
                return vw + (off < last ? off : last);
            }
            const int x = (off - Tile::KWORDS) / 16, y = x - MP;
            if (x < MP) {
                const int t = 32 * (x / (2 * CH)), tc = t < n_live ? t : n_live - 1;
                return sp_pick((x / CH & 1) != 0, kz, ks) + (tc >> gshift) * D * 2 + x % CH * 16;
            }
            const int t = y % TP * 8, tc = t < n_live ? t : (n_live - 1) / 8 * 8;
            return sp_pick((y / TP & 1) != 0, vz, vs) + ((y / (2 * TP) * 32 >> gshift) * cap + tc) * 2;
        };
        const char *at[N ? N : 1];
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = lane_at(i, UNIT);
        const u32 raw0 = lds0 + Tile::BUF;
        int asked = t0, asked_live = live;
        u32 fill = raw0;
        auto fetch = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int p = piece_of(i);
                const char *from = at[i];
                if (asked_live < UNIT) from = lane_at(i, asked_live);
                if (p < Tile::KWORDS / 1024) from += (int64_t)asked * (KW * 4);
                else if (p < 2 * Tile::KWORDS / 1024) from += (int64_t)(asked / PER) * (D * 4);
                else from += p * 1024 + lane * 16 - 2 * Tile::KWORDS < Tile::META ? (int64_t)(asked >> gshift) * (D * 2) : (int64_t)asked * 2;
                span_copy16(from, fill + p * 1024);
            }
            asked += UNIT;
            asked_live -= UNIT;
            fill += Tile::RAW;
            if (fill == raw0 + RAWS * Tile::RAW) fill = raw0;
        };
        // a unit from the ring into a tile
        const SpanMagic<BB> magic;
        constexpr int KROWS = SP_THREADS / CH;             // slots that the threads cover at a time
        constexpr int VSTEPS = UNIT * D / 16 / SP_THREADS; // sixteen slots each, of a thread's channel
        const char *take = lds + Tile::BUF;
        auto make = [&](int n_live) __attribute__((always_inline)) {
            char *kd = lds, *vd = lds + Tile::KEYS;
            int id = tid;
            asm volatile("" : "+v"(id));   // (addresses are not to be worked out ahead, and held, for all units)
            const int kc = id % CH, kt = id / CH;   // keys: 8-channel piece, slot
            const int vc = id % D, vh = id / D;     // values: channel, which of the unit's stretches
            const uint4 *kmeta = (const uint4 *)(take + 2 * Tile::KWORDS);
            const uint4 *vmeta = (const uint4 *)(take + 2 * Tile::KWORDS + Tile::META);
#pragma unroll
            for (int i = 0; i < UNIT / KROWS; ++i) {
                const int t = kt + KROWS * i;
                const u32 w = ((const u32 *)take)[t * KW + (BB == 4 ? kc : kc / 2)];
                u32 code[4];
                sp_codes8<BB>(BB == 2 ? w >> (16 * (kc & 1)) : w, magic, code);
                *(u32x4 *)(kd + t * D * 2 + sp_kpiece<D>(t, kc) * 16) = sp_values8(code, kmeta[t / 32 * 2 * CH + kc], kmeta[(t / 32 * 2 + 1) * CH + kc]);
                __builtin_amdgcn_sched_barrier(0);
            }
            const u32 *words = (const u32 *)(take + Tile::KWORDS) + vc;
#pragma unroll
            for (int i = 0; i < VSTEPS; ++i) {
                const int step = vh * VSTEPS + i;
                const uint4 *meta = vmeta + vc / 32 * 2 * TP + 2 * step;
                u32x4 x[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {   // eight slots each
                    const u32 w = words[(BB == 4 ? 2 * step + k : step) * D];
                    u32 code[4];
                    sp_codes8<BB>(w, magic, code, 2 * k);
                    x[k] = sp_values8(code, meta[k], meta[TP + k]);
                }
                if (n_live < UNIT) {   // a slot past the live ones may hold anything: its weight is zero, its value has to be finite
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int t = 16 * step + 8 * k + 2 * e;
                            x[k][e] = t >= n_live ? 0u : t + 1 >= n_live ? x[k][e] & 0xFFFFu : x[k][e];
                        }
                }
                u32x4 *dst = (u32x4 *)(vd + vc * Tile::VROW + step * 32);
                dst[0] = u32x4{x[0][0], x[0][1], x[1][0], x[1][1]};
                dst[1] = u32x4{x[0][2], x[0][3], x[1][2], x[1][3]};
                __builtin_amdgcn_sched_barrier(0);
            }
            take += Tile::RAW;
            if (take == lds + Tile::BUF + RAWS * Tile::RAW) take -= RAWS * Tile::RAW;
        };
#pragma unroll 1
        for (int i = 0; i < RAWS && i < count; ++i) fetch();
#pragma unroll 1
        for (int i = 0; i < count; ++i, place += UNIT, live -= UNIT) {
            // unit i is in the ring once at most the RAWS - 1 units behind it are under way; past the barrier every wave has left the tile
            if (i + RAWS <= count) wait_copies<(RAWS - 1) * N>();
            else wait_copies<0>();
            lds_barrier();
            make(live);
            lds_barrier();
            if (i + RAWS < count) fetch();   // into the slot that unit i has left
            compute(std::true_type{}, lds0, place, live, Nothing{});
        }
        lds_barrier();
    };
    {
        int skip = w0, left = w1 - w0;
#pragma unroll 1
        for (int which = 0; which < 2 && left > 0; ++which) {
#pragma unroll
            for (int plain = 0; plain < 2; ++plain) {
                const int at = which ? (plain ? +tail1 : +before) : (plain ? +tail0 : 0), live = which ? (plain ? +nt1 : +np1) : (plain ? +nt0 : +np0);
                const int units = units_seen(at, live);
                const int mine = units - skip < left ? units - skip : left;
                if (mine > 0) {
                    const int t0 = ((blk_lo > at ? (blk_lo - at) / UNIT : 0) + skip) * UNIT;
                    if (plain) walk_rows(which, t0, mine, at + t0, live - t0);
                    else if constexpr (BITS != 0) walk_packed(which, t0, mine, at + t0, live - t0);
                    left -= mine;
                    skip = 0;
                } else {
                    skip -= units;
                }
            }
        }
    }

    // ---- results: the other half's part of the row, then the other map's
    float l = l_run + __shfl_xor(l_run, 32);   // both lanes of a row
    float4 *room = (float4 *)lds + (map * groups + rg) * (D / 8 * 64 + 64) + lane;   // 4 floats a lane and quarter of a channel tile; sum and maximum
    if (WT == 2) {
        lds_barrier();
        if (th == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 4; ++r) room[(4 * dt + r) * 64] = make_float4(O[dt][4 * r], O[dt][4 * r + 1], O[dt][4 * r + 2], O[dt][4 * r + 3]);
            room[DT * 4 * 64] = make_float4(m_run, l, 0.f, 0.f);
        }
        lds_barrier();
        if (th == 0) {
            const float4 ml = room[DT * 4 * 64];
            const float m = fmaxf(m_run, ml.x);
            const float f0 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m), f1 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
            m_run = m;
            l = l * f0 + ml.y * f1;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float4 x = room[(4 * dt + r) * 64];
                    O[dt][4 * r] = O[dt][4 * r] * f0 + x.x * f1;
                    O[dt][4 * r + 1] = O[dt][4 * r + 1] * f0 + x.y * f1;
                    O[dt][4 * r + 2] = O[dt][4 * r + 2] * f0 + x.z * f1;
                    O[dt][4 * r + 3] = O[dt][4 * r + 3] * f0 + x.w * f1;
                }
        }
    }
    // The wave's rows go out through its own room in LDS, where a row of W channels is contiguous: lanes n hold a row each, of which a store
    // would write eight or sixteen bytes (so written, three prompts of 1001 with heads of 256 channels took 95 us, so 50).
    const int first = j0 + 32 * rg;
    auto place_of = [&](auto width, char *mine, int dt, int r) __attribute__((always_inline)) {   // the lane's channels 32 dt + 2 r + 4 h .. + 3
        return (float4 *)(mine + n * (width.value * 4 + 16) + (32 * dt + 2 * r + 4 * h) * 4);
    };
    // put(row, its factor, channel, four values) for every row and channel c0 .. c0 + W - 1
    auto rows_out = [&](auto width, const char *mine, int c0, float factor, auto put) __attribute__((always_inline)) {
        constexpr int LANES = width.value / 4, AT_ONCE = 4;   // of a row
        asm volatile("" ::: "memory");   // (a wave's LDS accesses are in order; these are other lanes')
#pragma unroll 1
        for (int x0 = lane / LANES; x0 < 32; x0 += AT_ONCE * 64 / LANES) {
            int row[AT_ONCE];
            float f[AT_ONCE];
            float4 v[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int x = x0 + i * 64 / LANES;
                row[i] = __shfl((int)qrow, x);   // (fewer than 2^24 rows)
                f[i] = __shfl(factor, x);
                v[i] = *(const float4 *)(mine + x * (width.value * 4 + 16) + lane % LANES * 16);
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i)
                if (first + x0 + i * 64 / LANES < rows) put(row[i], f[i], c0 + lane % LANES * 4, v[i]);
        }
        asm volatile("" ::: "memory");
    };
    constexpr int CB = D < 128 ? D : 128;   // channels at a time, of waves that all have rows to write
    using Block = std::integral_constant<int, CB>;
    auto blocks_out = [&](char *mine, float factor, auto put) __attribute__((always_inline)) {
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += CB) {
#pragma unroll
            for (int dt = 0; dt < CB / 32; ++dt)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x16 &o = O[c0 / 32 + dt];
                    *place_of(Block{}, mine, dt, r) = make_float4(o[r], o[r + 1], o[r + 2], o[r + 3]);
                }
            rows_out(Block{}, mine, c0, factor, put);
        }
    };
    const bool out_bf16 = BITS == 0 ? std::is_same_v<T, bf16_t> : a.dtype == VQ_BF16;
    auto store = [&](int row, int ch, float4 v) __attribute__((always_inline)) {
        *(uint2 *)((u16 *)a.out + (int64_t)row * D + ch) = out_bf16 ? make_uint2(SpanMma<bf16_t>::pack(v.x, v.y), SpanMma<bf16_t>::pack(v.z, v.w))
                                                                   : make_uint2(SpanMma<f16>::pack(v.x, v.y), SpanMma<f16>::pack(v.z, v.w));
    };
    if (WT != 2) lds_barrier();   // (all waves have left the tiles)
    if (c.nparts > 1) {
        if (th == 1) return;
        if (h == 0 && j < rows) *(float2 *)(c.ml + ((qrow * c.nparts + part) * MAPS + map) * 2) = make_float2(m_run, l);
        blocks_out(lds + (WT == 2 ? (map * groups + rg) * (D / 8 * 64 + 64) * 16 : wave * 32 * (CB * 4 + 16)), 1.f,
                   [&](int row, float, int ch, float4 v) __attribute__((always_inline)) {
                       *(float4 *)(c.sums + (((int64_t)row * c.nparts + part) * MAPS + map) * D + ch) = v;
                   });
        return;
    }
    float by = l > 0.f || l != l ? 1.f / l : 0.f;
    if constexpr (MAPS == 1) {
        if (WT == 2) lds_barrier();   // (another wave's room)
        if (th == 1) return;
        blocks_out(lds + rg * 32 * (CB * 4 + 16), by, [&](int row, float f, int ch, float4 v) __attribute__((always_inline)) {
            store(row, ch, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
        });
    } else {
        // the second map's rows, then the difference in their place
        using Row = std::integral_constant<int, D>;
        char *room = lds + rg * (D / 8 * 64 + 64) * 16;
        if (WT == 2) lds_barrier();
        if (map == 1 && th == 0) {
            by *= -span_lam(a, hkv * G + rem % G);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; r += 4) *place_of(Row{}, room, dt, r) = make_float4(O[dt][r] * by, O[dt][r + 1] * by, O[dt][r + 2] * by, O[dt][r + 3] * by);
        }
        lds_barrier();
        if (map == 1 || th == 1) return;
        float sq = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                float4 *at = place_of(Row{}, room, dt, r), x = *at;
                x = make_float4(__builtin_fmaf(O[dt][r], by, x.x), __builtin_fmaf(O[dt][r + 1], by, x.y), __builtin_fmaf(O[dt][r + 2], by, x.z), __builtin_fmaf(O[dt][r + 3], by, x.w));
                sq = __builtin_fmaf(x.x, x.x, sq); sq = __builtin_fmaf(x.y, x.y, sq); sq = __builtin_fmaf(x.z, x.z, sq); sq = __builtin_fmaf(x.w, x.w, sq);
                *at = x;
            }
        }
        float gain = a.gain;
        float4 weight = make_float4(1.f, 1.f, 1.f, 1.f);   // of the lane's channels
        if (a.norm_weight != nullptr) {
            gain /= sqrtf((sq + __shfl_xor(sq, 32)) * (1.f / D) + a.norm_eps);
            const int ch = lane % (D / 4) * 4;
            weight = make_float4(span_ld(a.norm_weight, a.norm_dtype, ch), span_ld(a.norm_weight, a.norm_dtype, ch + 1),
                                 span_ld(a.norm_weight, a.norm_dtype, ch + 2), span_ld(a.norm_weight, a.norm_dtype, ch + 3));
        }
        rows_out(Row{}, room, 0, gain, [&](int row, float f, int ch, float4 v) __attribute__((always_inline)) {
            store(row, ch, make_float4(v.x * f * weight.x, v.y * f * weight.y, v.z * f * weight.z, v.w * f * weight.w));
        });
    }
}

template <int BITS, typename T, int D, int MAPS> __device__ __forceinline__ void span_mfma_block(const SpanCall &c, int id) {
    if (D != 256 && (id < span_shared_blocks(c) ? c.pwt : c.owt) == 2) span_mfma_block<BITS, T, D, MAPS, D == 256 ? 1 : 2>(c, id);
    else span_mfma_block<BITS, T, D, MAPS, 1>(c, id);
}

template <int BITS, typename T, int D, int MAPS>
__global__ __launch_bounds__(SP_THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void span_mfma_kernel(SpanCall c) {
    span_mfma_block<BITS, T, D, MAPS>(c, (int)blockIdx.x);
}

// More than 64 KB of block-shared memory has to be allowed per kernel and device, once (a second setter repeats the same call).
inline int span_allow_lds(const void *kernel, int bytes, std::atomic<bool> *allowed) {
    if (bytes <= 64 * 1024) return VQ_OK;
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (dev >= 0 && dev < 64 && allowed[dev].load(std::memory_order_acquire)) return VQ_OK;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    VQ_REQUIRE(e == hipSuccess, VQ_ERR_HIP, "attention over spans: %d bytes of block-shared memory: %s", bytes, hipGetErrorString(e));
    if (dev >= 0 && dev < 64) allowed[dev].store(true, std::memory_order_release);
    return VQ_OK;
}

template <int BITS, typename T, int D, int MAPS> int launch_span_mfma_as(const SpanCall &c) {
    constexpr int bytes = SpanTile<BITS, D>::LDS;
    const auto kernel = span_mfma_kernel<BITS, T, D, MAPS>;
    static std::atomic<bool> allowed[64] = {};
    if (int rc = span_allow_lds((const void *)kernel, bytes, allowed)) return rc;
    const int64_t blocks = (c.apart && !c.pfew ? (int64_t)c.psplits * c.ptiles * c.a.Hkv : 0) + (c.ofew ? 0 : c.a.B * c.a.Hkv * c.otiles * c.osplits);
    if (blocks == 0) return VQ_OK;
    VQ_REQUIRE(blocks < (INT64_C(1) << 23), VQ_ERR_UNSUPPORTED, "attention over spans: too many sequences and heads for one launch");
    kernel<<<(unsigned)blocks, SP_THREADS, bytes, (hipStream_t)c.a.stream>>>(c);
    VQ_HIP_CHECK_LAUNCH("attention over spans");
    return VQ_OK;
}

// one translation unit each
int launch_span_rows_f16(const SpanCall &c, int maps);
int launch_span_rows_bf16(const SpanCall &c, int maps);
int launch_span_packed2(const SpanCall &c, int maps);
int launch_span_packed4(const SpanCall &c, int maps);

#define VQ_SPAN_LAUNCHER(NAME, BITS, T)                                                                                  \
    namespace vq {                                                                                                      \
    int NAME(const SpanCall &c, int maps) {                                                                             \
        switch (c.a.D * 4 + maps) {                                                                                     \
            case 64 * 4 + 1: return launch_span_mfma_as<BITS, T, 64, 1>(c);                                             \
            case 128 * 4 + 1: return launch_span_mfma_as<BITS, T, 128, 1>(c);                                           \
            case 256 * 4 + 1: return launch_span_mfma_as<BITS, T, 256, 1>(c);                                           \
            case 64 * 4 + 2: return launch_span_mfma_as<BITS, T, 64, 2>(c);                                             \
            case 128 * 4 + 2: return launch_span_mfma_as<BITS, T, 128, 2>(c);                                           \
            default: return launch_span_mfma_as<BITS, T, 256, 2>(c);                                                    \
        }                                                                                                               \
    }                                                                                                                   \
    }

}  // namespace vq
