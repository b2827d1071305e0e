// Attention over spans of packed slots for few query rows: tiles of up to 32 rows of one kv head, or 16 with two maps (gfx950, wave64).
//
// Bound by the bytes of the slots and by reconstructing them, so no wave waits for another: every wave walks its own units of 32 slots,
// every WAVES-th of the block's run, from its own ring in LDS that asynchronous copies fill RING - 1 units ahead, and reconstructs
// them straight into operands of v_mfma_f32_32x32x16_f16 (layout in attend_span_mfma.hpp: lane n = lane % 32, h = lane / 32).  A product sums
// over its k-slots in any order, so each lane takes what it can read in one piece:
//
//   keys    lane (n, h) of S^T = K Q^T owns half h of slot n's channels, sixteen bytes of words at a time; step ks takes channels
//           8 (h D/16 + ks) .. + 7.  With two maps half h is map h's: rows 0 - 15 carry the first map's queries and zeros in the
//           other half, rows 16 - 31 the second's, and one pass of products and one softmax serve both.
//   values  tile dt of O^T = V^T P^T takes channels (D/32) n + dt, so that lane n's words of one word row are adjacent; of the words of
//           sixteen slots lane half h needs the slots that its scores hold, 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3.
//
// Plain rows are copied into the same room, a unit of 32 slots a wave; keys are read as above, values row by row and transposed between
// registers.  At the end the waves' rows are added up in LDS, each wave's room holding its accumulators.
#pragma once
#include "attend_span_mfma.hpp"

namespace vq {

// Four waves a block, two blocks a CU (one with heads of 256 channels).  Eight waves for rows of few slots, which they walk without parts.
template <int BITS, int D, int WAVES_> struct SpanFew {
    static constexpr int WAVES = WAVES_, THREADS = 64 * WAVES, UNIT = 32;
    static constexpr int PER = 32 / BITS, KROW = D * BITS / 8, WORDS = UNIT * KROW;   // bytes of a slot's key words, of a unit's key (value) words
    static constexpr int META = 4 * D;                     // bytes of a unit's key (value) scales and zeros
    static constexpr int RAW = 2 * WORDS + 2 * META;
    static constexpr int ROOM = UNIT * D * 4;              // a wave's: plain keys and values of a unit, or its accumulators
    static constexpr int RING = ROOM / RAW;
    static constexpr int PIECES = (RAW + 1023) / 1024;     // copies of 1 KB (the last one partly, with heads of 64 channels)
    static constexpr int LDS = WAVES * ROOM + WAVES * 32 * 8;
    static_assert(RING >= 3 && LDS <= 160 * 1024, "room for a unit at work and two under way");
};

template <int BITS, int D, int MAPS, int WAVES> __device__ __forceinline__ void span_few_block(const SpanCall &c, int id) {
    extern __shared__ __align__(16) char lds[];
    using F = SpanFew<BITS, D, WAVES>;
    using M = SpanMma<f16>;
    constexpr int KS = D / 16, DT = D / 32, CH = D / 8, UNIT = F::UNIT, PER = F::PER;
    const vq_store_attend_args &a = c.a;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int Hkv = (int)a.Hkv, G = (int)(a.Hq / a.Hkv), Sq = (int)a.Sq, r1 = G * Sq;
    const int before = (int)span_prefix_slots(a);

    // ---- the block: the prefix under the rows of all sequences, or a sequence's slots under its rows; kv head fastest
    const int shared_blocks = c.apart && c.pfew ? c.psplits * c.ptiles * Hkv : 0;
    const bool shared = id < shared_blocks;
    if (!shared) id -= shared_blocks;
    const int hkv = id % Hkv;
    id /= Hkv;
    const int b = shared ? 0 : id % (int)a.B;
    if (!shared) id /= (int)a.B;
    const int splits = shared ? c.psplits : c.osplits, split = id % splits, part = shared || !c.apart ? split : c.psplits + split;
    const int rows = shared ? (int)a.B * r1 : r1;

    // ---- this lane's query row: positions outermost
    constexpr int ROWS = 32 / MAPS;
    const int j0 = id / splits * ROWS, here = rows - j0 < ROWS ? rows - j0 : ROWS;   // the block's tile of rows
    const int map = MAPS == 2 ? n >> 4 : 0, j = n % ROWS, jc = j < here ? j : here - 1;
    auto row_of = [&](int x, int &jb, int &pos) __attribute__((always_inline)) {   // flattened [B, Hq, Sq] row of tile row x
        x += j0;
        const int rem = shared ? x % r1 : x;
        jb = shared ? x / r1 : b;
        pos = rem / G;
        return ((int64_t)jb * a.Hq + hkv * G + rem % G) * Sq + pos;
    };
    int jb, pos;
    const int64_t qrow = row_of(jc, jb, pos);
    int64_t lo64, hi64;
    span_visible(a, before + span_own_live(a, jb), pos, lo64, hi64);
    const int lane_lo = (int)lo64, lane_hi = (int)hi64;
    int all_lo = lane_lo, all_hi = lane_hi, any_lo = lane_lo, any_hi = lane_hi;   // slots that every row sees, that some row sees
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

    // ---- the walk, in units that some row sees; this block's run of them
    auto units_seen = [&](int place, int live) __attribute__((always_inline)) {
        const int hi = any_hi - place, seen = hi < live ? hi : live;
        const int units = (seen + UNIT - 1) / UNIT - (any_lo > place ? (any_lo - place) / UNIT : 0);
        return seen > 0 && units > 0 ? units : 0;
    };
    const int np0 = shared || !c.apart ? (int)a.prefix.n_packed : 0, nt0 = shared || !c.apart ? (int)a.prefix.n_tail : 0;
    const int own = shared ? 0 : own_live, np1 = own < (int)a.own.n_packed ? own : (int)a.own.n_packed, nt1 = own - np1;
    const int tail0 = (int)a.prefix.n_packed, tail1 = before + (int)a.own.n_packed;
    const int total = units_seen(0, np0) + units_seen(tail0, nt0) + units_seen(before, np1) + units_seen(tail1, nt1);
    const int run = total / splits, longer = total % splits;   // (the first runs a unit longer)
    const int w0 = split * run + (split < longer ? split : longer), w1 = w0 + run + (split < longer ? 1 : 0);
    if (w0 == w1 && c.nparts > 1) {   // (uniform) nothing: sums are not written
        if (tid < here * MAPS) {
            int x, y;
            *(float2 *)(c.ml + ((row_of(tid / MAPS, x, y) * c.nparts + part) * MAPS + tid % MAPS) * 2) = make_float2(-INFINITY, 0.f);
        }
        return;
    }

    // ---- queries as the B operand of the scores
    u32x4 q[KS];
    {
        const u16 *src = (const u16 *)a.q + qrow * D + h * (D / 2);
        const u32 sign = a.scale < 0.f ? 0x80008000u : 0u;   // the softmax takes the maximum of the scores themselves
        const bool q_bf16 = a.dtype == VQ_BF16, mine = a.scale != 0.f && (MAPS == 1 || map == h);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) q[ks] = *(const u32x4 *)(src + 8 * ks);
        if (q_bf16) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) q[ks] = sp_bf16_to_f16(q[ks]);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) q[ks][i] = mine ? q[ks][i] ^ sign : 0u;
    }
    const float cc = a.scale == 0.f ? 1.f : __builtin_fabsf(a.scale) * LOG2E;

    f32x16 O[DT];
    float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] = 0.f;

    // weights of a unit's scores, P[s] the B operand of the second product for slots 16 s .. 16 s + 15
    auto softmax = [&](f32x16 &S, int place, int live, u32x4 (&P)[2]) __attribute__((always_inline)) {
        const int end = place + live;
        if (place + UNIT > (all_hi < end ? all_hi : end) || place < all_lo) {
            const int hi = (lane_hi < end ? lane_hi : end) - place - 4 * h, lo = lane_lo - place - 4 * h;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int t = 8 * (r / 4) + r % 4;
                if (t >= hi || t < lo) S[r] = -INFINITY;
            }
        }
        // (as in attend_span_mfma.hpp: the maximum only where the weights' sum asks for it)
        float l2[2], nm;
        auto form = [&]() __attribute__((always_inline)) {
            nm = m_run == -INFINITY ? 0.f : SP_LIFT - m_run;
            l2[0] = l2[1] = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const u32 p = M::pack(__builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * r], cc, nm)), __builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * r + 1], cc, nm)));
                P[r / 4][r % 4] = p;
                l2[r & 1] = M::add_pair(p, l2[r & 1]);
            }
        };
        form();
        const bool late = l2[0] + l2[1] > SP_MOST || m_run == -INFINITY;
        if (__any(late)) {
            const int other = __shfl_xor(late ? 1 : 0, 32);   // (by all lanes)
            const bool needed = late || other != 0;
            float mx = fmaxf(S[0], S[1]);
#pragma unroll
            for (int r = 2; r < 16; r += 2) mx = sp_max3(mx, S[r], S[r + 1]);
            const float top = fmaxf(mx, __shfl_xor(mx, 32)) * cc, m = needed ? fmaxf(m_run, top) : m_run;
            const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m);
            m_run = m;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) O[dt][r] *= alpha;
            form();
        }
        l_run += l2[0] + l2[1];
    };

    const u32 room = lds_addr(lds) + wave * F::ROOM;   // this wave's
    const char *room_p = lds + wave * F::ROOM;
    using Args = const __attribute__((address_space(4))) SpanCall;
    using Store = const __attribute__((address_space(4))) vq_kv_store;
    auto fresh = []() __attribute__((always_inline)) {   // (see attend_span_mfma.hpp)
        Args *p = (Args *)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(p));
        return p;
    };

    // `count` units of packed slots, every WAVES-th from slot t0 on
    auto walk_packed = [&](int which, int t0, int count, int place, int live) __attribute__((always_inline)) {
        constexpr int STEP = UNIT * F::WAVES, N = F::PIECES, RING = F::RING;
        Args *args = fresh();
        Store *s = &args->a.prefix + which;
        const int gshift = __builtin_ctz(args->a.group);
        const int64_t bh = (which ? (int64_t)b : 0) * Hkv + hkv, cap = s->cap_tokens;
        const char *kw = (const char *)s->k_packed + bh * cap * F::KROW, *vw = (const char *)s->v_packed + bh * (cap / PER) * D * 4;
        const char *ks = (const char *)s->k_scale + bh * (cap >> gshift) * D * 2, *kz = (const char *)s->k_zero + bh * (cap >> gshift) * D * 2;
        const char *vs = (const char *)s->v_scale + bh * (D >> gshift) * cap * 2, *vz = (const char *)s->v_zero + bh * (D >> gshift) * cap * 2;
        // Copies of a unit: key words, slot t's sixteen-byte pieces rotated so that the lanes that read them spread over the banks; value words
        // as they lie; [scale, zero][channels] of its key group; [scale, zero][32 channels][slots] of its values.  What lies past
        // the live slots is not read: the last live one's is, again.
        constexpr int C = F::KROW / 16;   // pieces of a slot's key words (of 1, 2, 4 or 8)
        auto kpiece = [&](int t, int p) __attribute__((always_inline)) { return C == 1 ? 0 : p ^ (t / (8 / C) & (C - 1)); };
        auto lane_at = [&](int i, int n_live) __attribute__((always_inline)) -> const char * {   // in the span's first unit
            int off = i * 1024 + lane * 16;
            if (off >= F::RAW) off = F::RAW - 16;   // (lanes that are left over)
            if (i * 1024 < F::WORDS && (F::WORDS % 1024 == 0 || off < F::WORDS)) {
                const int t = off / F::KROW, p = off % F::KROW / 16;
                return kw + (t < n_live ? t : n_live - 1) * F::KROW + kpiece(t, p) * 16;
            }
            off -= F::WORDS;
            if (off < F::WORDS) {
                const int last = (n_live + PER - 1) / PER * D * 4 - 16;
                return vw + (off < last ? off : last);
            }
            off -= F::WORDS;
            if (off < F::META) return sp_pick(off >= F::META / 2, kz, ks) + off % (F::META / 2);
            off -= F::META;
            const int y = off % (F::META / 2), c32 = y / 64, t = y % 64 / 2, tc = t < n_live ? t : (n_live - 1) / 8 * 8;
            return sp_pick(off >= F::META / 2, vz, vs) + ((c32 * 32 >> gshift) * cap + tc) * 2;
        };
        const char *at[N];
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = lane_at(i, UNIT);
        int asked = t0, asked_live = live;
        u32 fill = room;
        auto fetch = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const char *from = at[i];
                if (asked_live < UNIT) from = lane_at(i, asked_live);
                const int off = i * 1024 + lane * 16;
                const int64_t key = (int64_t)asked * F::KROW, value = (int64_t)(asked / PER) * (D * 4), kmeta = (int64_t)(asked >> gshift) * (D * 2),
                              vmeta = (int64_t)asked * 2;
                from += off < F::WORDS ? key : off < 2 * F::WORDS ? value : off < 2 * F::WORDS + F::META ? kmeta : vmeta;
                if (i * 1024 + 1024 <= F::RAW || lane * 16 < F::RAW - i * 1024) span_copy16(from, fill + i * 1024);
            }
            asked += STEP;
            asked_live -= STEP;
            fill += F::RAW;
            if (fill == room + RING * F::RAW) fill = room;
        };
        const SpanMagic<BITS> magic;
        const char *take = room_p;
        auto step = [&]() __attribute__((always_inline)) {
            // scores
            f32x16 S;
#pragma unroll
            for (int r = 0; r < 16; ++r) S[r] = 0.f;
            const uint4 *kmeta = (const uint4 *)(take + 2 * F::WORDS) + h * (CH / 2);
            constexpr int KP = KS * BITS / 16 > 0 ? KS * BITS / 16 : 1;   // sixteen-byte pieces of a lane's half of the key words
#pragma unroll
            for (int p = 0; p < KP; ++p) {
                u32 w[4];
                if constexpr (F::KROW == 16) {   // (heads of 64 channels at 2 bits: half a piece)
                    const uint2 x = *(const uint2 *)(take + n * 16 + h * 8);
                    w[0] = x.x; w[1] = x.y; w[2] = w[3] = 0u;
                } else {
                    const uint4 x = *(const uint4 *)(take + n * F::KROW + kpiece(n, h * KP + p) * 16);
                    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
                }
                constexpr int PERP = KS / KP;   // steps that a piece holds
#pragma unroll
                for (int e = 0; e < PERP; ++e) {
                    const int k = p * PERP + e;
                    u32 code[4];
                    sp_codes8<BITS>(BITS == 4 ? w[e % 4] : w[e / 2], magic, code, 2 * (e & 1));
                    S = M::mma(sp_values8(code, kmeta[k], kmeta[CH + k]), q[k], S);
                }
            }
            // (the values' words are asked for ahead of the softmax)
            const char *vw_p = take + F::WORDS;
            u32 lo[2][DT], hi[2][DT];   // of sixteen slots (4 bits: of eight each)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                sp_load_words<DT>(vw_p + ((BITS == 4 ? 2 * s : s) * D + DT * n) * 4, lo[s]);
                if constexpr (BITS == 4) sp_load_words<DT>(vw_p + ((2 * s + 1) * D + DT * n) * 4, hi[s]);
            }
            __builtin_amdgcn_sched_barrier(0);
            u32x4 P[2];
            softmax(S, place, live, P);
            // sums: channels DT n + dt
            const char *vmeta = take + 2 * F::WORDS + F::META + (DT * n / 32) * 64 + 8 * h;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                // scales and zeros of slots 16 s + 4 h .. + 3 and 16 s + 8 + 4 h .. + 3
                const uint2 s0 = *(const uint2 *)(vmeta + 32 * s), s1 = *(const uint2 *)(vmeta + 32 * s + 16);
                const uint2 z0 = *(const uint2 *)(vmeta + F::META / 2 + 32 * s), z1 = *(const uint2 *)(vmeta + F::META / 2 + 32 * s + 16);
                uint4 sc = make_uint4(s0.x, s0.y, s1.x, s1.y), ze = make_uint4(z0.x, z0.y, z1.x, z1.y);
                if (live < UNIT) {   // a slot past the live ones may hold anything: its weight is zero, its value has to be finite
                    u32 m[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = 16 * s + 4 * h + 2 * (e & 1) + 8 * (e >> 1);
                        m[e] = t >= live ? 0u : t + 1 >= live ? 0xFFFFu : ~0u;
                    }
                    sc = make_uint4(sc.x & m[0], sc.y & m[1], sc.z & m[2], sc.w & m[3]);
                    ze = make_uint4(ze.x & m[0], ze.y & m[1], ze.z & m[2], ze.w & m[3]);
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    // 4 bits: this half's sixteen bits of either word; 2 bits: bytes h and 2 + h of the one
                    const u32 w = BITS == 4 ? __builtin_amdgcn_perm(hi[s][dt], lo[s][dt], h ? 0x07060302u : 0x05040100u)
                                            : __builtin_amdgcn_perm(0u, lo[s][dt], h ? 0x0C0C0301u : 0x0C0C0200u);
                    u32 code[4];
                    sp_codes8<BITS>(w, magic, code);
                    const u32x4 v = sp_values8(code, sc, ze);
                    O[dt] = M::mma(v, P[s], O[dt]);
                }
            }
            take += F::RAW;
            if (take == room_p + RING * F::RAW) take = room_p;
        };
#pragma unroll 1
        for (int i = 0; i < RING - 1 && i < count; ++i) fetch();
#pragma unroll 1
        for (int i = 0; i < count; ++i, place += STEP, live -= STEP) {
            // this unit is here once at most the later ones' copies are under way; the slot that the unit before it has left is filled
            if (i + RING - 1 <= count) wait_copies<(RING - 2) * N>();
            else wait_copies<0>();
            if (i + RING - 1 < count) fetch();
            step();
            // (the slot's reads are over before a copy may land in it)
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    };
    // `count` units of plain rows likewise
    auto walk_rows = [&](int which, int t0, int count, int place, int live) __attribute__((always_inline)) {
        constexpr int STEP = UNIT * F::WAVES, VT = UNIT * D * 2;   // the values' place in the room
        Args *args = fresh();
        Store *s = &args->a.prefix + which;
        const int64_t sb = which ? b : 0, kst = s->k_strides[2] * 2, vst = s->v_strides[2] * 2;
        const bool bf16 = args->a.tail_dtype == VQ_BF16;
        const char *kb = (const char *)s->k_tail + (sb * s->k_strides[0] + hkv * s->k_strides[1]) * 2 + t0 * kst;
        const char *vb = (const char *)s->v_tail + (sb * s->v_strides[0] + hkv * s->v_strides[1]) * 2 + t0 * vst;
#pragma unroll 1
        for (int i = 0; i < count; ++i, kb += STEP * kst, vb += STEP * vst, place += STEP, live -= STEP) {
#pragma unroll 1
            for (int x = 0; x < UNIT * CH / 64; ++x) {   // a row past the live ones repeats the last
                const int slot = x * 64 + lane, t = slot / CH, p = slot % CH, r = t < live ? t : live - 1;
                lds_copy16<0>(kb, (u32)r * (u32)kst + sp_kpiece<D>(t, p) * 16, room + x * 1024);
                lds_copy16<0>(vb, (u32)r * (u32)vst + p * 16, room + VT + x * 1024);
            }
            wait_copies<0>();
            if (bf16) {   // in place, the lane's own pieces
                u32x4 *piece = (u32x4 *)(lds + wave * F::ROOM) + lane;
#pragma unroll 1
                for (int x = 0; x < UNIT * CH / 32; ++x) piece[x * 64] = sp_bf16_to_f16(piece[x * 64]);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
            f32x16 S;
#pragma unroll
            for (int r = 0; r < 16; ++r) S[r] = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k) S = M::mma(*(const u32x4 *)(room_p + n * D * 2 + sp_kpiece<D>(n, h * KS + k) * 16), q[k], S);
            u32x4 P[2];
            softmax(S, place, live, P);
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                // eight slots' DT channels of this lane, then a pair of slots a register
                u32 x[8][DT / 2];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int t = 16 * s2 + 4 * h + (e & 3) + 8 * (e >> 2);
                    sp_load_words<DT / 2>(room_p + VT + t * D * 2 + n * DT * 2, x[e]);
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    u32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = dt & 1 ? pair_hi(x[2 * e][dt / 2], x[2 * e + 1][dt / 2]) : pair_lo(x[2 * e][dt / 2], x[2 * e + 1][dt / 2]);
                    O[dt] = M::mma(v, P[s2], O[dt]);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the room's reads are over)
        }
    };
    {
        int skip = w0, left = w1 - w0, turn = wave;   // the wave's first unit of what is left
#pragma unroll 1
        for (int which = 0; which < 2 && left > 0; ++which) {
#pragma unroll
            for (int plain = 0; plain < 2; ++plain) {
                const int at = which ? (plain ? +tail1 : +before) : (plain ? +tail0 : 0), live = which ? (plain ? +nt1 : +np1) : (plain ? +nt0 : +np0);
                const int units = units_seen(at, live);
                const int run = units - skip < left ? units - skip : left;
                if (run > 0) {
                    const int mine = turn < run ? (run - turn + F::WAVES - 1) / F::WAVES : 0;
                    const int t0 = ((any_lo > at ? (any_lo - at) / UNIT : 0) + skip + turn) * UNIT;
                    if (mine > 0) {
                        if (plain) walk_rows(which, t0, mine, at + t0, live - t0);
                        else walk_packed(which, t0, mine, at + t0, live - t0);
                    }
                    turn = (turn - run % F::WAVES + F::WAVES) % F::WAVES;
                    left -= run;
                    skip = 0;
                } else {
                    skip -= units;
                }
            }
        }
    }

    // ---- the waves' rows: row x's channels DT m .. DT m + DT - 1 of a wave at place m ^ x of its room
    const float l = l_run + __shfl_xor(l_run, 32);   // both lanes of a row
    float2 *mls = (float2 *)(lds + F::WAVES * F::ROOM);
    lds_barrier();
    {
        float *mine = (float *)(lds + wave * F::ROOM) + n * D;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int m = 8 * (r / 4) + 4 * h + r % 4;
            float *dst = mine + (m ^ n) * DT;
#pragma unroll
            for (int dt = 0; dt < DT; dt += 2) *(float2 *)(dst + dt) = make_float2(O[dt][r], O[dt + 1][r]);
        }
        if (h == 0) mls[wave * 32 + n] = make_float2(m_run, l);
    }
    lds_barrier();
    const int ch = tid & 31;
#pragma unroll 1
    for (int x = tid >> 5; x < here; x += F::THREADS / 32) {
        int jb2, pos2;
        const int64_t row = row_of(x, jb2, pos2);
        float o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = 0.f;
#pragma unroll
        for (int w = 0; w < MAPS; ++w) {
            const int y = x + 16 * w;
            float m = -INFINITY, den = 0.f, num[DT];
#pragma unroll
            for (int v = 0; v < F::WAVES; ++v) m = fmaxf(m, mls[v * 32 + y].x);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) num[dt] = 0.f;
#pragma unroll
            for (int v = 0; v < F::WAVES; ++v) {
                const float2 ml = mls[v * 32 + y];
                const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - m);
                den = __builtin_fmaf(f, ml.y, den);
                const float *src = (const float *)(lds + v * F::ROOM) + y * D + (ch ^ y) * DT;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) num[dt] = __builtin_fmaf(f, src[dt], num[dt]);
            }
            if (c.nparts > 1) {
                const int64_t rec = (row * c.nparts + part) * MAPS + w;
                if (ch == 0) *(float2 *)(c.ml + rec * 2) = make_float2(m, den);
                float *dst = c.sums + rec * D + ch * DT;
#pragma unroll
                for (int dt = 0; dt < DT; dt += 2) *(float2 *)(dst + dt) = make_float2(num[dt], num[dt + 1]);
            }
            const float by = den > 0.f || den != den ? (w == 0 ? 1.f : -span_lam(a, hkv * G + (shared ? (j0 + x) % r1 : j0 + x) % G)) / den : 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_fmaf(num[dt], by, o[dt]);
        }
        if (c.nparts > 1) continue;
        if (MAPS == 2) {
            float gain = a.gain;
            if (a.norm_weight != nullptr) {
                float sq = 0.f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) sq = __builtin_fmaf(o[dt], o[dt], sq);
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) sq += __shfl_xor(sq, off);   // the row's 32 lanes
                gain /= sqrtf(sq * (1.f / D) + a.norm_eps);
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= a.norm_weight != nullptr ? gain * span_ld(a.norm_weight, a.norm_dtype, ch * DT + dt) : gain;
        }
        u16 *dst = (u16 *)a.out + row * D + ch * DT;
#pragma unroll
        for (int dt = 0; dt < DT; dt += 2)
            *(u32 *)(dst + dt) = a.dtype == VQ_BF16 ? SpanMma<bf16_t>::pack(o[dt], o[dt + 1]) : SpanMma<f16>::pack(o[dt], o[dt + 1]);
    }
}

template <int BITS, int D, int MAPS, int WAVES>
__global__ __launch_bounds__((64 * WAVES)) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2, D == 256 ? 1 : 2))) void span_few_kernel(SpanCall c) {
    span_few_block<BITS, D, MAPS, WAVES>(c, (int)blockIdx.x);
}

// Blocks of a prefix in tiles and behind them blocks of own slots, which share the CUs with them (128 sequences of 1k slots on a prefix of 32k:
// 184 us in two launches, 161 together; with the kinds in turn a CU held two of one kind, 55 us more than behind each other).
template <int BITS, int D> __global__ __launch_bounds__(SP_THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void span_both_kernel(SpanCall c) {
    const int id = (int)blockIdx.x, tiles = span_shared_blocks(c);
    if (id < tiles) span_mfma_block<BITS, f16, D, 1>(c, id);
    else span_few_block<BITS, D, 1, 4>(c, id - tiles);
}

template <int BITS, int D> int launch_span_both_as(const SpanCall &c) {
    constexpr int bytes = SpanTile<BITS, D>::LDS > SpanFew<BITS, D, 4>::LDS ? SpanTile<BITS, D>::LDS : SpanFew<BITS, D, 4>::LDS;
    const auto kernel = span_both_kernel<BITS, D>;
    static std::atomic<bool> allowed[64] = {};
    if (int rc = span_allow_lds((const void *)kernel, bytes, allowed)) return rc;
    const int64_t tiles = (int64_t)c.psplits * c.ptiles * c.a.Hkv, few = c.a.B * c.a.Hkv * c.osplits * c.otiles, blocks = tiles + few;
    VQ_REQUIRE(blocks < (INT64_C(1) << 23), VQ_ERR_UNSUPPORTED, "attention over spans: too many sequences and heads for one launch");
    kernel<<<(unsigned)blocks, SP_THREADS, bytes, (hipStream_t)c.a.stream>>>(c);
    VQ_HIP_CHECK_LAUNCH("attention over spans");
    return VQ_OK;
}

template <int BITS, int D, int MAPS, int WAVES> int launch_span_few_of(const SpanCall &c) {
    constexpr int bytes = SpanFew<BITS, D, WAVES>::LDS;
    const auto kernel = span_few_kernel<BITS, D, MAPS, WAVES>;
    static std::atomic<bool> allowed[64] = {};
    if (int rc = span_allow_lds((const void *)kernel, bytes, allowed)) return rc;
    const int64_t blocks = (c.apart && c.pfew ? (int64_t)c.psplits * c.ptiles * c.a.Hkv : 0) + (c.ofew ? c.a.B * c.a.Hkv * c.osplits * c.otiles : 0);
    if (blocks == 0) return VQ_OK;
    VQ_REQUIRE(blocks < (INT64_C(1) << 23), VQ_ERR_UNSUPPORTED, "attention over spans: too many sequences and heads for one launch");
    kernel<<<(unsigned)blocks, 64 * WAVES, bytes, (hipStream_t)c.a.stream>>>(c);
    VQ_HIP_CHECK_LAUNCH("attention over spans");
    return VQ_OK;
}
template <int BITS, int D, int MAPS> int launch_span_few_as(const SpanCall &c) {
    if constexpr (D != 256) {
        if (c.owaves == 8) return launch_span_few_of<BITS, D, MAPS, 8>(c);
    }
    return launch_span_few_of<BITS, D, MAPS, 4>(c);
}

int launch_span_few2(const SpanCall &c, int maps);
int launch_span_few4(const SpanCall &c, int maps);
int launch_span_both2(const SpanCall &c);
int launch_span_both4(const SpanCall &c);

#define VQ_SPAN_FEW_LAUNCHER(NAME, BITS)                                                                                \
    namespace vq {                                                                                                      \
    int NAME(const SpanCall &c, int maps) {                                                                             \
        switch (c.a.D * 4 + maps) {                                                                                     \
            case 64 * 4 + 1: return launch_span_few_as<BITS, 64, 1>(c);                                                 \
            case 128 * 4 + 1: return launch_span_few_as<BITS, 128, 1>(c);                                               \
            case 256 * 4 + 1: return launch_span_few_as<BITS, 256, 1>(c);                                               \
            case 64 * 4 + 2: return launch_span_few_as<BITS, 64, 2>(c);                                                 \
            case 128 * 4 + 2: return launch_span_few_as<BITS, 128, 2>(c);                                               \
            default: return launch_span_few_as<BITS, 256, 2>(c);                                                        \
        }                                                                                                               \
    }                                                                                                                   \
    }

}  // namespace vq
