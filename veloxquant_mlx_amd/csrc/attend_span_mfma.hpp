// Attention over spans of slots on the matrix units (gfx950, wave64): one kernel for the shared prefix, for a sequence's own slots
// and for both maps of differential attention.
//
// A block of four waves walks units of 64 slots of one kv head.  A unit's keys and values are staged in LDS once for the
// block, double-buffered: plain rows by asynchronous copies, packed slots through registers, reconstructed to fp16 (one packed
// fused multiply-add for two codes: exactly fp16(code * scale + zero)).  Each wave holds 32 query rows; the rows are those of all
// sequences that share the kv head (prefix), or of one sequence (own slots) -- 128 a block, or 64 rows with two waves on
// each 32, one for either half of every unit.
//
// v_mfma_f32_32x32x16 with n = lane % 32, h = lane / 32: A[i = n][k = 8 h + j], B[k = 8 h + j][n], j = 0..7, and
// D[i = 8 (r / 4) + 4 h + r % 4][n] in register r = 0..15.  Scores are formed transposed, S^T = K Q^T: a lane then holds sixteen slots of
// ONE query row, n, so the softmax is lane-local up to the other half's lane, and its registers 8 s .. 8 s + 7 -- slots 16 s +
// {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3} -- are already the B operand of the second product O^T = V^T P^T.  Its A operand takes the
// values of the same slots: from row-major values by transposing LDS reads (ds_read_b64_tr_b16: of each sixteen lanes' four rows of
// sixteen columns, lane i gets column i), from packed ones by storing them transposed in that very order.  Sums, maxima
// and accumulators stay in the lane of their row.
//
// The softmax keeps a reference maximum that follows the true one lazily (within 8 powers of two), so accumulators are rescaled a few
// times a run; weights are rounded to the operand type, and their sum is that of the rounded ones.
#pragma once
#include <atomic>

#include "attend_span.hpp"

namespace vq {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int SP_UNIT = 64;         // slots a unit
constexpr int SP_THREADS = 256;
constexpr int SP_VROW = 2 * SP_UNIT + 16;   // bytes of a channel's row of transposed values (144: conflict-free b128 access)

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

// Eight codes of a packed word (4 bits: the word; 2 bits: its lower half) as fp16, in order.
template <int BITS> __device__ __forceinline__ void sp_codes8(u32 w, u32 magic, u32 (&c)[4]) {
    const u32x4 r = __builtin_bit_cast(u32x4, unpack8<BITS>(w, magic));
    if (BITS == 4) {   // pairs (0,4) (1,5) (2,6) (3,7)
        c[0] = pair_lo(r[0], r[1]); c[1] = pair_lo(r[2], r[3]); c[2] = pair_hi(r[0], r[1]); c[3] = pair_hi(r[2], r[3]);
    } else {           // pairs (0,8) (1,9) (2,10) (3,11), and of the word eight bits on (4,12) ...
        const u32x4 s = __builtin_bit_cast(u32x4, unpack8<BITS>(w >> 8, magic));
        c[0] = pair_lo(r[0], r[1]); c[1] = pair_lo(r[2], r[3]); c[2] = pair_lo(s[0], s[1]); c[3] = pair_lo(s[2], s[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = as_u(as_h2(c[i]) + as_h2(Magic<BITS>::neg_off_pair));
}
__device__ __forceinline__ u32x4 sp_values8(const u32 (&c)[4], uint4 scale, uint4 zero) {
    const u32 s[4] = {scale.x, scale.y, scale.z, scale.w}, z[4] = {zero.x, zero.y, zero.z, zero.w};
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = as_u(__builtin_elementwise_fma(as_h2(c[i]), as_h2(s[i]), as_h2(z[i])));
    return o;
}

template <int BITS, int D> struct SpanTile {
    static constexpr int KEYS = SP_UNIT * D * 2;
    static constexpr int VALUES = BITS && D * SP_VROW > KEYS ? D * SP_VROW : KEYS;
    static constexpr int BUF = KEYS + VALUES;
    static constexpr int LDS = 2 * BUF;
};

template <int BITS, typename T, int D, int MAPS>
__global__ __launch_bounds__(SP_THREADS) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2, D == 256 ? 1 : 2)))
void span_mfma_kernel(SpanCall c) {
    extern __shared__ __align__(16) char lds[];
    using M = SpanMma<T>;
    using Tile = SpanTile<BITS, D>;
    constexpr int KS = D / MAPS / 16, DT = D / 32, CH = D / 8;   // channel steps of a score, channel tiles, 16-byte pieces a row
    const vq_store_attend_args &a = c.a;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int Hkv = (int)a.Hkv, G = (int)(a.Hq / a.Hkv), Sq = (int)a.Sq, B = (int)a.B, r1 = G * Sq;
    const int before = (int)span_prefix_slots(a);

    // ---- the block: kv head fastest (blocks of one kv head and run, which read the same slots, lie a multiple of the head count
    // apart), under a causal mask the row tiles that see most first
    int id = (int)blockIdx.x;
    const int shared_blocks = c.apart ? c.psplits * c.ptiles * Hkv : 0;
    const bool shared = id < shared_blocks;
    int b = 0, split, tile, splits, wt, rows, part;
    const int hkv = shared ? id % Hkv : (id - shared_blocks) % Hkv;
    if (shared) {
        id /= Hkv;
        splits = c.psplits; split = id % splits; tile = id / splits;
        wt = c.pwt; rows = B * r1; part = split * wt;
    } else {
        id = (id - shared_blocks) / Hkv;
        b = id % B; id /= B;
        splits = c.osplits; split = id % splits; tile = c.otiles - 1 - id / splits;
        wt = c.owt; rows = r1; part = (c.apart ? c.psplits * c.pwt : 0) + split * wt;
    }
    // the waves: one map each, 32 rows each; the waves that are left over share rows, each with its half of every unit
    const int map = MAPS == 2 ? wave & 1 : 0, rest = MAPS == 2 ? wave >> 1 : wave, groups = 4 / MAPS / wt;
    const int rt = 32 * groups, rg = rest % groups, th = rest / groups;
    part += th;

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

    // ---- the spans: live slots, place of the first, units that the block's rows see
    const bool with_prefix = shared || !c.apart, with_own = !shared;
    int live[4], at[4], first[4], end[4], total = 0;
    live[0] = with_prefix ? (int)a.prefix.n_packed : 0;
    live[1] = with_prefix ? (int)a.prefix.n_tail : 0;
    live[2] = with_own ? (own_live < (int)a.own.n_packed ? own_live : (int)a.own.n_packed) : 0;
    live[3] = with_own ? own_live - live[2] : 0;
    at[0] = 0; at[1] = (int)a.prefix.n_packed; at[2] = before; at[3] = before + (int)a.own.n_packed;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int hi = blk_hi - at[s], lo = blk_lo - at[s];
        const int seen = hi < 0 ? 0 : hi < live[s] ? hi : live[s];
        first[s] = lo <= 0 ? 0 : lo / SP_UNIT;
        const int units = (seen + SP_UNIT - 1) / SP_UNIT - first[s];
        total += units > 0 ? units : 0;
        end[s] = total;
    }
    const int w0 = (int)((int64_t)total * split / splits), w1 = (int)((int64_t)total * (split + 1) / splits);

    struct Unit { int s, t0, place, live; };   // span, first token in it, its slot, live tokens of the span
    auto unit = [&](int w) {
        Unit u;
        if (w < end[0]) u = {0, w + first[0], at[0], live[0]};
        else if (w < end[1]) u = {1, w - end[0] + first[1], at[1], live[1]};
        else if (w < end[2]) u = {2, w - end[1] + first[2], at[2], live[2]};
        else u = {3, w - end[2] + first[3], at[3], live[3]};
        u.t0 *= SP_UNIT;
        u.place += u.t0;
        return u;
    };

    // ---- queries as the B operand: row n, channels 16 ks + 8 h .. + 7
    const float c2 = __builtin_fabsf(a.scale) * LOG2E;
    u32x4 q[KS];
    {
        const u16 *src = (const u16 *)a.q + qrow * D + map * (D / MAPS) + 8 * h;
        const u32 sign = a.scale < 0.f ? 0x80008000u : 0u;   // the softmax takes the maximum of the scores themselves
        const bool q_bf16 = a.dtype == VQ_BF16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            u32x4 x = *(const u32x4 *)(src + 16 * ks);
            if (sizeof(T) == 2 && BITS != 0 && q_bf16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = as_u(f16x2{(f16)bf16_to_f32((u16)x[i]), (f16)bf16_to_f32((u16)(x[i] >> 16))});
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) q[ks][i] = a.scale == 0.f ? 0u : x[i] ^ sign;
        }
    }
    const float cc = a.scale == 0.f ? 1.f : c2;

    // ---- staging
    const u32 lds0 = lds_addr(lds);
    constexpr int COPIES = D / 32;   // copies of 1 KB a wave for a tile
    struct Words { u32 k[BITS ? D / 32 : 1], v[BITS == 4 ? D / 32 : BITS == 2 ? D / 64 : 1]; };
    constexpr int KROWS = SP_THREADS / CH;            // key tokens the threads cover at a time
    constexpr int PER = BITS ? 32 / BITS : 8, KW = D / PER;
    constexpr int VSTEPS = D / 64;                     // sixteen-token steps of a thread's channel
    const u32 magic = BITS ? vreg_const(Magic<BITS ? BITS : 4>::bits) : 0u;
    const int kc = tid % CH, kt = tid / CH;            // packed keys: 8-channel piece, token
    const int vc = tid % D, vh = tid / D;              // packed values: channel, which of the unit's stretches
    auto fetch = [&](const Unit &u, int buf, Words &wd) {
        const vq_kv_store &s = u.s < 2 ? a.prefix : a.own;
        const int64_t sb = u.s < 2 ? 0 : b;
        const int last = u.live - 1 - u.t0;            // last live token of the unit, if it is not whole
        if (BITS && !(u.s & 1)) {
            const int64_t bh = sb * Hkv + hkv;
            const u32 *kw = (const u32 *)s.k_packed + (bh * s.cap_tokens + u.t0) * KW;
            const u32 *vw = (const u32 *)s.v_packed + (bh * (s.cap_tokens / PER) + u.t0 / PER) * D;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const int t = kt + KROWS * i;
                wd.k[i] = kw[(t < last ? t : last) * KW + (BITS == 4 ? kc : kc / 2)];
            }
            const int lastw = last / PER;
#pragma unroll
            for (int i = 0; i < (int)(sizeof(wd.v) / 4); ++i) {
                const int x = vh * (int)(sizeof(wd.v) / 4) + i;
                wd.v[i] = vw[(x < lastw ? x : lastw) * D + vc];
            }
            return;
        }
        if (BITS && a.tail_dtype == VQ_BF16) return;   // (converted on the way: store_unit)
        const int64_t ks = s.k_strides[2] * 2, vs = s.v_strides[2] * 2;
        const char *kb = (const char *)s.k_tail + (sb * s.k_strides[0] + hkv * s.k_strides[1]) * 2 + u.t0 * ks;
        const char *vb = (const char *)s.v_tail + (sb * s.v_strides[0] + hkv * s.v_strides[1]) * 2 + u.t0 * vs;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int slot = (wave * COPIES + i) * 64 + lane, t = slot / CH, p = slot % CH;
            const u32 r = (u32)(t < last ? t : last), dst = lds0 + buf * Tile::BUF + (wave * COPIES + i) * 1024;
            lds_copy16<0>(kb, r * (u32)ks + sp_kpiece<D>(t, p) * 16, dst);
            lds_copy16<0>(vb, r * (u32)vs + sp_vpiece<D>(t, p) * 16, dst + Tile::KEYS);
        }
    };
    auto store_unit = [&](const Unit &u, int buf, const Words &wd) {
        if (!BITS) return;
        const vq_kv_store &s = u.s < 2 ? a.prefix : a.own;
        const int64_t sb = u.s < 2 ? 0 : b;
        const int last = u.live - 1 - u.t0;
        char *kd = lds + buf * Tile::BUF, *vd = kd + Tile::KEYS;
        if (u.s & 1) {
            if (a.tail_dtype != VQ_BF16) return;
            const u16 *kb = (const u16 *)s.k_tail + sb * s.k_strides[0] + hkv * s.k_strides[1] + u.t0 * s.k_strides[2];
            const u16 *vb = (const u16 *)s.v_tail + sb * s.v_strides[0] + hkv * s.v_strides[1] + u.t0 * s.v_strides[2];
            for (int i = 0; i < D / 32; ++i) {
                const int t = kt + KROWS * i, r = t < last ? t : last;
                *(f16x8 *)(kd + t * D * 2 + sp_kpiece<D>(t, kc) * 16) = ld_tail8(kb, r * s.k_strides[2] + 8 * kc, true);
                *(f16x8 *)(vd + t * D * 2 + sp_vpiece<D>(t, kc) * 16) = ld_tail8(vb, r * s.v_strides[2] + 8 * kc, true);
            }
            return;
        }
        constexpr int BB = BITS ? BITS : 4;
        const int gshift = __builtin_ctz(a.group);
        const int64_t bh = sb * Hkv + hkv;
        const int64_t kg = bh * (s.cap_tokens >> gshift);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            // the unit's first and second 32 tokens are one key group or two
            const int t = kt + KROWS * i, g32 = KROWS * i / 32;
            const int64_t g = (kg + ((u.t0 + (32 * g32 < last ? 32 * g32 : last)) >> gshift)) * D + 8 * kc;
            u32 code[4];
            sp_codes8<BB>(BITS == 2 ? wd.k[i] >> (16 * (kc & 1)) : wd.k[i], magic, code);
            *(u32x4 *)(kd + t * D * 2 + sp_kpiece<D>(t, kc) * 16) =
                sp_values8(code, *(const uint4 *)((const f16 *)s.k_scale + g), *(const uint4 *)((const f16 *)s.k_zero + g));
        }
        const int64_t vg = (bh * (D >> gshift) + (vc >> gshift)) * s.cap_tokens + u.t0;
        const bool whole = last >= SP_UNIT - 1;
#pragma unroll
        for (int i = 0; i < VSTEPS; ++i) {
            const int step = vh * VSTEPS + i;
            u32x4 x[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {   // eight tokens each
                int t = 16 * step + 8 * k;
                const int tc = t <= last ? t : last / 8 * 8;   // (past the live tokens: any that are)
                u32 code[4];
                sp_codes8<BB>(BITS == 4 ? wd.v[BITS == 4 ? 2 * i + k : 0] : wd.v[BITS == 4 ? 0 : i] >> (16 * k), magic, code);
                x[k] = sp_values8(code, *(const uint4 *)((const f16 *)s.v_scale + vg + tc), *(const uint4 *)((const f16 *)s.v_zero + vg + tc));
                if (!whole) {   // a token past the live ones may hold anything: its weight is zero, its value has to be finite
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (t + 2 * e > last) x[k][e] = 0u;
                        else if (t + 2 * e + 1 > last) x[k][e] &= 0xFFFFu;
                    }
                }
            }
            u32x4 *dst = (u32x4 *)(vd + vc * SP_VROW + step * 32);
            dst[0] = u32x4{x[0][0], x[0][1], x[1][0], x[1][1]};
            dst[1] = u32x4{x[0][2], x[0][3], x[1][2], x[1][3]};
        }
    };

    // ---- state of the lane's row
    f32x16 O[DT];
    float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] = 0.f;

    auto work = [&](const Unit &u, int buf, int half) {   // 32 slots of the unit
        const char *kd = lds + buf * Tile::BUF, *vd = kd + Tile::KEYS;
        const int place = u.place + 32 * half;
        if (place >= any_hi || place + 32 <= any_lo || 32 * half >= u.live - u.t0) return;
        f32x16 S;
#pragma unroll
        for (int r = 0; r < 16; ++r) S[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            S = M::mma(*(const u32x4 *)(kd + (32 * half + n) * D * 2 + sp_kpiece<D>(n, 2 * (map * KS + ks) + h) * 16), q[ks], S);
        const int live_end = u.place + u.live - u.t0;   // slot past the span's live tokens
        if (place + 32 > (all_hi < live_end ? all_hi : live_end) || place < all_lo) {
            const int hi = (lane_hi < live_end ? lane_hi : live_end) - place - 4 * h, lo = lane_lo - place - 4 * h;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int t = 8 * (r / 4) + r % 4;
                if (t >= hi || t < lo) S[r] = -INFINITY;
            }
        }
        float mx = fmaxf(S[0], S[1]);
#pragma unroll
        for (int r = 2; r < 16; ++r) mx = fmaxf(mx, S[r]);
        if (__any(mx * cc > m_run + RESCALE_SLACK)) {
            const float top = fmaxf(mx, __shfl_xor(mx, 32)) * cc, m = fmaxf(m_run, top);
            const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m);
            m_run = m;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) O[dt][r] *= alpha;
        }
        const float nm = m_run == -INFINITY ? 0.f : -m_run;
        u32 P[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            P[r] = M::pack(__builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * r], cc, nm)), __builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * r + 1], cc, nm)));
            l_run = M::add_pair(P[r], l_run);
        }
        const bool transposed = BITS && !(u.s & 1);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                u32x4 v;
                if (transposed) {
                    v = *(const u32x4 *)(vd + (32 * dt + n) * SP_VROW + (2 * half + s) * 32 + 16 * h);
                } else {
                    const int i = lane & 15, t = 4 * h + (i >> 2), p = 4 * dt + 2 * (lane >> 4 & 1) + ((i & 3) >> 1);
                    const char *row = vd + (32 * half + 16 * s + t) * D * 2 + sp_vpiece<D>(t, p) * 16 + (i & 1) * 8;
                    using L = __attribute__((address_space(3))) s16x4;
                    const uint2 v0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)(uintptr_t)lds_addr(row)));
                    const uint2 v1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)(uintptr_t)lds_addr(row + 8 * D * 2)));
                    v = u32x4{v0.x, v0.y, v1.x, v1.y};
                }
                O[dt] = M::mma(v, u32x4{P[4 * s], P[4 * s + 1], P[4 * s + 2], P[4 * s + 3]}, O[dt]);
            }
        }
    };
    const int half0 = wt == 1 ? 0 : th, half1 = wt == 1 ? 2 : th + 1;

    if (w0 < w1) {
        Words wd;
        Unit u = unit(w0);
        fetch(u, 0, wd);
        store_unit(u, 0, wd);
        wait_copies<0>();
        lds_barrier();
        int buf = 0;
        for (int w = w0; w < w1; ++w, buf ^= 1) {
            const bool more = w + 1 < w1;
            Unit next = u;
            if (more) {
                next = unit(w + 1);
                fetch(next, buf ^ 1, wd);
            }
            if (wave_works) {
#pragma unroll 1
                for (int half = half0; half < half1; ++half) work(u, buf, half);
            }
            if (more) {
                store_unit(next, buf ^ 1, wd);
                wait_copies<0>();
                lds_barrier();
                u = next;
            }
        }
    }

    // ---- results
    float l = l_run + __shfl_xor(l_run, 32);   // both halves of a row
    if (c.nparts > 1) {
        if (j >= rows) return;
        const int64_t rec = (qrow * c.nparts + part) * MAPS + map;
        if (h == 0) *(float2 *)(c.ml + rec * 2) = make_float2(m_run, l);
        float *dst = c.sums + rec * D + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; r += 4) *(float4 *)(dst + 32 * dt + 2 * r) = make_float4(O[dt][r], O[dt][r + 1], O[dt][r + 2], O[dt][r + 3]);
        return;
    }
    float by = l > 0.f || l != l ? 1.f / l : 0.f, gain = 1.f, sq = 0.f;
    if (MAPS == 2 && map == 1) by *= -span_lam(a, hkv * G + rem % G);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] *= by;
    bool norm = false;
    if (MAPS == 2) {
        // the second map's wave hands its rows over in LDS, a channel tile's quarter of 4 floats a lane at a time
        static_assert(Tile::LDS >= 2 * D * 32 * 4 || MAPS == 1, "room for the rows of both row groups");
        float4 *room = (float4 *)lds + rg * (D / 8) * 64 + lane;
        lds_barrier();
        if (map == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 4; ++r) room[(4 * dt + r) * 64] = make_float4(O[dt][4 * r], O[dt][4 * r + 1], O[dt][4 * r + 2], O[dt][4 * r + 3]);
        }
        lds_barrier();
        if (map == 1) return;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 x = room[(4 * dt + r) * 64];
                O[dt][4 * r] += x.x; O[dt][4 * r + 1] += x.y; O[dt][4 * r + 2] += x.z; O[dt][4 * r + 3] += x.w;
            }
        gain = a.gain;
        norm = a.norm_weight != nullptr;
        if (norm) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) sq = __builtin_fmaf(O[dt][r], O[dt][r], sq);
            gain /= sqrtf((sq + __shfl_xor(sq, 32)) * (1.f / D) + a.norm_eps);
        }
    }
    if (j >= rows) return;
    u16 *dst = (u16 *)a.out + qrow * D + 4 * h;
    const bool out_bf16 = a.dtype == VQ_BF16;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[e] = O[dt][r + e] * gain;
                if (norm) o[e] *= span_ld(a.norm_weight, a.norm_dtype, 32 * dt + 2 * r + 4 * h + e);
            }
            const uint2 x = out_bf16 ? make_uint2(SpanMma<bf16_t>::pack(o[0], o[1]), SpanMma<bf16_t>::pack(o[2], o[3]))
                                     : make_uint2(SpanMma<f16>::pack(o[0], o[1]), SpanMma<f16>::pack(o[2], o[3]));
            *(uint2 *)(dst + 32 * dt + 2 * r) = x;
        }
}

template <int BITS, typename T, int D, int MAPS> int launch_span_mfma_as(const SpanCall &c) {
    constexpr int bytes = SpanTile<BITS, D>::LDS;
    const auto kernel = span_mfma_kernel<BITS, T, D, MAPS>;
    if (bytes > 64 * 1024) {   // has to be allowed per kernel and device, once; a second setter repeats the same call
        static std::atomic<bool> allowed[64] = {};
        int dev = 0;
        (void)hipGetDevice(&dev);
        if (dev < 0 || dev >= 64 || !allowed[dev].load(std::memory_order_acquire)) {
            (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (dev >= 0 && dev < 64) allowed[dev].store(true, std::memory_order_release);
        }
    }
    const int64_t blocks = (c.apart ? (int64_t)c.psplits * c.ptiles * c.a.Hkv : 0) + c.a.B * c.a.Hkv * c.otiles * c.osplits;
    VQ_REQUIRE(blocks < (INT64_C(1) << 24), VQ_ERR_UNSUPPORTED, "attention over spans: too many sequences and heads for one launch");
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
