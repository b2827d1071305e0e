// Attention over chosen blocks of a packed store and over all of its plain rows.
//
// Row (b, h, i) of a query sees, of the packed slots, those of the blocks that its tile's list names (tile i / query_block of its kv
// head), each entry's slots e block .. (e + 1) block - 1 as far as they are live and not behind the query; entries below zero or past
// the store name nothing, an entry that is named twice counts twice.  Behind them come the plain rows (the tail), up to the query's own
// place.  o = sum p v / sum p, p = exp(scale q k - max) over what it sees; a row that sees nothing is zero.
#include "attend_blocks.hpp"
#include "attend_span_mfma.hpp"

namespace vq {

namespace {

// Any head size up to 256, type, bit width, layout and strides, in float32: a block of four waves takes 16 RT rows of a kv head's query heads at the
// positions of one list, over a run of units of 32 slots, the list's slots in one line and then the tail's.  A unit's slots are looked up by one wave,
// reconstructed by all threads, a channel each, and laid down in LDS as float32 once for all rows; scores and sums are products of float32 numbers
// (v_mfma_f32_16x16x4: lane i + 16 h holds row or column i of step h, and rows 4 h .. 4 h + 3 of column i of the result; a lane's four channels or
// slots in a row are those of four steps, any order serving a sum), the softmax has TPR threads a row.
//
// Bound by the latencies of a unit, one after another (its entries of the list, then its words in four batches, five barriers), with two blocks a CU (one
// past 192 channels with 32 rows, past 224 with 16: LDS) to cover each other: 16 sequences of 8 kv heads, 3.2k of 8-bit slots each, 214 us; a chunk of 512 queries in 64 lists of 2k slots 682 (a wave a row,
// each with its own reconstruction: 1891 and 33827).  Eight slots' words under way in place of four take registers that the second block needs (1080);
// a third of the loads, keys' scales shared and values' by way of LDS, is no faster (248 and 722).
constexpr int ANY_SP = 36;          // floats from row to row of the scores
constexpr int ANY_INFO = 4 * 32 + 4;   // ints about a unit
template <int RT> constexpr size_t any_bytes(int D) {
    const int kp = (D + 15) / 16 * 16 + 4;
    return (size_t)((16 * RT + 64) * kp + (3 - RT) * 16 * RT * ANY_SP + 16 * RT + 2 * ANY_INFO) * 4;
}
template <int RT> __global__ __launch_bounds__(256) void blocks_any_kernel(BlockCall c) {
    constexpr int ROWS = 16 * RT, TPR = 256 / ROWS, SPT = 32 / TPR, HALVES = 3 - RT;   // (16 rows: two waves share a tile of scores, half of the channels each)
    extern __shared__ __align__(16) float any_lds[];
    const vq_store_attend_args &a = c.s.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, h = lane >> 4;
    const int D = (int)a.D, Dp = (D + 15) / 16 * 16, KP = Dp + 4, steps = Dp / 16, G = (int)(a.Hq / a.Hkv), n_packed = (int)a.own.n_packed;
    float *const Qs = any_lds, *const Ks = Qs + ROWS * KP, *const Vs = Ks + 32 * KP, *const Sb = Vs + 32 * KP, *const keeps = Sb + HALVES * ROWS * ANY_SP;
    int *const infos = (int *)(keeps + ROWS);
    u32 id = blockIdx.x;
    const int part = (int)(id % (u32)c.s.nparts);
    id /= (u32)c.s.nparts;
    const int j0 = (int)(id % (u32)c.row_tiles) * ROWS;
    id /= (u32)c.row_tiles;
    const int tile = (int)(id % (u32)c.tiles);
    const int64_t bh = id / (u32)c.tiles, b = bh / a.Hkv, hkv = bh % a.Hkv;
    const int pos0 = (int)(tile * c.query_block), at_once = (int)(a.Sq - pos0 < c.query_block ? a.Sq - pos0 : c.query_block);
    const int here = at_once * G - j0 < ROWS ? at_once * G - j0 : ROWS;
    if (here <= 0) return;   // (the last tile may hold fewer rows)
    auto row_of = [&](int x) __attribute__((always_inline)) { return (b * a.Hq + hkv * G + (j0 + x) % G) * a.Sq + pos0 + (j0 + x) / G; };
    const int64_t live = span_own_live(a, b);
    int64_t lo, hi, any_hi;
    const int mine = tid / TPR < here ? tid / TPR : here - 1;   // the row of this thread's softmax
    span_visible(a, live, pos0 + (j0 + mine) / G, lo, hi);
    span_visible(a, live, pos0 + (j0 + here - 1) / G, lo, any_hi);
    const int limit = (int)(any_hi < n_packed ? any_hi : n_packed);

    // ---- a channel and every step-th row or slot a thread
    const int step = 256 / Dp, d = tid % Dp, s0 = tid < step * Dp ? tid / Dp : 32, dd = d < D ? d : D - 1;
    for (int x = s0; x < ROWS; x += step) Qs[x * KP + d] = x < here && d < D ? span_ld(a.q, a.dtype, row_of(x) * D + d) : 0.f;
    const SpanPacked p = SpanPacked::of(a, a.own);
    const bool token = a.v_layout == VQ_V_TOKEN_PACKED;
    const int kd = dd / p.per, kshift = dd % p.per * p.bits, vg = dd / p.group;
    const int64_t kwords = bh * a.own.cap_tokens, kmeta = bh * p.GK, vwords = token ? bh * (a.own.cap_tokens / p.per) : kwords, vmeta = (bh * p.GV + vg) * a.own.cap_tokens;
    // a unit's packed slots, its places in `info`: slots (or another of the unit where there is none), groups, rows of words, shifts
    auto packed = [&](const int *info, u32 there, auto meta) __attribute__((always_inline)) {
        using T = decltype(meta);
        const T *const ksc = (const T *)a.own.k_scale, *const kz = (const T *)a.own.k_zero, *const vsc = (const T *)a.own.v_scale, *const vz = (const T *)a.own.v_zero;
        const u32 *const kp = (const u32 *)a.own.k_packed, *const vp = (const u32 *)a.own.v_packed;
        constexpr int N = 4;   // slots whose words are under way
#pragma unroll 1
        for (int s = s0; s < 32; s += N * step) {
            u32 kw[N], vw[N];
            T k_s[N], k_z[N], v_s[N], v_z[N];
            int vshift[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int x = s + j * step < 32 ? s + j * step : s, t = info[x];
                kw[j] = kp[(kwords + t) * p.W + kd];
                const int64_t km = (kmeta + info[32 + x]) * D + dd;
                k_s[j] = ksc[km];
                k_z[j] = kz[km];
                vw[j] = token ? vp[(vwords + info[64 + x]) * D + dd] : vp[(vwords + t) * p.W + kd];
                vshift[j] = token ? info[96 + x] : kshift;
                const int64_t vm = token ? vmeta + t : (kwords + t) * p.GV + vg;
                v_s[j] = vsc[vm];
                v_z[j] = vz[vm];
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int x = s + j * step;
                if (x >= 32) break;
                const bool is = d < D && there >> x & 1;
                const float k = (float)(f16)__builtin_fmaf((float)(kw[j] >> kshift & p.mask), (float)k_s[j], (float)k_z[j]);
                const float v = (float)(f16)__builtin_fmaf((float)(vw[j] >> vshift[j] & p.mask), (float)v_s[j], (float)v_z[j]);
                Ks[x * KP + d] = is ? k : 0.f;
                Vs[x * KP + d] = is ? v : 0.f;
            }
        }
    };
    auto mixed = [&](const int *info, u32 there) __attribute__((always_inline)) {
        for (int x = s0; x < 32; x += step) {
            float k = 0.f, v = 0.f;
            if (d < D && there >> x & 1) {
                const int t = info[x], r = t - n_packed;
                if (r < 0) {
                    k = p.key(bh, t, d);
                    v = p.value(bh, t, d);
                } else {
                    k = span_ld(a.own.k_tail, a.tail_dtype, b * a.own.k_strides[0] + hkv * a.own.k_strides[1] + r * a.own.k_strides[2] + d);
                    v = span_ld(a.own.v_tail, a.tail_dtype, b * a.own.v_strides[0] + hkv * a.own.v_strides[1] + r * a.own.v_strides[2] + d);
                }
            }
            Ks[x * KP + d] = k;
            Vs[x * KP + d] = v;
        }
    };

    const float scale = a.scale * LOG2E;
    const int32_t *const list = c.blocks + (bh * c.tiles + tile) * c.count;
    const u32 sub = (u32)c.sub;
    float m = -INFINITY, l = 0.f;
    f32x4 acc[4][RT];   // of 16 channels each, every fourth a wave
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[y][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t run = c.units / c.s.nparts, longer = c.units % c.s.nparts, u0 = part * run + (part < longer ? part : longer);   // (the first runs a unit longer)
    const int64_t u1 = u0 + run + (part < longer ? 1 : 0);
#pragma unroll 1
    for (int64_t u = u0; u < u1; ++u) {
        int *const info = infos + (int)(u & 1) * ANY_INFO;   // (two in turn: a unit that holds nothing is left without another barrier)
        if (wave == 0) {
            const int64_t at = u * 32 + (lane & 31);
            int t = -1;
            if (at < c.list_slots) {
                const int64_t e = c.list_slots >> 32 == 0 ? (int64_t)((u32)at / sub) : at / sub;
                const int64_t slot = (int64_t)list[e] * c.block_tokens + (at - e * sub);
                if (slot >= 0 && slot < limit) t = (int)slot;
            } else if (n_packed + (at - c.list_slots) < any_hi) {   // (what the last row sees lies within the store)
                t = n_packed + (int)(at - c.list_slots);
            }
            const u32 there = (u32)__ballot(t >= 0), tail = (u32)__ballot(t >= n_packed);
            if (there != 0) t = t >= 0 ? t : __shfl(t, __builtin_ctz(there));
            if (lane < 32 && there != 0) {
                info[lane] = t;
                info[32 + lane] = (int)((u32)t / (u32)p.group);
                info[64 + lane] = (int)((u32)t / (u32)p.per);
                info[96 + lane] = (int)((u32)t % (u32)p.per) * p.bits;
            }
            if (lane == 0) { info[128] = (int)there; info[129] = tail != 0; }
        }
        __syncthreads();
        const u32 there = (u32)__builtin_amdgcn_readfirstlane(info[128]);
        if (there == 0) continue;
        if (__builtin_amdgcn_readfirstlane(info[129])) mixed(info, there);
        else if (a.meta_dtype == VQ_F16) packed(info, there, (f16)0.f);
        else packed(info, there, 0.f);
        // (a unit's own slots, for the softmax behind the next barrier)
        __syncthreads();
        {
            const int rt = RT == 2 ? wave & 1 : 0, st = RT == 2 ? wave >> 1 : wave & 1, half = RT == 2 ? 0 : wave >> 1;
            const int k0 = half ? steps / 2 : 0, k1 = RT == 2 || half ? steps : steps / 2;
            f32x4 S = {0.f, 0.f, 0.f, 0.f};
            const float *const x = Qs + (rt * 16 + i) * KP + 4 * h, *const y = Ks + (st * 16 + i) * KP + 4 * h;
            for (int k = k0; k < k1; ++k) {
                const f32x4 x4 = *(const f32x4 *)(x + 16 * k), y4 = *(const f32x4 *)(y + 16 * k);
#pragma unroll
                for (int e = 0; e < 4; ++e) S = __builtin_amdgcn_mfma_f32_16x16x4f32(x4[e], y4[e], S, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) Sb[(half * ROWS + rt * 16 + 4 * h + r) * ANY_SP + st * 16 + i] = S[r];
        }
        __syncthreads();
        {
            float *const s = Sb + tid / TPR * ANY_SP + tid % TPR * SPT;
            float x[SPT], top = m;
#pragma unroll
            for (int j = 0; j < SPT; ++j) {
                const int at = tid % TPR * SPT + j;
                x[j] = (HALVES == 2 ? s[j] + s[ROWS * ANY_SP + j] : s[j]) * scale;
                if (!(there >> at & 1) || info[at] >= hi) x[j] = -INFINITY;
                top = fmaxf(top, x[j]);
            }
#pragma unroll
            for (int off = 1; off < TPR; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
            const float keep = top == -INFINITY ? 1.f : exp2f(m - top);
            l *= keep;
#pragma unroll
            for (int j = 0; j < SPT; ++j) {
                const float y = top == -INFINITY && x[j] == x[j] ? 0.f : exp2f(x[j] - top);
                l += y;
                s[j] = y;
            }
            m = top;
            if (tid % TPR == 0) keeps[tid / TPR] = keep;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const f32x4 keep = *(const f32x4 *)(keeps + r * 16 + 4 * h);
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[y][r][e] *= keep[e];
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            f32x4 w[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) w[r] = *(const f32x4 *)(Sb + (r * 16 + i) * ANY_SP + 16 * g + 4 * h);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int ct = wave + 4 * y;
                if (ct >= steps) break;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = Vs[(16 * g + 4 * h + e) * KP + ct * 16 + i];
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[y][r] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r][e], v, acc[y][r], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int off = 1; off < TPR; off <<= 1) l += __shfl_xor(l, off);
    if (tid % TPR == 0 && tid / TPR < here) {
        float *const ml = c.s.ml + (row_of(tid / TPR) * c.s.nparts + part) * 2;
        ml[0] = m;
        ml[1] = l;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int x = r * 16 + 4 * h + e;
            if (x >= here) continue;
            float *const sums = c.s.sums + (row_of(x) * c.s.nparts + part) * D;
#pragma unroll
            for (int y = 0; y < 4; ++y)
                if ((wave + 4 * y) * 16 + i < D) sums[(wave + 4 * y) * 16 + i] = acc[y][r][e];
        }
}

template <int RT> int launch_blocks_any(const char *fn, const BlockCall &c, int64_t blocks) {
    const size_t bytes = any_bytes<RT>((int)c.s.a.D);
    static std::atomic<bool> allowed[64] = {};
    if (bytes > 64 * 1024)
        if (int rc = span_allow_lds((const void *)blocks_any_kernel<RT>, (int)any_bytes<RT>(SPAN_MAX_D), allowed)) return rc;
    blocks_any_kernel<RT><<<(unsigned)blocks, 256, bytes, (hipStream_t)c.s.a.stream>>>(c);
    VQ_HIP_CHECK_LAUNCH(fn);
    return VQ_OK;
}

int check_blocks(const char *fn, const vq_block_attend_args *args) {
    VQ_REQUIRE(args != nullptr, VQ_ERR_INVALID, "%s: null argument block", fn);
    const vq_store_attend_args &a = args->store;
    if (int rc = span_check_call(fn, &a, 1)) return rc;
    VQ_REQUIRE(span_prefix_slots(a) == 0, VQ_ERR_INVALID, "%s: takes no shared prefix", fn);
    VQ_REQUIRE(a.sliding_window == 0, VQ_ERR_INVALID, "%s: takes no sliding window", fn);
    VQ_REQUIRE(args->block_tokens >= 1 && args->block_tokens < (INT64_C(1) << 30), VQ_ERR_INVALID, "%s: bad block size", fn);
    VQ_REQUIRE(args->query_block >= 1 && args->query_block < (INT64_C(1) << 30), VQ_ERR_INVALID, "%s: query_block must be at least 1", fn);
    VQ_REQUIRE(args->count >= 0 && args->count < (INT64_C(1) << 30), VQ_ERR_INVALID, "%s: bad list length", fn);
    VQ_REQUIRE(args->count == 0 || args->blocks != nullptr, VQ_ERR_INVALID, "%s: null blocks", fn);
    return VQ_OK;
}

// The matrix-unit kernel takes what it takes of attention over spans, where blocks are whole units of 32 slots: tiles of 32 rows of a kv head's
// query heads at the positions of one list, each over the list's units, in as many runs as fill the chip.
bool plan_few(BlockCall &c, const vq_block_attend_args &args) {
    const vq_store_attend_args &a = c.s.a;
    if (c.block_tokens % 32 != 0 || !span_mfma_supported(a)) return false;
    const int64_t all = cdiv(a.own.n_packed, 32), sub = c.block_tokens / 32 < all ? c.block_tokens / 32 : all;
    const int64_t qb = c.query_block < a.Sq ? c.query_block : a.Sq, row_tiles = cdiv(a.Hq / a.Hkv * qb, 32);
    if (c.count * sub >= (1 << 24)) return false;
    const int64_t units = c.count * sub + cdiv(a.own.n_tail, 32), items = a.B * a.Hkv * c.tiles * row_tiles;
    // One round of blocks of equal runs, two blocks a CU (one with heads of 256 channels), two units a wave or
    // more, of long lists four (8 kv heads: 69 units 15.1 us in runs of eight, 15.6 of sixteen; 261 units 16.4 and 14.9)
    int64_t run = cdiv(items * units, a.D == 256 ? 256 : 512);
    if (run < (units > 128 ? 16 : 8)) run = units > 128 ? 16 : 8;
    if (run > BLOCK_UNITS) run = BLOCK_UNITS;
    const int64_t splits = units > 0 ? cdiv(units, run) : 1;
    if (items * splits >= (1 << 22) || splits > 65535 || c.tiles * row_tiles > 65535) return false;
    c.s.apart = c.s.pfew = 0;
    c.s.ofew = 1;
    c.s.owaves = 4;
    c.s.osplits = c.s.nparts = (int)splits;
    // Parts are added up in the launch where a tile's are 32 KB at most, which the one block that does it reads past its caches at 9 to 14 GB/s (4 rows of 128
    // channels in nine parts, 18 KB: 1.9 us; 9 rows of 256 in eleven, 99 KB: 7.5, and a launch of its own 4 to 5)
    const int64_t rows = a.Hq / a.Hkv * qb < 32 ? a.Hq / a.Hkv * qb : 32;
    const bool join = splits > 1 && items <= args.counters_len && rows * splits * a.D * 4 <= 32 * 1024;
    c.lists = {c.blocks, (int)c.tiles, (int)c.count, (int)c.block_tokens, (int)qb, (int)cdiv(a.own.n_packed, c.block_tokens), (int)sub, (int)(c.count * sub),
               (int)units, (int)(units / splits), (int)(units % splits), (int)row_tiles, join ? args.counters : nullptr};
    c.few = 1;
    return true;
}

BlockCall cut_blocks(const vq_block_attend_args &args) {
    BlockCall c = {};
    c.s.a = args.store;
    c.blocks = args.blocks;
    c.count = args.count;
    c.block_tokens = args.block_tokens;
    c.query_block = args.query_block;
    const vq_store_attend_args &a = c.s.a;
    c.tiles = cdiv(a.Sq, c.query_block);
    if (plan_few(c, args)) return c;
    // two blocks a CU, two units or more a run (8 kv heads, 69 units of 8-bit slots: 35 us, in runs of four 45)
    const int64_t G = a.Hq / a.Hkv;
    if (c.query_block > a.Sq) c.query_block = a.Sq;
    c.rows16 = G * c.query_block > 16 ? 2 : 1;
    c.row_tiles = (int)cdiv(G * c.query_block, 16 * c.rows16);
    c.sub = c.block_tokens < a.own.n_packed ? c.block_tokens : a.own.n_packed;
    c.list_slots = c.count * c.sub;
    c.units = cdiv(c.list_slots + a.own.n_tail, 32);
    int64_t parts = cdiv(512, a.B * a.Hkv * c.tiles * c.row_tiles);
    if (parts > c.units / 2) parts = c.units / 2;
    c.s.nparts = (int)(parts < 1 ? 1 : parts);
    return c;
}

int64_t block_floats(const BlockCall &c, int64_t &sums);
size_t block_bytes(const BlockCall &c) {
    int64_t sums;
    return c.few && c.s.nparts == 1 ? 0 : (size_t)block_floats(c, sums) * 4;
}

// (the sums take whole 16 bytes, so that the pairs behind them are aligned with odd heads too)
int64_t block_floats(const BlockCall &c, int64_t &sums) {
    const int64_t recs = c.s.a.B * c.s.a.Hq * c.s.a.Sq * c.s.nparts;
    sums = cdiv(recs * c.s.a.D, 4) * 4;
    return sums + recs * 2;
}

}  // namespace

}  // namespace vq

extern "C" size_t vq_block_attend_workspace(const vq_block_attend_args *args) {
    using namespace vq;
    if (check_blocks("vq_block_attend", args) != VQ_OK) return 0;
    if (args->store.own.n_packed == 0) return vq_shared_prefix_attend_workspace(&args->store);   // (no list names a slot)
    return block_bytes(cut_blocks(*args));
}

extern "C" int vq_block_attend(const vq_block_attend_args *args) {
    using namespace vq;
    const char *fn = "vq_block_attend";
    if (int rc = check_blocks(fn, args)) return rc;
    if (args->store.own.n_packed == 0) return vq_shared_prefix_attend(&args->store);
    BlockCall c = cut_blocks(*args);
    const vq_store_attend_args &a = c.s.a;
    const size_t need = block_bytes(c);
    VQ_REQUIRE(need == 0 || (a.workspace != nullptr && a.workspace_bytes >= need && ((uintptr_t)a.workspace & 15) == 0), VQ_ERR_WORKSPACE,
               "%s: workspace of %zu bytes required, 16-byte aligned", fn, need);
    if (need > 0) {
        int64_t sums;
        (void)block_floats(c, sums);
        c.s.sums = (float *)a.workspace;
        c.s.ml = c.s.sums + sums;
    }
    if (c.few) {
        if (int rc = a.pack_bits == 4 ? launch_blocks_few4(c.s, c.lists) : launch_blocks_few2(c.s, c.lists)) return rc;
        return need > 0 && c.lists.counters == nullptr ? launch_span_merge1(fn, c.s) : VQ_OK;
    }
    const int64_t blocks = a.B * a.Hkv * c.tiles * c.row_tiles * c.s.nparts;   // (no more than query rows, or 1024)
    if (int rc = c.rows16 == 2 ? launch_blocks_any<2>(fn, c, blocks) : launch_blocks_any<1>(fn, c, blocks)) return rc;
    return launch_span_merge1(fn, c.s);
}
