// Attention over chosen blocks of a packed store and over all of its plain rows.
//
// Row (b, h, i) of a query sees, of the packed slots, those of the blocks that its tile's list names (tile i / query_block of its kv
// head), each entry's slots e block .. (e + 1) block - 1 as far as they are live and not behind the query; entries below zero or past
// the store name nothing, an entry that is named twice counts twice.  Behind them come the plain rows (the tail), up to the query's own
// place.  o = sum p v / sum p, p = exp(scale q k - max) over what it sees; a row that sees nothing is zero.
#include "attend_blocks.hpp"

namespace vq {

namespace {

// Any head size up to 256, type, bit width, layout and strides, in float32 on the vector units: a wave takes a query row over a run
// of its list's entries and a run of its tail, lanes along the channels.
__global__ __launch_bounds__(256) void blocks_any_kernel(BlockCall c) {
    constexpr int E = SPAN_MAX_D / 64;
    const vq_store_attend_args &a = c.s.a;
    const int lane = threadIdx.x & 63;
    const int64_t wid = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (wid >= a.B * a.Hq * a.Sq * c.s.nparts) return;   // whole waves leave together
    const int64_t row = wid / c.s.nparts, part = wid % c.s.nparts;
    const int64_t pos = row % a.Sq, h = row / a.Sq % a.Hq, b = row / (a.Sq * a.Hq);
    const int64_t hkv = h / (a.Hq / a.Hkv), D = a.D, bh = b * a.Hkv + hkv;
    int64_t lo, hi;
    span_visible(a, span_own_live(a, b), pos, lo, hi);
    const float scale = a.scale * LOG2E;
    const int32_t *list = c.blocks + (bh * c.tiles + pos / c.query_block) * c.count;

    float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int64_t d = lane + 64 * e;
        q[e] = d < D ? span_ld(a.q, a.dtype, row * D + d) : 0.f;
        acc[e] = 0.f;
    }
    const SpanPacked p = SpanPacked::of(a, a.own);
    auto take = [&](int64_t t) {
        float v[E], dot = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t d = lane + 64 * e;
            v[e] = 0.f;
            if (d >= D) continue;
            float k;
            if (t < a.own.n_packed) {
                k = p.key(bh, t, d);
                v[e] = p.value(bh, t, d);
            } else {
                const int64_t r = t - a.own.n_packed;
                k = span_ld(a.own.k_tail, a.tail_dtype, b * a.own.k_strides[0] + hkv * a.own.k_strides[1] + r * a.own.k_strides[2] + d);
                v[e] = span_ld(a.own.v_tail, a.tail_dtype, b * a.own.v_strides[0] + hkv * a.own.v_strides[1] + r * a.own.v_strides[2] + d);
            }
            dot = __builtin_fmaf(q[e], k, dot);
        }
        const float x = span_wave_sum(dot) * scale, mn = fmaxf(m, x);
        const float keep = mn == -INFINITY ? 1.f : exp2f(m - mn), y = mn == -INFINITY && x == x ? 0.f : exp2f(x - mn);
        l = l * keep + y;
        m = mn;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = __builtin_fmaf(y, v[e], acc[e] * keep);
    };
    const int64_t packed = hi < a.own.n_packed ? hi : a.own.n_packed;
    for (int64_t i = c.count * part / c.s.nparts; i < c.count * (part + 1) / c.s.nparts; ++i) {
        const int64_t t0 = (int64_t)list[i] * c.block_tokens;
        if (t0 < 0) continue;
        const int64_t t1 = t0 + c.block_tokens < packed ? t0 + c.block_tokens : packed;
        for (int64_t t = t0; t < t1; ++t) take(t);
    }
    const int64_t n = hi > a.own.n_packed ? hi - a.own.n_packed : 0;
    for (int64_t t = n * part / c.s.nparts; t < n * (part + 1) / c.s.nparts; ++t) take(a.own.n_packed + t);
    const int64_t rec = row * c.s.nparts + part;
    if (lane == 0) { c.s.ml[rec * 2] = m; c.s.ml[rec * 2 + 1] = l; }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 64 * e < D) c.s.sums[rec * D + lane + 64 * e] = acc[e];
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
    // Parts are added up in the launch where a tile's are 32 KB at most, which the one block that does it reads past its caches at ~20 GB/s (4 rows of 128
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
    // as many waves as fill the chip eight deep, runs of 64 slots or more
    const int64_t rows = a.B * a.Hq * a.Sq;
    double slots = (double)c.count * (double)c.block_tokens;
    slots = (slots < (double)a.own.n_packed ? slots : (double)a.own.n_packed) + (double)a.own.n_tail;
    int64_t parts = 8192 / rows;
    if ((double)parts > slots / 64.) parts = (int64_t)(slots / 64.);
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
    blocks_any_kernel<<<(unsigned)cdiv(a.B * a.Hq * a.Sq * c.s.nparts, 4), 256, 0, (hipStream_t)a.stream>>>(c);
    VQ_HIP_CHECK_LAUNCH(fn);
    return launch_span_merge1(fn, c.s);
}
