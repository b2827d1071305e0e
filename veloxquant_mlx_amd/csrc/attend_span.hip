// Entry points of attention over a shared prefix and of differential attention: checks, the cut of a call into parts, the kernel
// that takes any shape, the merge of the parts.
#include "attend_span.hpp"

namespace vq {

namespace {

constexpr int SPAN_MAX_D = 256;

// One element of a packed store's key or value as the fp16 number it stands for.
struct SpanPacked {
    const vq_kv_store *s;
    int bits, per, group, meta, v_layout;
    uint32_t mask;
    int64_t D, W, GV, GK;
    __device__ __forceinline__ float fp16_of(uint32_t word, int slot, const void *scale, const void *zero, int64_t at) const {
        const float code = (float)((word >> (slot * bits)) & mask);
        return (float)(f16)__builtin_fmaf(code, span_ld(scale, meta, at), span_ld(zero, meta, at));
    }
    __device__ __forceinline__ float key(int64_t bh, int64_t t, int64_t d) const {
        const uint32_t w = ((const uint32_t *)s->k_packed)[(bh * s->cap_tokens + t) * W + d / per];
        return fp16_of(w, (int)(d % per), s->k_scale, s->k_zero, (bh * GK + t / group) * D + d);
    }
    __device__ __forceinline__ float value(int64_t bh, int64_t t, int64_t d) const {
        if (v_layout == VQ_V_CHANNEL_PACKED) {
            const uint32_t w = ((const uint32_t *)s->v_packed)[(bh * s->cap_tokens + t) * W + d / per];
            return fp16_of(w, (int)(d % per), s->v_scale, s->v_zero, (bh * s->cap_tokens + t) * GV + d / group);
        }
        const uint32_t w = ((const uint32_t *)s->v_packed)[(bh * (s->cap_tokens / per) + t / per) * D + d];
        return fp16_of(w, (int)(t % per), s->v_scale, s->v_zero, (bh * GV + d / group) * s->cap_tokens + t);
    }
};

// Any head size up to 256, type, bit width, layout and strides, in float32 on the vector units: a wave takes a query row over
// a run of its slots, lanes along the channels.  For the shapes that the matrix-unit kernel does not take (float32 rows,
// head sizes other than 64, 128 and 256, fields of 1, 3 and 5 to 8 bits, groups of 16, channel-packed values, float32 scale and zero).
// A correct path, not a fast one: bound by vector instructions, most of them 64-bit divisions of a slot's place by the group and the word, paid
// by every query row for itself.  One token over 8k slots of 8 bits takes 455 us, 21 sequences on 16k of them 16.9 ms, two maps of a float32
// prompt of 1024 9.9 ms -- the plain form in torch 475 us, 1.6 ms and 0.9 ms.
template <int MAPS> __global__ __launch_bounds__(256) void span_any_kernel(SpanCall c) {
    constexpr int E = SPAN_MAX_D / 64;
    const vq_store_attend_args &a = c.a;
    const int lane = threadIdx.x & 63;
    const int64_t wid = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (wid >= a.B * a.Hq * a.Sq * c.nparts) return;   // whole waves leave together
    const int64_t row = wid / c.nparts, part = wid % c.nparts;
    const int64_t pos = row % a.Sq, h = row / a.Sq % a.Hq, b = row / (a.Sq * a.Hq);
    const int64_t hkv = h / (a.Hq / a.Hkv), D = a.D;
    const int64_t before = span_prefix_slots(a), total = before + span_own_live(a, b);
    int64_t lo, hi;
    span_visible(a, total, pos, lo, hi);
    const int64_t n = hi > lo ? hi - lo : 0;
    const int64_t t0 = lo + n * part / c.nparts, t1 = lo + n * (part + 1) / c.nparts;
    const float scale = a.scale * LOG2E;

    float q[E], acc[MAPS][E], m[MAPS], l[MAPS];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int64_t d = lane + 64 * e;
        q[e] = d < D ? span_ld(a.q, a.dtype, row * D + d) : 0.f;
#pragma unroll
        for (int w = 0; w < MAPS; ++w) acc[w][e] = 0.f;
    }
#pragma unroll
    for (int w = 0; w < MAPS; ++w) { m[w] = -INFINITY; l[w] = 0.f; }

    for (int64_t g = t0; g < t1; ++g) {
        const bool shared = g < before;
        const vq_kv_store &s = shared ? a.prefix : a.own;
        const int64_t t = shared ? g : g - before, sb = shared ? 0 : b;
        const int per = 32 / a.pack_bits;
        auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
        const SpanPacked p = {&s, a.pack_bits, per, a.group, a.meta_dtype, a.v_layout, (1u << a.pack_bits) - 1u, D, up(D, per),
                              up(D, a.group), up(s.cap_tokens, a.group)};
        float v[E], dot[MAPS];
#pragma unroll
        for (int w = 0; w < MAPS; ++w) dot[w] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t d = lane + 64 * e;
            v[e] = 0.f;
            if (d >= D) continue;
            float k;
            if (t < s.n_packed) {
                k = p.key(sb * a.Hkv + hkv, t, d);
                v[e] = p.value(sb * a.Hkv + hkv, t, d);
            } else {
                const int64_t r = t - s.n_packed;
                k = span_ld(s.k_tail, a.tail_dtype, sb * s.k_strides[0] + hkv * s.k_strides[1] + r * s.k_strides[2] + d);
                v[e] = span_ld(s.v_tail, a.tail_dtype, sb * s.v_strides[0] + hkv * s.v_strides[1] + r * s.v_strides[2] + d);
            }
            if (MAPS == 1 || d < D / 2) dot[0] = __builtin_fmaf(q[e], k, dot[0]);
            else dot[MAPS - 1] = __builtin_fmaf(q[e], k, dot[MAPS - 1]);
        }
#pragma unroll
        for (int w = 0; w < MAPS; ++w) {
            const float x = span_wave_sum(dot[w]) * scale, mn = fmaxf(m[w], x);
            const float f = exp2f(m[w] - mn), y = mn == -INFINITY && x == x ? 0.f : exp2f(x - mn);
            const float keep = mn == -INFINITY ? 1.f : f;
            l[w] = l[w] * keep + y;
            m[w] = mn;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[w][e] = __builtin_fmaf(y, v[e], acc[w][e] * keep);
        }
    }
    const int64_t rec = (row * c.nparts + part) * MAPS;
#pragma unroll
    for (int w = 0; w < MAPS; ++w) {
        if (lane == 0) { c.ml[(rec + w) * 2] = m[w]; c.ml[(rec + w) * 2 + 1] = l[w]; }
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 64 * e < D) c.sums[(rec + w) * D + lane + 64 * e] = acc[w][e];
    }
}

// The parts' sums at their common maximum, over the sum of the weights; of two maps the difference, and the head's norm.  A row that sees
// nothing is zero.  Bound by latency: WAVES waves a row, each with every WAVES-th eight parts, whose sums are asked for at once
// (one wave and one part at a time took 46 us for 840 rows of 68 parts, this 6).
constexpr int MERGE_AT_ONCE = 8;
template <int MAPS, int WAVES> __global__ __launch_bounds__(256) void span_merge_kernel(SpanCall c) {
    constexpr int E = SPAN_MAX_D / 64;
    __shared__ float s_part[4][MAPS][SPAN_MAX_D + 2];
    const vq_store_attend_args &a = c.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
    if (row >= a.B * a.Hq * a.Sq) return;   // (the whole block where waves share a row)
    const int D = (int)a.D;
    const float *ml = c.ml + row * c.nparts * MAPS * 2, *sums = c.sums + row * c.nparts * MAPS * D;
    float num[MAPS][E], m[MAPS], l[MAPS];
#pragma unroll
    for (int w = 0; w < MAPS; ++w) {
        m[w] = -INFINITY; l[w] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) num[w][e] = 0.f;
        for (int p0 = wave % WAVES * MERGE_AT_ONCE; p0 < c.nparts; p0 += WAVES * MERGE_AT_ONCE) {
            float2 x[MERGE_AT_ONCE];
            float y[MERGE_AT_ONCE][E];
#pragma unroll
            for (int p = 0; p < MERGE_AT_ONCE; ++p) {
                const int at = (p0 + p < c.nparts ? p0 + p : p0) * MAPS + w;
                x[p] = *(const float2 *)(ml + at * 2);
#pragma unroll
                for (int e = 0; e < E; ++e) y[p][e] = lane + 64 * e < D ? sums[(int64_t)at * D + lane + 64 * e] : 0.f;
            }
            float mn = m[w];
#pragma unroll
            for (int p = 0; p < MERGE_AT_ONCE; ++p) mn = fmaxf(mn, x[p].x);
#pragma unroll
            for (int p = 0; p < MERGE_AT_ONCE; ++p) l[w] = x[p].y != x[p].y ? x[p].y : l[w];   // (a row of NaN has no maximum)
            if (mn == -INFINITY) continue;   // (parts without a visible slot: their sums are not written)
            const float f = exp2f(m[w] - mn);
            m[w] = mn;
            l[w] *= f;
#pragma unroll
            for (int e = 0; e < E; ++e) num[w][e] *= f;
#pragma unroll
            for (int p = 0; p < MERGE_AT_ONCE; ++p) {
                if (p0 + p >= c.nparts || x[p].x == -INFINITY) continue;
                const float by = exp2f(x[p].x - mn);
                l[w] = __builtin_fmaf(by, x[p].y, l[w]);
#pragma unroll
                for (int e = 0; e < E; ++e) num[w][e] = __builtin_fmaf(by, y[p][e], num[w][e]);
            }
        }
    }
    if (WAVES > 1) {
#pragma unroll
        for (int w = 0; w < MAPS; ++w) {
            if (lane == 0) { s_part[wave][w][0] = m[w]; s_part[wave][w][1] = l[w]; }
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (lane + 64 * e < D) s_part[wave][w][2 + lane + 64 * e] = num[w][e];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 0; w < MAPS; ++w)
            for (int v = 1; v < WAVES; ++v) {
                const float *o = s_part[v][w], mn = fmaxf(m[w], o[0]);
                if (o[1] != o[1]) l[w] = o[1];
                if (mn == -INFINITY) continue;
                const float f = exp2f(m[w] - mn), by = exp2f(o[0] - mn);
                m[w] = mn;
                l[w] = l[w] * f + o[1] * by;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (lane + 64 * e < D) num[w][e] = num[w][e] * f + o[2 + lane + 64 * e] * by;
            }
    }
    float o[E];
#pragma unroll
    for (int w = 0; w < MAPS; ++w) {
        const float by = l[w] > 0.f || l[w] != l[w] ? (w == 0 ? 1.f : -span_lam(a, row / a.Sq % a.Hq)) / l[w] : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = w == 0 ? num[0][e] * by : __builtin_fmaf(num[w][e], by, o[e]);
    }
    if (MAPS == 2) {
        float gain = a.gain;
        if (a.norm_weight != nullptr) {
            float sq = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) sq = __builtin_fmaf(o[e], o[e], sq);
            gain /= sqrtf(span_wave_sum(sq) / (float)D + a.norm_eps);
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            o[e] *= a.norm_weight != nullptr && lane + 64 * e < D ? gain * span_ld(a.norm_weight, a.norm_dtype, lane + 64 * e) : gain;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 64 * e < D) span_st(a.out, a.dtype, row * D + lane + 64 * e, o[e]);
}

int check_store(const char *fn, const char *which, const vq_store_attend_args &a, const vq_kv_store &s) {
    VQ_REQUIRE(s.n_packed >= 0 && s.n_tail >= 0, VQ_ERR_INVALID, "%s: negative token count (%s)", fn, which);
    if (s.n_packed > 0) {
        VQ_REQUIRE(s.k_packed && s.k_scale && s.k_zero && s.v_packed && s.v_scale && s.v_zero, VQ_ERR_INVALID, "%s: null packed pointer (%s)", fn, which);
        VQ_REQUIRE(a.pack_bits >= 1 && a.pack_bits <= 8, VQ_ERR_INVALID, "%s: pack_bits must be in 1..8", fn);
        VQ_REQUIRE(a.group >= 1, VQ_ERR_INVALID, "%s: group_size must be >= 1", fn);
        VQ_REQUIRE(a.meta_dtype == VQ_F32 || a.meta_dtype == VQ_F16, VQ_ERR_INVALID, "%s: meta dtype must be f32/f16", fn);
        VQ_REQUIRE(a.v_layout == VQ_V_CHANNEL_PACKED || a.v_layout == VQ_V_TOKEN_PACKED, VQ_ERR_INVALID, "%s: bad v_layout", fn);
        VQ_REQUIRE(s.cap_tokens >= s.n_packed, VQ_ERR_INVALID, "%s: n_packed exceeds cap_tokens (%s)", fn, which);
        VQ_REQUIRE(a.v_layout != VQ_V_TOKEN_PACKED || s.cap_tokens % (32 / a.pack_bits) == 0, VQ_ERR_INVALID, "%s: cap_tokens not word aligned (%s)", fn, which);
    }
    if (s.n_tail > 0) {
        VQ_REQUIRE(s.k_tail && s.v_tail, VQ_ERR_INVALID, "%s: null tail pointer (%s)", fn, which);
        VQ_REQUIRE(is_float_tag(a.tail_dtype), VQ_ERR_INVALID, "%s: unsupported tail dtype", fn);
    }
    return VQ_OK;
}

int check_call(const char *fn, const vq_store_attend_args *args, int maps) {
    VQ_REQUIRE(args != nullptr, VQ_ERR_INVALID, "%s: null argument block", fn);
    const vq_store_attend_args &a = *args;
    VQ_REQUIRE(a.B >= 1 && a.Hq >= 1 && a.Hkv >= 1 && a.Sq >= 1 && a.D >= 1, VQ_ERR_INVALID, "%s: bad sizes", fn);
    VQ_REQUIRE(a.D <= SPAN_MAX_D, VQ_ERR_INVALID, "%s: D=%lld must be <= %d", fn, (long long)a.D, SPAN_MAX_D);
    VQ_REQUIRE(a.Hq % a.Hkv == 0, VQ_ERR_INVALID, "%s: H_q=%lld must be a multiple of H_kv=%lld", fn, (long long)a.Hq, (long long)a.Hkv);
    VQ_REQUIRE(is_float_tag(a.dtype), VQ_ERR_INVALID, "%s: unsupported q/out dtype", fn);
    if (int rc = check_store(fn, "prefix", a, a.prefix)) return rc;
    if (int rc = check_store(fn, "own", a, a.own)) return rc;
    const int64_t slots = span_prefix_slots(a) + a.own.n_packed + a.own.n_tail;
    VQ_REQUIRE(slots >= 1, VQ_ERR_INVALID, "%s: no key/value slots to attend to", fn);
    VQ_REQUIRE(slots < (INT64_C(1) << 30) && a.Sq < (INT64_C(1) << 30), VQ_ERR_UNSUPPORTED, "%s: more than 2^30 slots or queries a sequence", fn);
    // (up to a block a row in the merge, 2^32 threads a launch at most)
    VQ_REQUIRE(a.B < (INT64_C(1) << 24) && a.Hq < (INT64_C(1) << 24) && a.B * a.Hq < (INT64_C(1) << 24) && a.B * a.Hq * a.Sq < (INT64_C(1) << 24),
               VQ_ERR_UNSUPPORTED, "%s: 2^24 or more query rows", fn);
    VQ_REQUIRE(!a.causal || a.Sq <= slots, VQ_ERR_INVALID, "%s: S_q=%lld exceeds the %lld slots; queries align to their end", fn, (long long)a.Sq, (long long)slots);
    VQ_REQUIRE(a.sliding_window >= 0, VQ_ERR_INVALID, "%s: negative sliding window", fn);
    VQ_REQUIRE(a.q != nullptr && a.out != nullptr, VQ_ERR_INVALID, "%s: null q or out", fn);
    if (maps == 2) {
        VQ_REQUIRE(a.D % 2 == 0, VQ_ERR_INVALID, "%s: D=%lld holds two halves and must be even", fn, (long long)a.D);
        VQ_REQUIRE(span_prefix_slots(a) == 0, VQ_ERR_INVALID, "%s: takes no shared prefix", fn);
        VQ_REQUIRE(a.lam != nullptr && (a.lam_stride == 0 || a.lam_stride == 1), VQ_ERR_INVALID, "%s: lam must be given, one value or one a head", fn);
        VQ_REQUIRE(a.norm_weight == nullptr || is_float_tag(a.norm_dtype), VQ_ERR_INVALID, "%s: unsupported norm weight dtype", fn);
    }
    return VQ_OK;
}

SpanCall cut(const vq_store_attend_args &a, int maps) {
    SpanCall c = {};
    c.a = a;
    // fields that no packed slot reads
    if (a.prefix.n_packed == 0 && a.own.n_packed == 0) { c.a.pack_bits = 8; c.a.group = 1; }
    if (span_mfma_supported(c.a)) {
        span_mfma_plan(c, maps);
        return c;
    }
    // as many waves as fill the chip eight deep, runs of 64 slots or more
    const int64_t rows = a.B * a.Hq * a.Sq, slots = span_prefix_slots(a) + a.own.n_packed + a.own.n_tail;
    int64_t parts = 8192 / rows;
    if (parts > cdiv(slots, 64)) parts = cdiv(slots, 64);
    c.nparts = (int)(parts < 1 ? 1 : parts);
    return c;
}

// (the sums take whole 16 bytes, so that the pairs (m, l) behind them, read and written whole, are aligned with odd heads too)
int64_t scratch_floats(const SpanCall &c, int maps, int64_t &sums) {
    const int64_t recs = c.a.B * c.a.Hq * c.a.Sq * c.nparts * maps;
    sums = cdiv(recs * c.a.D, 4) * 4;
    return sums + recs * 2;
}

size_t workspace(const char *fn, const vq_store_attend_args *args, int maps) {
    if (check_call(fn, args, maps) != VQ_OK) return 0;
    const SpanCall c = cut(*args, maps);
    if (c.nparts == 1 && span_mfma_supported(c.a)) return 0;
    int64_t sums;
    return (size_t)scratch_floats(c, maps, sums) * 4;
}

template <int MAPS> int attend(const char *fn, const vq_store_attend_args *args) {
    if (int rc = check_call(fn, args, MAPS)) return rc;
    SpanCall c = cut(*args, MAPS);
    const vq_store_attend_args &a = c.a;
    const bool mfma = span_mfma_supported(a), direct = mfma && c.nparts == 1;
    const int64_t rows = a.B * a.Hq * a.Sq;
    hipStream_t st = (hipStream_t)a.stream;
    if (!direct) {
        int64_t sums;
        const size_t need = (size_t)scratch_floats(c, MAPS, sums) * 4;
        VQ_REQUIRE(a.workspace != nullptr && a.workspace_bytes >= need && ((uintptr_t)a.workspace & 15) == 0, VQ_ERR_WORKSPACE,
                   "%s: workspace of %zu bytes required, 16-byte aligned", fn, need);
        c.sums = (float *)a.workspace;
        c.ml = c.sums + sums;
    }
    if (mfma) {
        if (int rc = launch_span_mfma(c, MAPS)) return rc;
    } else {
        const int64_t waves = rows * c.nparts;   // (at most 8192, or one a row)
        span_any_kernel<MAPS><<<(unsigned)cdiv(waves, 4), 256, 0, st>>>(c);
        VQ_HIP_CHECK_LAUNCH(fn);
    }
    if (!direct) {
        // (a row to a block where its parts are many, or rows too few to fill the chip with a wave each: 512 rows of 16 parts and two maps 9.8 us, a
        // wave each 11.1; 1920 rows of 11 parts 7.0, a wave each 5.2)
        if (c.nparts > 2 * MERGE_AT_ONCE || (c.nparts > MERGE_AT_ONCE && rows < 1024)) span_merge_kernel<MAPS, 4><<<(unsigned)rows, 256, 0, st>>>(c);
        else span_merge_kernel<MAPS, 1><<<(unsigned)cdiv(rows, 4), 256, 0, st>>>(c);
        VQ_HIP_CHECK_LAUNCH(fn);
    }
    return VQ_OK;
}

}  // namespace

}  // namespace vq

extern "C" size_t vq_shared_prefix_attend_workspace(const vq_store_attend_args *a) { return vq::workspace("vq_shared_prefix_attend", a, 1); }
extern "C" int vq_shared_prefix_attend(const vq_store_attend_args *a) { return vq::attend<1>("vq_shared_prefix_attend", a); }
extern "C" size_t vq_differential_attend_workspace(const vq_store_attend_args *a) { return vq::workspace("vq_differential_attend", a, 2); }
extern "C" int vq_differential_attend(const vq_store_attend_args *a) { return vq::attend<2>("vq_differential_attend", a); }
