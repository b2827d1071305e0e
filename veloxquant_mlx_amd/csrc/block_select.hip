// The blocks of packed keys that a query attends to, chosen by a bound on its scores.
//
// A group of packed keys lies in channel c between zero_c and zero_c + L scale_c (L the top code), so no key of it has a product
// with a query above  sum_c max(q_c zero_c, q_c (zero_c + L scale_c)).  A block's score is the largest such bound over its groups, over
// the query heads of the kv head and over the queries of a tile, which choose together; the bounds are what the store keeps anyway.
//
// Which blocks are chosen must not hang on the order of a sum, so scores are formed in 64 bits: products of two 24-bit numbers and a
// code are exact there, and the sum of a head's channels is good to 1e-15 of its terms.  Equal scores: the lower block first.
//
// The chosen ones come out in ascending order, -1 behind them where fewer are visible: the first `first` and the last `recent` visible
// blocks always, the others by score.
#include "common.hpp"

namespace vq {

namespace {

struct SelectCall {
    vq_block_select_args a;
    int64_t tiles, total;   // tiles of queries a sequence, blocks of the store
    double *scores;         // [B][Hkv][tiles][total]
};

__device__ __forceinline__ float sel_ld(const void *p, int tag, int64_t i) {
    if (tag == VQ_F16) return (float)((const f16 *)p)[i];
    if (tag == VQ_BF16) return bf16_to_f32(((const u16 *)p)[i]);
    return ((const float *)p)[i];
}

// slots [0, end) of the packed ones that query i of sequence b sees
__device__ __forceinline__ int64_t sel_end(const vq_block_select_args &a, int64_t b, int64_t i) {
    const int64_t room = a.n_packed + a.n_tail;
    int64_t live = a.seq_lens == nullptr ? room : a.seq_lens[b];
    live = live < 0 ? 0 : live < room ? live : room;
    int64_t end = a.causal ? live - a.Sq + i + 1 : live;
    end = end < live ? end : live;
    return end < 0 ? 0 : end < a.n_packed ? end : a.n_packed;
}
__device__ __forceinline__ int64_t sel_last(const vq_block_select_args &a, int64_t tile) {
    const int64_t last = (tile + 1) * a.query_block;
    return (last < a.Sq ? last : a.Sq) - 1;
}

// A wave a (tile, block): lanes along the channels.
__global__ __launch_bounds__(256) void block_score_kernel(SelectCall c) {
    const vq_block_select_args &a = c.a;
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= a.B * a.Hkv * c.tiles * c.total) return;
    const int64_t j = id % c.total, tile = id / c.total % c.tiles, bh = id / (c.total * c.tiles), hkv = bh % a.Hkv, b = bh / a.Hkv;
    const int64_t G = a.Hq / a.Hkv, i1 = sel_last(a, tile), groups = (a.cap_tokens + a.group - 1) / a.group;
    double best = -INFINITY;
    for (int64_t t = j * a.block_tokens; t < (j + 1) * a.block_tokens; t += a.group)
        for (int64_t i = tile * a.query_block; i <= i1; ++i) {
            if (t >= sel_end(a, b, i)) continue;
            for (int64_t g = 0; g < G; ++g) {
                double s = 0.;
                for (int64_t d = lane; d < a.D; d += 64) {
                    const int64_t at = (bh * groups + t / a.group) * a.D + d;
                    const double q = sel_ld(a.q, a.dtype, ((b * a.Hq + hkv * G + g) * a.Sq + i) * a.D + d);
                    const double z = sel_ld(a.k_zero, a.meta_dtype, at), r = q * (double)sel_ld(a.k_scale, a.meta_dtype, at) * a.levels;
                    s += q * z + (r > 0. ? r : r != r ? r : 0.);
                }
#pragma unroll
                for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
                best = s > best || s != s ? s : best;
            }
        }
    if (lane == 0) c.scores[id] = best;
}

// A block of threads a tile: the least score among the chosen by a radix select over the scores' bits, then the chosen in order.
constexpr int PICK_THREADS = 256;
__device__ __forceinline__ uint64_t pick_key(double s) {   // ascending with the score, NaN above all
    if (s != s) return ~UINT64_C(0);
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.);
    return u >> 63 ? ~u : u | (UINT64_C(1) << 63);
}
__global__ __launch_bounds__(PICK_THREADS) void block_pick_kernel(SelectCall c) {
    const vq_block_select_args &a = c.a;
    __shared__ uint32_t hist[256];
    __shared__ uint32_t waves[2][PICK_THREADS / 64];
    __shared__ uint64_t s_key;
    __shared__ int64_t s_left;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x, tile = row % c.tiles, b = row / c.tiles / a.Hkv;
    const int64_t V = (sel_end(a, b, sel_last(a, tile)) + a.block_tokens - 1) / a.block_tokens;
    int32_t *out = a.out + row * a.count;
    if (V <= a.count) {
        for (int64_t i = tid; i < a.count; i += PICK_THREADS) out[i] = i < V ? (int32_t)i : -1;
        return;
    }
    const double *score = c.scores + row * c.total;
    const int64_t lo = a.first, hi = V - a.recent, want = a.count - a.first - a.recent;   // of [lo, hi)
    for (int64_t i = tid; i < a.first; i += PICK_THREADS) out[i] = (int32_t)i;
    for (int64_t i = tid; i < a.recent; i += PICK_THREADS) out[a.count - a.recent + i] = (int32_t)(hi + i);
    if (want == 0) return;
    uint64_t key = 0;
    int64_t left = want;   // how many of those that share the key's upper bits
    for (int shift = 56; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int64_t j = lo + tid; j < hi; j += PICK_THREADS) {
            const uint64_t k = pick_key(score[j]);
            if (shift == 56 || (k ^ key) >> (shift + 8) == 0) atomicAdd(&hist[k >> shift & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            int64_t above = 0;
            int digit = 255;
            while (digit > 0 && above + hist[digit] < left) above += hist[digit--];
            s_key = key | (uint64_t)digit << shift;
            s_left = left - above;
        }
        __syncthreads();
        key = s_key;
        left = s_left;
    }
    // those above the key, and the first `left` of those that equal it
    int64_t done = 0, equal = 0;
    for (int64_t j0 = lo; j0 < hi; j0 += PICK_THREADS) {
        const int64_t j = j0 + tid;
        const uint64_t k = j < hi ? pick_key(score[j]) : 0;
        const bool eq = j < hi && k == key, gt = j < hi && k > key;
        const uint64_t e = __ballot(eq), below = (UINT64_C(1) << lane) - 1;
        if (lane == 0) waves[0][wave] = (uint32_t)__popcll(e);
        __syncthreads();
        int64_t rank = equal + __popcll(e & below);
        for (int w = 0; w < PICK_THREADS / 64; ++w) {
            if (w < wave) rank += waves[0][w];
            equal += waves[0][w];
        }
        const bool take = gt || (eq && rank < left);
        const uint64_t m = __ballot(take);
        if (lane == 0) waves[1][wave] = (uint32_t)__popcll(m);
        __syncthreads();
        int64_t at = done + __popcll(m & below);
        for (int w = 0; w < PICK_THREADS / 64; ++w) {
            if (w < wave) at += waves[1][w];
            done += waves[1][w];
        }
        if (take) out[lo + at] = (int32_t)j;
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
    VQ_REQUIRE(rows * (double)cdiv(a.n_packed, a.block_tokens) < 67108864., VQ_ERR_UNSUPPORTED, "%s: 2^26 or more scores", fn);
    VQ_REQUIRE(a.q != nullptr && a.out != nullptr && (a.n_packed == 0 || (a.k_scale != nullptr && a.k_zero != nullptr)), VQ_ERR_INVALID,
               "%s: null q, out, scale or zero", fn);
    return VQ_OK;
}

SelectCall cut_select(const vq_block_select_args &a) {
    SelectCall c = {};
    c.a = a;
    c.tiles = cdiv(a.Sq, a.query_block);
    c.total = cdiv(a.n_packed, a.block_tokens);
    return c;
}
size_t select_bytes(const SelectCall &c) { return c.total <= c.a.count ? 0 : (size_t)(c.a.B * c.a.Hkv * c.tiles * c.total) * 8; }

}  // namespace

}  // namespace vq

extern "C" size_t vq_block_select_workspace(const vq_block_select_args *args) {
    using namespace vq;
    if (check_select("vq_block_select", args) != VQ_OK) return 0;
    return select_bytes(cut_select(*args));
}

extern "C" int vq_block_select(const vq_block_select_args *args) {
    using namespace vq;
    const char *fn = "vq_block_select";
    if (int rc = check_select(fn, args)) return rc;
    SelectCall c = cut_select(*args);
    const vq_block_select_args &a = c.a;
    const size_t need = select_bytes(c);
    VQ_REQUIRE(need == 0 || (a.workspace != nullptr && a.workspace_bytes >= need && ((uintptr_t)a.workspace & 15) == 0), VQ_ERR_WORKSPACE,
               "%s: workspace of %zu bytes required, 16-byte aligned", fn, need);
    c.scores = (double *)a.workspace;
    hipStream_t st = (hipStream_t)a.stream;
    const int64_t rows = a.B * a.Hkv * c.tiles;
    if (need > 0) {
        block_score_kernel<<<(unsigned)cdiv(rows * c.total, 4), 256, 0, st>>>(c);
        VQ_HIP_CHECK_LAUNCH(fn);
    }
    block_pick_kernel<<<(unsigned)rows, PICK_THREADS, 0, st>>>(c);
    VQ_HIP_CHECK_LAUNCH(fn);
    return VQ_OK;
}
