// Attention of a row over up to four spans of slots -- the packed and the plain slots of a prefix that all sequences share,
// then those of the row's own sequence -- with one softmax map a head or two (differential attention).
//
// The slots of a sequence lie one behind the other: prefix packed, prefix plain, own packed, own plain.  A query at position i
// of Sq aligns to the end: with n live slots in all it sees slots below n - Sq + i + 1 (causal) or n, and under a sliding window
// those from n - Sq + i + 1 - window on.  A packed slot stands for the fp16 number code * scale + zero.
#pragma once
#include "attend_mfma.hpp"

namespace vq {

constexpr int SPAN_MAX_D = 256;

// A call and how it is cut.  Every kernel writes partials -- per (query row, part, map) the sums of exp2(s - m) v over its
// slots, and (m, the sum of exp2(s - m)), m in log2 units -- unless there is one part a row, where it writes the output.
struct SpanCall {
    vq_store_attend_args a;
    int nparts;            // parts a row
    int psplits, osplits;  // runs of the prefix / of a sequence's own slots (MFMA: see attend_span_mfma.hpp)
    int ptiles, otiles;    // row tiles of the prefix / of a sequence
    int pwt, owt;          // waves that share a row (1 or 2), each with its half of every unit
    int pfew, ofew;        // 1: that side by the kernel for few rows (attend_span_few.hpp)
    int owaves;            // waves of a block of that kernel: 4, or 8 (own slots and prefix together, one part)
    int apart;             // 1: prefix and own slots belong to different blocks; 0: the blocks of a row walk both
    float *sums;           // [rows][nparts][maps][D]
    float *ml;             // [rows][nparts][maps][2]
};

// Lists of blocks of packed slots (attend_blocks.hip), one a tile of queries of a kv head, in units of 32 slots for the kernel for few rows: a
// list's unit v is unit v % sub of its entry v / sub, then come the tail's.
struct BlockLists {
    const int32_t *blocks;          // [B][Hkv][tiles][count]
    int tiles, count;               // lists a kv head, entries a list
    int block_tokens, query_block;
    int total;                      // blocks of the store
    int sub, packed_units, units;   // units of an entry, of a list, and with the tail
    int run, longer;                // units of a run, and how many runs have one more
    int row_tiles;                  // tiles of rows of a tile of queries
    int32_t *counters;              // zeros, one a tile of rows: the last block of a tile adds up its parts; NULL: another launch does
};
constexpr int BLOCK_UNITS = 1024;   // units of a list that a block of threads walks, at most

__device__ __forceinline__ int64_t span_own_live(const vq_store_attend_args &a, int64_t b) {
    const int64_t room = a.own.n_packed + a.own.n_tail;
    if (a.seq_lens == nullptr) return room;
    const int64_t n = a.seq_lens[b];
    return n < 0 ? 0 : n < room ? n : room;
}
__device__ __host__ __forceinline__ int64_t span_prefix_slots(const vq_store_attend_args &a) { return a.prefix.n_packed + a.prefix.n_tail; }
// slots [lo, hi) that the query at position `pos` sees of `total` live ones
__device__ __forceinline__ void span_visible(const vq_store_attend_args &a, int64_t total, int64_t pos, int64_t &lo, int64_t &hi) {
    const int64_t end = total - a.Sq + pos + 1;
    hi = a.causal ? (end < 0 ? 0 : end) : total;
    lo = a.sliding_window > 0 && end > a.sliding_window ? end - a.sliding_window : 0;
}
__device__ __forceinline__ float span_ld(const void *p, int tag, int64_t i) {
    if (tag == VQ_F16) return (float)((const f16 *)p)[i];
    if (tag == VQ_BF16) return bf16_to_f32(((const u16 *)p)[i]);
    return ((const float *)p)[i];
}
__device__ __forceinline__ void span_st(void *p, int tag, int64_t i, float v) {
    if (tag == VQ_F16) ((f16 *)p)[i] = (f16)v;
    else if (tag == VQ_BF16) ((u16 *)p)[i] = f32_to_bf16(v);
    else ((float *)p)[i] = v;
}
__device__ __forceinline__ float span_wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}
__device__ __forceinline__ float span_lam(const vq_store_attend_args &a, int64_t h) { return a.lam[h * a.lam_stride]; }

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
    static __device__ __forceinline__ SpanPacked of(const vq_store_attend_args &a, const vq_kv_store &s) {
        const int per = 32 / a.pack_bits;
        auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
        return {&s, a.pack_bits, per, a.group, a.meta_dtype, a.v_layout, (1u << a.pack_bits) - 1u, a.D, up(a.D, per), up(a.D, a.group),
                up(s.cap_tokens, a.group)};
    }
};

// the checks of a call, the merge of the parts of rows of one map (attend_span.hip)
int span_check_call(const char *fn, const vq_store_attend_args *args, int maps);
int launch_span_merge1(const char *fn, const SpanCall &c);

// whether the matrix-unit kernel takes the call, its cut, its launch (attend_span_mfma.hip)
bool span_mfma_supported(const vq_store_attend_args &a);
void span_mfma_plan(SpanCall &c, int maps);
int launch_span_mfma(const SpanCall &c, int maps);

}  // namespace vq
