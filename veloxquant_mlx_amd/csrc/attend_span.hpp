// Attention of a row over up to four spans of slots -- the packed and the plain slots of a prefix that all sequences share,
// then those of the row's own sequence -- with one softmax map a head or two (differential attention).
//
// The slots of a sequence lie one behind the other: prefix packed, prefix plain, own packed, own plain.  A query at position i
// of Sq aligns to the end: with n live slots in all it sees slots below n - Sq + i + 1 (causal) or n, and under a sliding window
// those from n - Sq + i + 1 - window on.  A packed slot stands for the fp16 number code * scale + zero.
#pragma once
#include "attend_mfma.hpp"

namespace vq {

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

// whether the matrix-unit kernel takes the call, its cut, its launch (attend_span_mfma.hip)
bool span_mfma_supported(const vq_store_attend_args &a);
void span_mfma_plan(SpanCall &c, int maps);
int launch_span_mfma(const SpanCall &c, int maps);

}  // namespace vq
