// Rotary positions of queries and keys in one launch.
//
// Channel pair i of a row at position p turns by the angle t = p w_i:
//   (a, b) -> f (a cos t - b sin t, b cos t + a sin t)        (inverse: -t)
// with a, b channels i and i + r/2 (half layout) or 2i and 2i + 1 (interleaved); channels r .. D - 1 pass through.
//
// A far position loses its angle in float32 (p = 10^6 at w = 1: 0.03 rad of error), so the angle is formed in double and
// reduced to a part of a turn there: t / 2 pi = p (w / 2 pi), of which the nearest integer is taken away; what is left, in
// [-1/2, 1/2], is rounded to float32 (2^-26 of a turn at most, 1e-7 rad) and goes through sincospif.  The turn itself is
// float32 and rounded once to the element type.
//
// Bound by memory: every row is read and written once.  A thread holds the sines and cosines of one 16-byte piece of the
// head at one position (both halves' pieces in the half layout) and walks over the heads, queries then keys, four rows in
// flight, so the double arithmetic (~500 instructions of a piece of eight pairs) is paid once for all heads of a thread.
// Threads of a wave lie along the head, then along the tokens: contiguous rows for [B, H, S, D] tensors, whole rows of 128
// bytes or more for views of [B, S, H, D] projections, which is how the transpose costs nothing.  Heads are dealt to more
// threads only while the launch would not fill the chip.
#include "common.hpp"

namespace vq {

namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_FLIGHT = 4;              // rows a thread has in flight
constexpr int64_t RT_FILL = 256 * 1024;   // threads that fill the chip: 16 waves a CU

struct RotaryCall {
    vq_rotary_args a;
    int units, rot_units;   // threads along a row, of which the first rot_units turn a piece and the others copy one
    int heads_per_thread;
};

template <typename T, int N> struct alignas(sizeof(T) * N) Piece { T v[N]; };

// N channels a piece (1: any strides and alignment)
template <typename T, int N, bool HALF> __global__ __launch_bounds__(RT_THREADS) void rotary_kernel(RotaryCall c) {
    const vq_rotary_args &a = c.a;
    constexpr int PAIRS = HALF || N == 1 ? N : N / 2;
    // the block's first (position, piece) in 64 bits, this thread's distance from it in 32
    const int64_t base = (int64_t)blockIdx.x * RT_THREADS;
    const int64_t tok0 = base / c.units;
    const uint32_t at = (uint32_t)(base - tok0 * c.units) + threadIdx.x;
    const int u = (int)(at % (uint32_t)c.units);
    const int64_t tok = tok0 + at / (uint32_t)c.units;
    if (tok >= a.B * a.S) return;
    const int64_t b = tok / a.S, s = tok - b * a.S;
    const bool turns = u < c.rot_units;
    // the two pieces of the row (the second only where the layout keeps pairs apart): channel of each
    int64_t c0, c1 = 0;
    bool second = false;
    if (turns) {
        if (HALF) { c0 = (int64_t)u * N; c1 = c0 + a.dims / 2; second = true; }
        else if (N == 1) { c0 = 2 * (int64_t)u; c1 = c0 + 1; second = true; }
        else c0 = (int64_t)u * N;
    } else {
        c0 = a.dims + (int64_t)(u - c.rot_units) * N;
    }
    float cs[PAIRS], sn[PAIRS];
    if (turns) {
        int64_t p = a.offset + (a.add_index ? s : 0);
        if (a.positions != nullptr) {
            const int64_t i = b * a.pos_stride_b + s * a.pos_stride_s;
            p += a.pos_dtype == VQ_I64 ? ((const int64_t *)a.positions)[i] : ((const int32_t *)a.positions)[i];
        }
        const double place = (double)p * 0.15915494309189533577;   // turns per radian
        const int64_t i0 = (HALF || N == 1) ? (int64_t)u * N : (int64_t)u * (N / 2);
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            const double w = a.freq_dtype == VQ_F64 ? ((const double *)a.inv_freq)[i0 + j] : (double)((const float *)a.inv_freq)[i0 + j];
            const double r = place * w;
            sincospif(2.f * (float)(r - rint(r)), &sn[j], &cs[j]);
            cs[j] *= a.attention_factor;
            sn[j] *= a.inverse ? -a.attention_factor : a.attention_factor;
        }
    }
    using P = Piece<T, N>;
    auto turn = [&](P &x0, P &x1) {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            T *pa = HALF || N == 1 ? &x0.v[j] : &x0.v[2 * j], *pb = HALF || N == 1 ? &x1.v[j] : &x0.v[(2 * j + 1) % N];
            const float xa = Elem<T>::ld(pa), xb = Elem<T>::ld(pb);
            Elem<T>::st(pa, __builtin_fmaf(xa, cs[j], -(xb * sn[j])));
            Elem<T>::st(pb, __builtin_fmaf(xb, cs[j], xa * sn[j]));
        }
    };
    const int64_t h0 = (int64_t)blockIdx.y * c.heads_per_thread;
    const int64_t h1 = h0 + c.heads_per_thread < a.heads[0] + a.heads[1] ? h0 + c.heads_per_thread : a.heads[0] + a.heads[1];
    for (int64_t h = h0; h < h1; h += RT_FLIGHT) {
        P x0[RT_FLIGHT], x1[RT_FLIGHT];
        T *to[RT_FLIGHT];
#pragma unroll
        for (int k = 0; k < RT_FLIGHT; ++k) {
            const int64_t hh = h + k < h1 ? h + k : h;   // (a group's missing heads read its first again)
            const int w = hh >= a.heads[0];
            const int64_t head = hh - (w ? a.heads[0] : 0);
            const T *from = (const T *)a.x[w] + b * a.x_strides[w][0] + head * a.x_strides[w][1] + s * a.x_strides[w][2];
            to[k] = (T *)a.out[w] + b * a.out_strides[w][0] + head * a.out_strides[w][1] + s * a.out_strides[w][2];
            x0[k] = *(const P *)(from + c0);
            if (second) x1[k] = *(const P *)(from + c1);
        }
#pragma unroll
        for (int k = 0; k < RT_FLIGHT; ++k) {
            if (h + k >= h1) break;
            if (turns) turn(x0[k], x1[k]);
            *(P *)(to[k] + c0) = x0[k];
            if (second) *(P *)(to[k] + c1) = x1[k];
        }
    }
}

template <typename T> int launch_rotary(const vq_rotary_args &a, hipStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    RotaryCall c;
    c.a = a;
    const bool half = a.layout == VQ_ROTARY_HALF;
    const int heads = (int)(a.heads[0] + a.heads[1]);
    // 16-byte pieces where every row of every tensor is aligned for them and no pair is cut
    bool wide = a.D % N == 0 && (half ? a.dims / 2 : a.dims) % N == 0;
    bool in_place = true;
    for (int w = 0; w < 2; ++w) {
        if (a.heads[w] == 0) continue;
        wide = wide && (((uintptr_t)a.x[w] | (uintptr_t)a.out[w]) & 15) == 0;
        in_place = in_place && a.x[w] == a.out[w];
        for (int d = 0; d < 3; ++d) wide = wide && a.x_strides[w][d] % N == 0 && a.out_strides[w][d] % N == 0;
    }
    const int n = wide ? N : 1;
    c.rot_units = (int)(half ? a.dims / 2 / n : n == 1 ? a.dims / 2 : a.dims / n);
    c.units = c.rot_units + (in_place ? 0 : (int)((a.D - a.dims) / n));   // nothing to copy in place
    const int64_t threads = a.B * a.S * c.units;
    VQ_REQUIRE(threads < (INT64_C(1) << 32) - RT_THREADS, VQ_ERR_UNSUPPORTED, "vq_rotary: too many rows for one launch");
    c.heads_per_thread = heads;
    while (c.heads_per_thread > 1 && threads * cdiv(heads, c.heads_per_thread) < RT_FILL)
        c.heads_per_thread = c.heads_per_thread > RT_FLIGHT ? (int)cdiv(cdiv(c.heads_per_thread, 2), RT_FLIGHT) * RT_FLIGHT
                                                           : c.heads_per_thread / 2;
    const dim3 grid((unsigned)cdiv(threads, RT_THREADS), (unsigned)cdiv(heads, c.heads_per_thread));
    if (wide && half) rotary_kernel<T, N, true><<<grid, RT_THREADS, 0, st>>>(c);
    else if (wide) rotary_kernel<T, N, false><<<grid, RT_THREADS, 0, st>>>(c);
    else if (half) rotary_kernel<T, 1, true><<<grid, RT_THREADS, 0, st>>>(c);
    else rotary_kernel<T, 1, false><<<grid, RT_THREADS, 0, st>>>(c);
    VQ_HIP_CHECK_LAUNCH("vq_rotary");
    return VQ_OK;
}

}  // namespace

}  // namespace vq

extern "C" int vq_rotary(const vq_rotary_args *args, void *stream) {
    using namespace vq;
    VQ_REQUIRE(args != nullptr, VQ_ERR_INVALID, "vq_rotary: no arguments");
    const vq_rotary_args &a = *args;
    VQ_REQUIRE(is_float_tag(a.dtype), VQ_ERR_INVALID, "vq_rotary: unsupported dtype tag %d", a.dtype);
    VQ_REQUIRE(a.B >= 0 && a.S >= 0 && a.D >= 1 && a.heads[0] >= 0 && a.heads[1] >= 0, VQ_ERR_INVALID, "vq_rotary: bad sizes");
    VQ_REQUIRE(a.dims >= 2 && a.dims % 2 == 0 && a.dims <= a.D, VQ_ERR_INVALID,
               "vq_rotary: dims=%lld must be even, at least 2 and at most the head size %lld", (long long)a.dims, (long long)a.D);
    VQ_REQUIRE(a.layout == VQ_ROTARY_HALF || a.layout == VQ_ROTARY_INTERLEAVED, VQ_ERR_INVALID, "vq_rotary: unknown layout %d", a.layout);
    VQ_REQUIRE(a.freq_dtype == VQ_F64 || a.freq_dtype == VQ_F32, VQ_ERR_INVALID, "vq_rotary: frequencies must be float64 or float32");
    VQ_REQUIRE(a.positions == nullptr || a.pos_dtype == VQ_I32 || a.pos_dtype == VQ_I64, VQ_ERR_INVALID,
               "vq_rotary: positions must be int32 or int64");
    const int64_t heads = a.heads[0] + a.heads[1];
    VQ_REQUIRE(heads <= 65535 && a.D <= 65536 && a.S < (INT64_C(1) << 31), VQ_ERR_UNSUPPORTED,
               "vq_rotary: at most 65535 heads, 65536 channels and 2^31 - 1 positions a sequence");
    if (a.B == 0 || a.S == 0 || heads == 0) return VQ_OK;
    VQ_REQUIRE(a.B < (INT64_C(1) << 31), VQ_ERR_UNSUPPORTED, "vq_rotary: too many rows for one launch");
    VQ_REQUIRE(a.inv_freq != nullptr, VQ_ERR_INVALID, "vq_rotary: frequencies must be given");
    for (int w = 0; w < 2; ++w)
        VQ_REQUIRE(a.heads[w] == 0 || (a.x[w] != nullptr && a.out[w] != nullptr), VQ_ERR_INVALID, "vq_rotary: rows and outputs must be given");
    const int64_t sizes[2][3] = {{a.B, a.heads[0], a.S}, {a.B, a.heads[1], a.S}};
    for (int w = 0; w < 2; ++w)
        for (int d = 0; d < 3; ++d)
            VQ_REQUIRE(a.heads[w] == 0 || a.x[w] != a.out[w] || sizes[w][d] < 2 || a.x_strides[w][d] == a.out_strides[w][d], VQ_ERR_INVALID,
                       "vq_rotary: rows turned in place keep their strides");
    VQ_DISPATCH_FLOAT(a.dtype, T, return launch_rotary<T>(a, (hipStream_t)stream));
    return VQ_OK;
}
