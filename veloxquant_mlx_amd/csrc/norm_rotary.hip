// Norm of every head's row and rotary positions, of queries and keys, in one launch.
//
// y_c = x_c w_c / sqrt(mean(x^2) + eps) over the D channels of a head, w the norm's weight (one row, or one a head; none: ones); then
// channel pair i of the first `dims` turns by the angle p w_i as in rotary.hip, channels dims .. D - 1 of y pass through.  Squares, their sum
// and the turn are float32, the angle is formed in double; a value is rounded once, to the element type.
//
// Bound by HBM, a read and a write of every row: 40 heads of 128 channels, 8192 tokens of a projection's view in bf16 41 us, 4.1 TB/s (a wave a row, read
// twice: 223); 16 heads of 256, 7 x 1003 tokens, a weight row a head 24.6 us, 4.7 TB/s; one token 5.3, latency.  Four waves a SIMD by a cap on registers: 58 us in place
// of 41.
#include "common.hpp"

namespace vq {

namespace {

__device__ __forceinline__ float nr_ld(const void *p, int tag, int64_t i) {
    if (tag == VQ_F16) return (float)((const f16 *)p)[i];
    if (tag == VQ_BF16) return bf16_to_f32(((const u16 *)p)[i]);
    return ((const float *)p)[i];
}

// 1 / sqrt(t) within two units of the last place; t below the normal numbers too, which the instruction takes for zero
__device__ __forceinline__ float nr_rsqrt(float t) {
    const bool small = t < 0x1p-96f;
    return __builtin_amdgcn_rsqf(small ? t * 0x1p64f : t) * (small ? 0x1p32f : 1.f);
}

// x of another lane of the same sixteen
template <int CTRL> __device__ __forceinline__ float nr_moved(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}

__device__ __forceinline__ int64_t nr_position(const vq_rotary_args &a, int64_t b, int64_t s) {
    int64_t p = a.offset + (a.add_index ? s : 0);
    if (a.positions != nullptr) {
        const int64_t i = b * a.pos_stride_b + s * a.pos_stride_s;
        p += a.pos_dtype == VQ_I64 ? ((const int64_t *)a.positions)[i] : ((const int32_t *)a.positions)[i];
    }
    return p;
}

// Sine and cosine of the angle of pair i at `place` = position / 2 pi, times the factor (see rotary.hip)
__device__ __forceinline__ void nr_angle(const vq_rotary_args &a, double place, int64_t i, float &c, float &s) {
    const double w = a.freq_dtype == VQ_F64 ? ((const double *)a.inv_freq)[i] : (double)((const float *)a.inv_freq)[i];
    const double r = place * w;
    sincospif(2.f * (float)(r - rint(r)), &s, &c);
    c *= a.attention_factor;
    s *= a.attention_factor;
}

// Any head size, strides and alignment: a wave a row, twice over it.
template <typename T> __global__ __launch_bounds__(256) void norm_rotary_any_kernel(vq_norm_rotary_args c) {
    const vq_rotary_args &a = c.rotary;
    const int lane = threadIdx.x & 63;
    const int64_t heads = a.heads[0] + a.heads[1];
    int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.B * heads * a.S) return;
    const int64_t s = row % a.S;
    row /= a.S;
    const int64_t hh = row % heads, b = row / heads;
    const int w = hh >= a.heads[0];
    const int64_t h = hh - (w ? a.heads[0] : 0);
    const T *x = (const T *)a.x[w] + b * a.x_strides[w][0] + h * a.x_strides[w][1] + s * a.x_strides[w][2];
    T *out = (T *)a.out[w] + b * a.out_strides[w][0] + h * a.out_strides[w][1] + s * a.out_strides[w][2];
    float sum = 0.f;
    for (int64_t d = lane; d < a.D; d += 64) {
        const float v = Elem<T>::ld(x + d);
        sum = __builtin_fmaf(v, v, sum);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    const float r = nr_rsqrt(sum / (float)a.D + c.eps);
    auto normed = [&](int64_t d) {
        const float y = Elem<T>::ld(x + d) * r;
        return c.weight[w] == nullptr ? y : y * nr_ld(c.weight[w], c.weight_dtype, h * c.weight_stride[w] + d);
    };
    const double place = (double)nr_position(a, b, s) * 0.15915494309189533577;   // turns per radian
    for (int64_t i = lane; i < a.dims / 2; i += 64) {
        const int64_t c0 = a.layout == VQ_ROTARY_HALF ? i : 2 * i, c1 = a.layout == VQ_ROTARY_HALF ? i + a.dims / 2 : 2 * i + 1;
        float cs, sn;
        nr_angle(a, place, i, cs, sn);
        const float y0 = normed(c0), y1 = normed(c1);
        Elem<T>::st(out + c0, __builtin_fmaf(y0, cs, -(y1 * sn)));
        Elem<T>::st(out + c1, __builtin_fmaf(y1, cs, y0 * sn));
    }
    for (int64_t d = a.dims + lane; d < a.D; d += 64) Elem<T>::st(out + d, normed(d));
}

constexpr int NR_THREADS = 256;
constexpr int NR_FLIGHT = 4;              // rows a lane has in flight
constexpr int64_t NR_FILL = 256 * 1024;   // threads that fill the chip: 16 waves a CU

struct NormRotaryCall {
    vq_norm_rotary_args n;
    int lanes_log2;         // lanes of a row, of which the first `units` hold channels and the first `rot_units` of those turn
    int units, rot_units;
    int heads_per_thread;
    float by_d;             // 1 / D
    int wide_weight;        // 1: weights of the element type, read in whole pieces
};

template <typename T, int N> struct alignas(sizeof(T) * N) NormPiece { T v[N]; };
__device__ __forceinline__ void nr_st(f16 *p, float v) { *p = (f16)v; }
__device__ __forceinline__ void nr_st(bf16_t *p, float v) { p->bits = __builtin_bit_cast(u16, (__bf16)v); }   // (one instruction for two)
__device__ __forceinline__ void nr_st(float *p, float v) { *p = v; }

// Rows in whole pieces of 16 bytes.  The lanes of a row hold two pieces each, in the half layout a piece and the one that its channels pair with
// (else half a row apart, so that a load of the lanes is one stretch), so the row is read once: the squares meet in log2(lanes) steps, norm and turn are applied to what the lane holds.  A lane keeps the sines
// and cosines of its pairs at one position and walks over heads, queries then keys; norm weight and turn are one factor a term
// (w_0 cos, w_1 sin, w_1 cos, w_0 sin), formed once for all heads that share a weight row, and the first rows are asked for ahead of the angles.
//
// OWN: a weight row a head; its pieces are asked for with the row's, in place of the factors.
template <typename T, int N, bool HALF, bool OWN> __global__ __launch_bounds__(NR_THREADS) void norm_rotary_kernel(NormRotaryCall c) {
    const vq_rotary_args &a = c.n.rotary;
    const int u = threadIdx.x & ((1 << c.lanes_log2) - 1);
    const int64_t tok = (int64_t)blockIdx.x * (NR_THREADS >> c.lanes_log2) + (threadIdx.x >> c.lanes_log2);
    if (tok >= a.B * a.S) return;   // (the lanes of a row leave together)
    const int64_t b = tok / a.S, s = tok - b * a.S;
    const int D = (int)a.D, dims = (int)a.dims;
    // the lane's two pieces: the channel of each, which of them are there, which turn
    int c0, c1;
    bool turn0, turn1;
    if (HALF) {
        turn0 = turn1 = u < c.rot_units;
        c0 = turn0 ? u * N : dims + (u - c.rot_units) * N;
        c1 = turn0 ? c0 + dims / 2 : c0 + (c.units - c.rot_units) * N;
    } else {
        c0 = u * N;
        c1 = c0 + c.units * N;
        turn0 = c0 < dims;
        turn1 = c1 < dims;
    }
    const bool has0 = u < c.units, has1 = has0 && c1 < D;
    if (!has1) c1 = 0;
    if (!has0) c0 = 0;
    using P = NormPiece<T, N>;
    const int Hq = (int)a.heads[0], heads = Hq + (int)a.heads[1];
    const int first = (int)blockIdx.y * c.heads_per_thread, end = first + c.heads_per_thread < heads ? first + c.heads_per_thread : heads;
    P x0[NR_FLIGHT], x1[NR_FLIGHT], w0[NR_FLIGHT], w1[NR_FLIGHT];
    // rows h .. of the heads up to `to`, all queries or all keys
    auto load = [&](int h, int to) __attribute__((always_inline)) {
        const int w = h >= Hq;
        const T *from = (const T *)a.x[w] + b * a.x_strides[w][0] + s * a.x_strides[w][2];
#pragma unroll
        for (int k = 0; k < NR_FLIGHT; ++k) {
            const int64_t head = (h + k < to ? h + k : h) - (w ? Hq : 0);   // (missing rows: the first again)
            const T *row = from + head * a.x_strides[w][1];
            x0[k] = *(const P *)(row + c0);
            x1[k] = *(const P *)(row + c1);
            if (OWN) {
                const T *weight = (const T *)c.n.weight[w] + head * c.n.weight_stride[w];
                w0[k] = *(const P *)(weight + c0);
                w1[k] = *(const P *)(weight + c1);
            }
        }
    };
    auto upto = [&](int h) __attribute__((always_inline)) { const int last = h < Hq && Hq < end ? Hq : end; return h + NR_FLIGHT < last ? h + NR_FLIGHT : last; };
    int h = first, to = upto(h);
    load(h, to);
    // sines and cosines: half layout of pair j, (c0 + j, c1 + j); interleaved of pairs j of the first piece, then of the second
    float cs[N], sn[N];
    if (turn0) {
        const double place = (double)nr_position(a, b, s) * 0.15915494309189533577;   // turns per radian
#pragma unroll
        for (int j = 0; j < N; ++j) {
            cs[j] = 1.f;
            sn[j] = 0.f;
            if (HALF) nr_angle(a, place, c0 + j, cs[j], sn[j]);
            else if (j < N / 2) nr_angle(a, place, c0 / 2 + j, cs[j], sn[j]);
            else if (turn1) nr_angle(a, place, c1 / 2 + j - N / 2, cs[j], sn[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) { cs[j] = 1.f; sn[j] = 0.f; }
    }
    // factors of a value by its own channel (A, C) and of its partner (B, E)
    float A[N], B[N], C[N], E[N];
    auto factors = [&](int w) __attribute__((always_inline)) {
        float f0[N], f1[N];
        if (c.n.weight[w] == nullptr) {
#pragma unroll
            for (int j = 0; j < N; ++j) f0[j] = f1[j] = 1.f;
        } else if (c.wide_weight) {
            const P y0 = *(const P *)((const T *)c.n.weight[w] + c0), y1 = *(const P *)((const T *)c.n.weight[w] + c1);
#pragma unroll
            for (int j = 0; j < N; ++j) { f0[j] = Elem<T>::ld(&y0.v[j]); f1[j] = Elem<T>::ld(&y1.v[j]); }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                f0[j] = nr_ld(c.n.weight[w], c.n.weight_dtype, c0 + j);
                f1[j] = nr_ld(c.n.weight[w], c.n.weight_dtype, c1 + j);
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (HALF) {
                A[j] = cs[j] * f0[j]; B[j] = sn[j] * f1[j];
                C[j] = cs[j] * f1[j]; E[j] = sn[j] * f0[j];
            } else {   // pair j / 2 of either piece
                A[j] = cs[j / 2] * f0[j]; C[j] = cs[N / 2 + j / 2] * f1[j];
                B[j] = sn[j / 2] * f0[j ^ 1]; E[j] = sn[N / 2 + j / 2] * f1[j ^ 1];
            }
        }
    };
    int weighted = -1;   // which factors are held: of the queries or of the keys
#pragma unroll 1
    for (;;) {
        const int w = h >= Hq;
        if (!OWN && weighted != w) factors(w);
        weighted = w;
        T *out = (T *)a.out[w] + b * a.out_strides[w][0] + s * a.out_strides[w][2];
        float sum[NR_FLIGHT];
#pragma unroll
        for (int k = 0; k < NR_FLIGHT; ++k) {
            float p0 = 0.f, p1 = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float v0 = Elem<T>::ld(&x0[k].v[j]), v1 = Elem<T>::ld(&x1[k].v[j]);
                p0 = __builtin_fmaf(v0, v0, p0);
                p1 = __builtin_fmaf(v1, v1, p1);
            }
            sum[k] = (has0 ? p0 : 0.f) + (has1 ? p1 : 0.f);
        }
        // (within sixteen lanes by moves, not through the LDS unit)
        auto meet = [&](auto other) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < NR_FLIGHT; ++k) sum[k] += other(sum[k]);
        };
        if (c.lanes_log2 > 0) meet([](float x) { return nr_moved<0xB1>(x); });    // quad_perm [1,0,3,2]
        if (c.lanes_log2 > 1) meet([](float x) { return nr_moved<0x4E>(x); });    // quad_perm [2,3,0,1]
        if (c.lanes_log2 > 2) meet([](float x) { return nr_moved<0x141>(x); });   // row_half_mirror
        if (c.lanes_log2 > 3) meet([](float x) { return nr_moved<0x140>(x); });   // row_mirror
        if (c.lanes_log2 > 4) meet([](float x) { return __shfl_xor(x, 16); });
        if (c.lanes_log2 > 5) meet([](float x) { return __shfl_xor(x, 32); });
#pragma unroll
        for (int k = 0; k < NR_FLIGHT; ++k) {
            if (h + k >= to) break;
            const float r = nr_rsqrt(__builtin_fmaf(sum[k], c.by_d, c.n.eps));
            P y0, y1;
            float v0[N], v1[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v0[j] = Elem<T>::ld(&x0[k].v[j]) * r;
                v1[j] = Elem<T>::ld(&x1[k].v[j]) * r;
                if (OWN) { v0[j] *= Elem<T>::ld(&w0[k].v[j]); v1[j] *= Elem<T>::ld(&w1[k].v[j]); }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int p = HALF ? j : j / 2, p1 = HALF ? j : N / 2 + j / 2;   // the pairs of channels j of either piece
                const float fa = OWN ? cs[p] : A[j], fb = OWN ? sn[p] : B[j], fc = OWN ? cs[p1] : C[j], fe = OWN ? sn[p1] : E[j];
                const float o0 = HALF ? v1[j] : v0[j ^ 1], o1 = HALF ? v0[j] : v1[j ^ 1];
                nr_st(&y0.v[j], turn0 ? __builtin_fmaf(v0[j], fa, !HALF && j & 1 ? o0 * fb : -(o0 * fb)) : OWN ? v0[j] : v0[j] * fa);
                nr_st(&y1.v[j], turn1 ? __builtin_fmaf(v1[j], fc, HALF || j & 1 ? o1 * fe : -(o1 * fe)) : OWN ? v1[j] : v1[j] * fc);
            }
            T *row = out + (int64_t)(h + k - (w ? Hq : 0)) * a.out_strides[w][1];
            if (has0) *(P *)(row + c0) = y0;
            if (has1) *(P *)(row + c1) = y1;
        }
        h = to;
        if (h >= end) break;
        to = upto(h);
        load(h, to);
    }
}

template <typename T> int launch_norm_rotary(const vq_norm_rotary_args &n, hipStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    const vq_rotary_args &a = n.rotary;
    const bool half = a.layout == VQ_ROTARY_HALF;
    const int heads = (int)(a.heads[0] + a.heads[1]);
    NormRotaryCall c;
    c.n = n;
    // 16-byte pieces where every row of every tensor is aligned for them, no pair is cut and a wave's lanes hold the row
    const int64_t pieces = a.D / N;
    c.rot_units = (int)(half ? a.dims / 2 / N : 0);
    c.units = (int)(half ? c.rot_units + cdiv(pieces - 2 * c.rot_units, 2) : cdiv(pieces, 2));
    bool wide = a.D % N == 0 && (half ? a.dims / 2 : a.dims) % N == 0 && pieces <= 128;
    // OWN: both (those that are there) have a row a head, in whole pieces of the element type; one of the two alone, another type: a wave a row
    bool wide_weight = true, own = false, shared = false;
    for (int w = 0; w < 2; ++w) {
        if (a.heads[w] == 0) continue;
        wide = wide && (((uintptr_t)a.x[w] | (uintptr_t)a.out[w]) & 15) == 0;
        for (int d = 0; d < 3; ++d) wide = wide && a.x_strides[w][d] % N == 0 && a.out_strides[w][d] % N == 0;
        (n.weight[w] != nullptr && n.weight_stride[w] != 0 ? own : shared) = true;
        if (n.weight[w] != nullptr) wide_weight = wide_weight && n.weight_dtype == a.dtype && ((uintptr_t)n.weight[w] & 15) == 0 && n.weight_stride[w] % N == 0;
    }
    const int64_t tokens = a.B * a.S;
    if (wide && !(own && (shared || !wide_weight))) {
        c.wide_weight = wide_weight;
        c.by_d = 1.f / (float)a.D;
        c.lanes_log2 = 0;
        while (1 << c.lanes_log2 < c.units) ++c.lanes_log2;
        const int64_t threads = tokens << c.lanes_log2;
        VQ_REQUIRE(threads < (INT64_C(1) << 32) - NR_THREADS, VQ_ERR_UNSUPPORTED, "vq_norm_rotary: too many rows for one launch");
        c.heads_per_thread = heads;
        while (c.heads_per_thread > 1 && threads * cdiv(heads, c.heads_per_thread) < NR_FILL)
            c.heads_per_thread = c.heads_per_thread > NR_FLIGHT ? (int)cdiv(cdiv(c.heads_per_thread, 2), NR_FLIGHT) * NR_FLIGHT : c.heads_per_thread / 2;
        const dim3 grid((unsigned)cdiv(threads, NR_THREADS), (unsigned)cdiv(heads, c.heads_per_thread));
        if (own && half) norm_rotary_kernel<T, N, true, true><<<grid, NR_THREADS, 0, st>>>(c);
        else if (own) norm_rotary_kernel<T, N, false, true><<<grid, NR_THREADS, 0, st>>>(c);
        else if (half) norm_rotary_kernel<T, N, true, false><<<grid, NR_THREADS, 0, st>>>(c);
        else norm_rotary_kernel<T, N, false, false><<<grid, NR_THREADS, 0, st>>>(c);
        VQ_HIP_CHECK_LAUNCH("vq_norm_rotary");
        return VQ_OK;
    }
    const int64_t rows = tokens * heads;
    VQ_REQUIRE(rows < (INT64_C(1) << 26), VQ_ERR_UNSUPPORTED, "vq_norm_rotary: too many rows for one launch");
    norm_rotary_any_kernel<T><<<(unsigned)cdiv(rows, 4), 256, 0, st>>>(n);
    VQ_HIP_CHECK_LAUNCH("vq_norm_rotary");
    return VQ_OK;
}

}  // namespace

}  // namespace vq

extern "C" int vq_norm_rotary(const vq_norm_rotary_args *args, void *stream) {
    using namespace vq;
    const char *fn = "vq_norm_rotary";
    VQ_REQUIRE(args != nullptr, VQ_ERR_INVALID, "%s: no arguments", fn);
    const vq_rotary_args &a = args->rotary;
    if (int rc = check_rotary(fn, a)) return rc;
    VQ_REQUIRE(a.inverse == 0, VQ_ERR_INVALID, "%s: a norm is not turned back", fn);
    VQ_REQUIRE(args->eps >= 0.f, VQ_ERR_INVALID, "%s: eps must not be negative", fn);
    for (int w = 0; w < 2; ++w) {
        if (args->weight[w] == nullptr) continue;
        VQ_REQUIRE(is_float_tag(args->weight_dtype), VQ_ERR_INVALID, "%s: unsupported weight dtype tag %d", fn, args->weight_dtype);
        VQ_REQUIRE(args->weight_stride[w] == 0 || args->weight_stride[w] >= a.D, VQ_ERR_INVALID, "%s: weight rows of %lld channels", fn, (long long)args->weight_stride[w]);
    }
    const int64_t heads = a.heads[0] + a.heads[1];
    if (a.B == 0 || a.S == 0 || heads == 0) return VQ_OK;
    VQ_REQUIRE((double)a.B * (double)a.S < 4294967296., VQ_ERR_UNSUPPORTED, "%s: too many rows for one launch", fn);
    VQ_DISPATCH_FLOAT(a.dtype, T, return launch_norm_rotary<T>(*args, (hipStream_t)stream));
    return VQ_OK;
}
