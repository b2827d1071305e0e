// Norm of every head's row and rotary positions, of queries and keys, in one launch.
//
// y_c = x_c w_c / sqrt(mean(x^2) + eps) over the D channels of a head, w the norm's weight (one row, or one a head; none: ones); then
// channel pair i of the first `dims` turns by the angle p w_i as in rotary.hip, channels dims .. D - 1 of y pass through.  Squares, their sum
// and the turn are float32, the angle is formed in double; a value is rounded once, to the element type.
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

template <typename T> int launch_norm_rotary(const vq_norm_rotary_args &c, hipStream_t st) {
    const vq_rotary_args &a = c.rotary;
    const int64_t rows = a.B * (a.heads[0] + a.heads[1]) * a.S;
    norm_rotary_any_kernel<T><<<(unsigned)cdiv(rows, 4), 256, 0, st>>>(c);
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
    VQ_REQUIRE((double)a.B * (double)a.S * (double)heads < 16777216. * 4., VQ_ERR_UNSUPPORTED, "%s: 2^26 or more rows", fn);
    VQ_DISPATCH_FLOAT(a.dtype, T, return launch_norm_rotary<T>(*args, (hipStream_t)stream));
    return VQ_OK;
}
