// An MLP's activation whose backward pass reads its input from 8 bits.
//
//   forward:   y = act(x), or act(x[:, :W]) x[:, W:] (gated), and x as codes: 32 consecutive values of the contiguous tensor share
//              2^e, the smallest power of two with max|x| <= 127 2^e (int8) or 448 2^e (e4m3), one byte e + 127 a block
//   backward:  with z the value of the codes: dx = grad act'(z); gated: grad z_up act'(z_gate), grad act(z_gate).  The same pass
//              gives act(z) (times z_up) again, which the weight gradient of the layer behind reads: y need not be kept either
//
// The unit is a power of two so that x / 2^e is exact and the code is the format's one rounding to nearest even: int8 holds x to
// 2^(e-1), e4m3 to 2^-4 of itself and at best to 2^(e-10), its smallest steps (below that, 2^-18 of the block's largest, 0).  An infinity is held as the format's largest value, a NaN as 0x7f (e4m3) or -128 (int8); they
// do not count for the unit.
//
// Bound by memory: forward 2 accesses and 33/32 byte a value, backward 33/32 byte and 2 to 3 accesses.  A thread takes 8 values;
// four threads share a block's unit through two lane exchanges.  Rows of an odd width put chunks at any alignment: the loads and
// stores are written for the element's alignment (the hardware takes 16 bytes at any address).
#include "adk_common.hpp"

namespace adk {

enum { A8_GELU = 0, A8_GELU_TANH = 1, A8_SILU = 2 };

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) A8Eight { T e[8]; };
struct __attribute__((packed, aligned(1))) A8Codes { uint32_t lo, hi; };

__device__ __forceinline__ float a8_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }

template <int KIND> __device__ __forceinline__ float a8_value(float x) {
    if (KIND == A8_SILU) return x * a8_sigmoid(x);
    if (KIND == A8_GELU) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    return x * a8_sigmoid(x * (1.5957691216057308f + 0.071354816272600385f * x * x)); // (1 + tanh t) / 2 = sigmoid(2 t)
}
// act(x) and act'(x)
template <int KIND> __device__ __forceinline__ float a8_slope(float x, float& value) {
    if (KIND == A8_SILU) {
        const float s = a8_sigmoid(x);
        value = x * s;
        return s * (1.f + x * (1.f - s));
    }
    if (KIND == A8_GELU) {
        const float c = 0.5f * (1.f + erff(x * 0.70710678118654752f));
        value = x * c;
        return c + x * 0.39894228040143268f * __builtin_amdgcn_exp2f(-0.72134752044448170f * x * x);
    }
    const float xx = fminf(x * x, 1e30f); // an infinite square would meet a zero below
    const float s = a8_sigmoid(x * (1.5957691216057308f + 0.071354816272600385f * xx));
    value = x * s;
    return s + x * s * (1.f - s) * (1.5957691216057308f + 0.21406444881780115f * xx);
}

template <typename T> __device__ __forceinline__ void a8_load(const T* p, float* v) {
    const A8Eight<T> t = *reinterpret_cast<const A8Eight<T>*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)t.e[j];
}
template <typename T> __device__ __forceinline__ void a8_store(T* p, const float* v) {
    A8Eight<T> t;
#pragma unroll
    for (int j = 0; j < 8; ++j) t.e[j] = (T)v[j];
    *reinterpret_cast<A8Eight<T>*>(p) = t;
}

// The biased exponent of the unit for a block whose largest finite magnitude is `top`.
template <bool E4M3> __device__ __forceinline__ int a8_unit(float top) {
    const int bits = (int)__float_as_uint(top), e = bits >> 23, m = bits & 0x7fffff;
    return max(1, E4M3 ? e - 8 + (m > 0x600000) : e - 6 + (m > 0x7e0000));
}
template <bool E4M3> __device__ __forceinline__ A8Codes a8_encode(const float* v, int unit) {
    const float inv = __uint_as_float((uint32_t)(254 - unit) << 23);
    if (E4M3) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = v[j] * inv;
            if (fabsf(w[j]) > 448.f) w[j] = copysignf(448.f, w[j]); // infinities
        }
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(w[4], w[5], 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(w[6], w[7], hi, true);
        return A8Codes{(uint32_t)lo, (uint32_t)hi};
    }
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float w = rintf(fminf(fmaxf(v[j] * inv, -127.f), 127.f));
        const int code = v[j] != v[j] ? -128 : (int)w;
        c[j >> 2] |= (uint32_t)(code & 255) << (8 * (j & 3));
    }
    return A8Codes{c[0], c[1]};
}
// the eight codes' values in units
template <bool E4M3> __device__ __forceinline__ void a8_decode(const A8Codes& c, float* v) {
    if (E4M3) {
        v[0] = __builtin_amdgcn_cvt_f32_fp8((int)c.lo, 0); v[1] = __builtin_amdgcn_cvt_f32_fp8((int)c.lo, 1);
        v[2] = __builtin_amdgcn_cvt_f32_fp8((int)c.lo, 2); v[3] = __builtin_amdgcn_cvt_f32_fp8((int)c.lo, 3);
        v[4] = __builtin_amdgcn_cvt_f32_fp8((int)c.hi, 0); v[5] = __builtin_amdgcn_cvt_f32_fp8((int)c.hi, 1);
        v[6] = __builtin_amdgcn_cvt_f32_fp8((int)c.hi, 2); v[7] = __builtin_amdgcn_cvt_f32_fp8((int)c.hi, 3);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int code = (int8_t)((j < 4 ? c.lo : c.hi) >> (8 * (j & 3)));
        v[j] = code == -128 ? __uint_as_float(0x7fc00000u) : (float)code;
    }
}
__device__ __forceinline__ float a8_unit_value(int unit) { return __uint_as_float((uint32_t)unit << 23); }

// A thread's 8 consecutive values, from value i of the flat tensor on.  width: columns of the gate (0: not gated).  codes: null where nothing is
// kept (16384 x 2 x 5461 bf16, gated: 114 us, 164 where x is kept).
template <typename T, int KIND, bool E4M3, bool GATED>
__global__ __launch_bounds__(256) void a8_fwd_kernel(const T* __restrict__ x, int64_t n, int64_t width, T* __restrict__ y, uint8_t* __restrict__ codes,
                                                     uint8_t* __restrict__ units)
{
    // neighbouring chunks on one XCD: a gate chunk reads the up values that its neighbours a row half further on have just brought to its L2
    const int64_t i = ((int64_t)xcd_remap(blockIdx.x, gridDim.x) * 256 + threadIdx.x) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const bool whole = i + 8 <= n;
    if (whole) a8_load(x + i, v);
    else
        for (int j = 0; j < 8; ++j)
            if (i + j < n) v[j] = (float)x[i + j];
    if (codes) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]) < INFINITY ? fabsf(v[j]) : 0.f);
        top = fmaxf(top, __shfl_xor(top, 1));
        top = fmaxf(top, __shfl_xor(top, 2));
        if (i >= ((n + 31) & ~(int64_t)31)) return; // the codes' room ends with the last block
        const int unit = a8_unit<E4M3>(top);
        *reinterpret_cast<A8Codes*>(codes + i) = a8_encode<E4M3>(v, unit);
        if ((i & 31) == 0) units[i >> 5] = (uint8_t)unit;
    }
    if (!GATED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = a8_value<KIND>(v[j]);
        if (whole) a8_store(y + i, v);
        else
            for (int j = 0; j < 8; ++j)
                if (i + j < n) y[i + j] = (T)v[j];
        return;
    }
    const int64_t row = n >> 32 ? i / (2 * width) : (uint32_t)i / (uint32_t)(2 * width), col = i - row * 2 * width;
    if (whole && col + 8 <= width) {
        float up[8];
        a8_load(x + i + width, up);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = a8_value<KIND>(v[j]) * up[j];
        a8_store(y + row * width + col, v);
    } else if (col < width || col + 8 > 2 * width) { // the chunk holds an end of the gate's columns, or a beginning
        for (int j = 0; j < 8; ++j) {
            const int64_t at = i + j, r = at / (2 * width), c = at - r * 2 * width;
            if (at < n && c < width) y[r * width + c] = (T)(a8_value<KIND>(v[j]) * (float)x[at + width]);
        }
    }
}

// A thread's 8 values of the output's rows: the gate's codes and, gated, the codes `width` further on.
template <typename T, int KIND, bool E4M3, bool GATED>
__global__ __launch_bounds__(256) void a8_bwd_kernel(const T* __restrict__ grad, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ units, int64_t n,
                                                     int64_t width, T* __restrict__ dx, T* __restrict__ again)
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t i, at, left; // the chunk in x, in y, and the values that are left there
    if (GATED) {
        const int64_t rows = n / (2 * width), chunks = (width + 7) >> 3;
        const int64_t row = (rows * chunks) >> 32 ? id / chunks : (uint32_t)id / (uint32_t)chunks, col = (id - row * chunks) * 8;
        if (row >= rows) return;
        i = row * 2 * width + col;
        at = row * width + col;
        left = width - col;
    } else {
        i = at = id * 8;
        left = n - i;
        if (left <= 0) return;
    }
    auto kept = [&](int64_t p, float* v) { // the values of codes p .. p + 7, of one or two blocks
        A8Codes c = {0, 0};
        if (left >= 8) c = *reinterpret_cast<const A8Codes*>(codes + p);
        else
            for (int j = 0; j < left; ++j) (j < 4 ? c.lo : c.hi) |= (uint32_t)codes[p + j] << (8 * (j & 3));
        a8_decode<E4M3>(c, v);
        const float u0 = a8_unit_value(units[p >> 5]);
        if (!GATED) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= u0;
            return;
        }
        const float u1 = a8_unit_value(units[(p + (left < 8 ? left : 8) - 1) >> 5]);
        const int turn = 32 - (int)(p & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= j < turn ? u0 : u1;
    };
    float z[8], g[8], d[8], w[8];
    kept(i, z);
    if (left >= 8) a8_load(grad + at, g);
    else
        for (int j = 0; j < 8; ++j) g[j] = j < left ? (float)grad[at + j] : 0.f;
    if (GATED) {
        float up[8], du[8];
        kept(i + width, up);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float value;
            d[j] = g[j] * up[j] * a8_slope<KIND>(z[j], value);
            du[j] = g[j] * value;
            w[j] = value * up[j];
        }
        if (left >= 8) a8_store(dx + i + width, du);
        else
            for (int j = 0; j < left; ++j) dx[i + width + j] = (T)du[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = g[j] * a8_slope<KIND>(z[j], w[j]);
    }
    if (left >= 8) {
        a8_store(dx + i, d);
        if (again) a8_store(again + at, w);
    } else
        for (int j = 0; j < left; ++j) {
            dx[i + j] = (T)d[j];
            if (again) again[at + j] = (T)w[j];
        }
}

struct A8Call {
    const void *x, *grad;
    void *y, *dx, *again;
    uint8_t *codes, *units;
    int64_t n, width;
};

template <typename T, int KIND, bool E4M3, bool GATED> static int a8_launch(const A8Call& c, bool forward, hipStream_t stream) {
    const int64_t chunks = forward ? ceil_div(c.n, 32) * 4 : GATED ? c.n / (2 * c.width) * ceil_div(c.width, 8) : ceil_div(c.n, 8);
    const int64_t blocks = ceil_div(chunks, 256);
    if (blocks > 0xffffff) return ADK_EUNSUPPORTED; // a launch has fewer than 2^32 threads
    if (forward)
        hipLaunchKernelGGL((a8_fwd_kernel<T, KIND, E4M3, GATED>), dim3((unsigned)blocks), dim3(256), 0, stream, static_cast<const T*>(c.x), c.n, c.width,
                           static_cast<T*>(c.y), c.codes, c.units);
    else
        hipLaunchKernelGGL((a8_bwd_kernel<T, KIND, E4M3, GATED>), dim3((unsigned)blocks), dim3(256), 0, stream, static_cast<const T*>(c.grad), c.codes, c.units, c.n,
                           c.width, static_cast<T*>(c.dx), static_cast<T*>(c.again));
    ADK_RETURN_LAST_ERROR();
}
template <typename T, int KIND> static int a8_format(const A8Call& c, int e4m3, bool forward, hipStream_t s) {
    if (c.width) return e4m3 ? a8_launch<T, KIND, true, true>(c, forward, s) : a8_launch<T, KIND, false, true>(c, forward, s);
    return e4m3 ? a8_launch<T, KIND, true, false>(c, forward, s) : a8_launch<T, KIND, false, false>(c, forward, s);
}
template <typename T> static int a8_kind(const A8Call& c, int kind, int e4m3, bool forward, hipStream_t s) {
    if (kind == A8_GELU) return a8_format<T, A8_GELU>(c, e4m3, forward, s);
    if (kind == A8_GELU_TANH) return a8_format<T, A8_GELU_TANH>(c, e4m3, forward, s);
    return a8_format<T, A8_SILU>(c, e4m3, forward, s);
}
static int a8_call(const A8Call& c, int dtype, int kind, int e4m3, bool forward, hipStream_t s) {
    if (dtype == 0) return a8_kind<_Float16>(c, kind, e4m3, forward, s);
    if (dtype == 1) return a8_kind<float>(c, kind, e4m3, forward, s);
    return a8_kind<__bf16>(c, kind, e4m3, forward, s);
}
static int a8_check(int dtype, int64_t rows, int64_t width, int kind, int gated, int format) {
    if (dtype < 0 || dtype > 2 || kind < 0 || kind > 2 || format < 0 || format > 1) return ADK_EUNSUPPORTED;
    if (rows < 0 || width < 0 || (width && rows > ((int64_t)1 << 40) / width)) return ADK_EINVAL;
    return 0;
}

} // namespace adk

extern "C" int adk_activation8_fwd(const void* x, int dtype, int64_t rows, int64_t width, int kind, int gated, int format, void* y, uint8_t* codes, uint8_t* units,
                                   hipStream_t stream)
{
    const int e = adk::a8_check(dtype, rows, width, kind, gated, format);
    if (e) return e;
    if (rows == 0 || width == 0) return 0;
    if (!x || !y || !codes != !units || ((uintptr_t)codes & 7)) return ADK_EINVAL;
    adk::A8Call c = {};
    c.x = x; c.y = y; c.codes = codes; c.units = units;
    c.n = rows * width * (gated ? 2 : 1); c.width = gated ? width : 0;
    return adk::a8_call(c, dtype, kind, format, true, stream);
}

extern "C" int adk_activation8_bwd(const void* grad, const uint8_t* codes, const uint8_t* units, int dtype, int64_t rows, int64_t width, int kind, int gated, int format,
                                   void* dx, void* again, hipStream_t stream)
{
    const int e = adk::a8_check(dtype, rows, width, kind, gated, format);
    if (e) return e;
    if (rows == 0 || width == 0) return 0;
    if (!grad || !codes || !units || !dx || ((uintptr_t)codes & 7)) return ADK_EINVAL;
    adk::A8Call c = {};
    c.grad = grad; c.codes = const_cast<uint8_t*>(codes); c.units = const_cast<uint8_t*>(units); c.dx = dx; c.again = again;
    c.n = rows * width * (gated ? 2 : 1); c.width = gated ? width : 0;
    return adk::a8_call(c, dtype, kind, format, false, stream);
}
