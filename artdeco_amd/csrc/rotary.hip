// Rotary positions, out of place or in place: every pair (u, v) of a head's first channels becomes
//   (u cos - v sin, v cos + u sin) * factor,   angle = position * frequency[pair],
// or, for the gradient, the same with -angle (the transpose).  Pairs are (m, m + pairs) of a segment ("half") or (2m, 2m + 1)
// ("interleaved"); with several axes the turned channels are equal segments, each turned by a position of its own.  Channels
// behind the turned ones, and heads behind the turned heads, are copied (out of place) or left (in place).
//
// The angle of position 1e6 has no correct bit left in 32-bit turns, so position * frequency / 2 pi is formed in 64 bits, its
// whole turns are dropped there, and cos / sin are taken of the rest in 32 bits.
//
// Bound by memory: 2 accesses an element.  A thread owns one 16-byte chunk column of a token (both chunks of its pairs) and walks
// every `slices`-th head with it, so the trigonometry is done once a column; neighbouring threads take neighbouring columns, then
// heads.
#include "adk_common.hpp"

namespace adk {

struct RotaryArgs {
    const void* x;
    void* y;
    const int64_t* positions;
    const double* frequencies;
    int64_t x_sb, x_sn, x_sh, y_sb, y_sn, y_sh, p_sb, p_sn, p_sa;
    int64_t tokens;
    int N, H, D, turned, pairs, axes, copy, slices;
    float factor, sign;
};

template <typename T, int W> struct alignas(sizeof(T) * W) RtPack { T e[W]; };

template <typename T> __device__ __forceinline__ float rt_to(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T rt_from(float x) { return (T)x; }

// W elements a chunk (1: any size and alignment); HALF: a unit is a chunk of first and the chunk of second channels, otherwise
// one chunk of W / 2 interleaved pairs (W = 1: the two elements of one pair).
template <typename T, int W, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a)
{
    constexpr int NP = HALF ? W : (W > 1 ? W / 2 : 1); // pairs a unit
    typedef RtPack<T, W> P;
    const int turn_units = a.axes * a.pairs / NP, R = 2 * a.axes * a.pairs, tail_units = a.copy ? (a.D - R) / W : 0;
    const int units = turn_units + tail_units, chunks = a.D / W;
    const int per_token = units * a.slices + (a.copy ? (a.H - a.turned) * chunks : 0);
    const int tpb = max(1, 256 / per_token);
    int64_t token;
    int u;
    if (per_token <= 256) {
        const int own = threadIdx.x / per_token;
        if (own >= tpb) return;
        token = (int64_t)blockIdx.x * tpb + own;
        u = threadIdx.x - own * per_token;
    } else {
        const int blocks = (per_token + 255) / 256;
        token = blockIdx.x / blocks;
        u = (blockIdx.x - (int)token * blocks) * 256 + threadIdx.x;
        if (u >= per_token) return;
    }
    if (token >= a.tokens) return;
    const int b = (int)(token / a.N), n = (int)(token - (int64_t)b * a.N);
    const T* xt = static_cast<const T*>(a.x) + b * a.x_sb + n * a.x_sn;
    T* yt = static_cast<T*>(a.y) + b * a.y_sb + n * a.y_sn;
    if (u >= units * a.slices) { // a head that is not turned
        u -= units * a.slices;
        const int head = a.turned + u / chunks, c = u % chunks * W;
        *reinterpret_cast<P*>(yt + head * a.y_sh + c) = *reinterpret_cast<const P*>(xt + head * a.x_sh + c);
        return;
    }
    const int first = u / units;
    u -= first * units;
    if (u >= turn_units) { // channels behind the turned ones
        const int c = R + (u - turn_units) * W;
        for (int head = first; head < a.turned; head += a.slices)
            *reinterpret_cast<P*>(yt + head * a.y_sh + c) = *reinterpret_cast<const P*>(xt + head * a.x_sh + c);
        return;
    }
    const int axis = u * NP / a.pairs, m0 = u * NP - axis * a.pairs; // a unit's pairs are of one axis
    const double at = (double)a.positions[b * a.p_sb + n * a.p_sn + axis * a.p_sa] * 0.15915494309189533577; // / 2 pi
    float cs[NP], sn[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const double turns = at * a.frequencies[m0 + j];
        float s, c;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        cs[j] = c * a.factor;
        sn[j] = s * a.factor * a.sign;
    }
    const int c0 = 2 * axis * a.pairs + (HALF ? m0 : 2 * m0);
    for (int head = first; head < a.turned; head += a.slices) {
        const T* xp = xt + head * a.x_sh + c0;
        T* yp = yt + head * a.y_sh + c0;
        if (HALF || W == 1) {
            const int other = HALF ? a.pairs : 1;
            const P p = *reinterpret_cast<const P*>(xp), q = *reinterpret_cast<const P*>(xp + other);
            P o, r;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float x0 = rt_to(p.e[j]), x1 = rt_to(q.e[j]);
                o.e[j] = rt_from<T>(x0 * cs[j] - x1 * sn[j]);
                r.e[j] = rt_from<T>(x1 * cs[j] + x0 * sn[j]);
            }
            *reinterpret_cast<P*>(yp) = o;
            *reinterpret_cast<P*>(yp + other) = r;
        } else {
            const P p = *reinterpret_cast<const P*>(xp);
            P o;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const float x0 = rt_to(p.e[2 * j]), x1 = rt_to(p.e[2 * j + 1]);
                o.e[2 * j] = rt_from<T>(x0 * cs[j] - x1 * sn[j]);
                o.e[2 * j + 1] = rt_from<T>(x1 * cs[j] + x0 * sn[j]);
            }
            *reinterpret_cast<P*>(yp) = o;
        }
    }
}

template <typename T, int W> static int rotary_launch(RotaryArgs& a, int half, hipStream_t stream) {
    const int np = half ? W : (W > 1 ? W / 2 : 1);
    const int64_t units = a.axes * a.pairs / np + (a.copy ? (a.D - 2 * a.axes * a.pairs) / W : 0);
    const int64_t rest = a.copy ? (int64_t)(a.H - a.turned) * (a.D / W) : 0;
    a.slices = 1;
    // Threads for two waves a SIMD, and at least 8 heads side by side.  More slices repeat the trigonometry (4 x 768 tokens, 32 of 48 heads of 64:
    // 11.4 us with 32 slices, 9.8 with 16, 11.5 with 8), fewer leave a wave 256 bytes at a time (32749 x 32 heads of 128: 130 us with one, 113
    // with two, 99.7 with eight, 5.4 TB/s; 110 with sixteen); element by element (W = 1) the trigonometry is all that counts.
    while (a.slices < a.turned && (a.tokens * units * a.slices < 128 * 1024 || (W > 1 && a.slices < 8))) a.slices *= 2;
    if (a.slices > a.turned) a.slices = a.turned;
    const int64_t per_token = units * a.slices + rest;
    if (per_token <= 0) return 0;
    if (per_token > 0x7fffffff) return ADK_EUNSUPPORTED;
    const int64_t blocks = per_token <= 256 ? ceil_div(a.tokens, 256 / per_token) : a.tokens * ceil_div(per_token, 256);
    if (blocks > 0xffffff) return ADK_EUNSUPPORTED; // a launch has fewer than 2^32 threads
    if (half) hipLaunchKernelGGL((rotary_kernel<T, W, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<T, W, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    ADK_RETURN_LAST_ERROR();
}

template <typename T> static int rotary_of(RotaryArgs& a, int half, hipStream_t stream) {
    constexpr int W = 16 / sizeof(T);
    const bool wide = !(((uintptr_t)a.x | (uintptr_t)a.y) & 15) && !((a.x_sb | a.x_sn | a.x_sh | a.y_sb | a.y_sn | a.y_sh) & (W - 1)) &&
                      a.D % W == 0 && a.pairs % (half ? W : W / 2) == 0 && (2 * a.axes * a.pairs) % W == 0;
    return wide ? rotary_launch<T, W>(a, half, stream) : rotary_launch<T, 1>(a, half, stream);
}

} // namespace adk

extern "C" int adk_rotary(const void* x, void* y, const int64_t* positions, const double* frequencies, int dtype, int B, int N, int H, int D, int turned, int pairs, int axes,
                          int half, int transpose, float factor, const int64_t* strides, hipStream_t stream)
{
    if (B < 0 || N < 0 || H < 0 || D < 0 || turned < 0 || turned > H || pairs < 1 || axes < 1 || (int64_t)2 * pairs * axes > D) return ADK_EINVAL;
    if (dtype < 0 || dtype > 2) return ADK_EUNSUPPORTED;
    if (B == 0 || N == 0 || H == 0) return 0;
    if (!x || !y || !positions || !frequencies || !strides) return ADK_EINVAL;
    adk::RotaryArgs a = {};
    a.x = x; a.y = y; a.positions = positions; a.frequencies = frequencies;
    a.x_sb = strides[0]; a.x_sn = strides[1]; a.x_sh = strides[2];
    a.y_sb = strides[3]; a.y_sn = strides[4]; a.y_sh = strides[5];
    a.p_sb = strides[6]; a.p_sn = strides[7]; a.p_sa = strides[8];
    a.tokens = (int64_t)B * N;
    a.N = N; a.H = H; a.D = D; a.turned = turned; a.pairs = pairs; a.axes = axes; a.copy = x != y;
    a.factor = factor; a.sign = transpose ? -1.f : 1.f;
    if (turned == 0 && !a.copy) return 0;
    if (dtype == 0) return adk::rotary_of<_Float16>(a, half, stream);
    if (dtype == 1) return adk::rotary_of<float>(a, half, stream);
    return adk::rotary_of<__bf16>(a, half, stream);
}
