// Attention with its gradient: softmax(scale q k^T) v over the visible keys, fp16 or bf16 operands, fp32 scores, softmax
// statistics and accumulation.  Head sizes 8..128 (multiples of 8), several query heads to a key head, causal order, a length
// for each sequence and a free boolean mask; a query that sees no key gives zeros and a logarithm of -inf.
//
//   s_ij = scale <q_i, k_j>,  lse_i = log sum_j exp s_ij,  P_ij = exp(s_ij - lse_i),  o_i = sum_j P_ij v_j
//   dV = P^T dO,  dP = dO V^T,  delta_i = <dO_i, o_i>,  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q
//
// The backward pass keeps nothing of size Nq x Nk: it recomputes P from q, k and lse.  Two kernels write the gradients, one
// owning rows (dQ), one owning keys (dK, dV), each summing in a fixed order in its own registers: no atomics, the same bits on
// every run, and the heads that share a key head are summed by the owner of the key.  That recomputes S and dP twice (7 products
// instead of 5); a single kernel would add its dQ tiles into memory in an order that changes from run to run.
//
// Rows: the G query heads of a key head are one list of G Nq rows (row = g Nq + i), cut into tiles: single-token calls with 8
// heads to a key head read K and V once for all 8, and the owner of a key walks all rows that see it.
//
// Layout (v_mfma_f32_32x32x16): lane (h, c) = (lane >> 5, lane & 31) holds A[c][8h + e], B[8h + e][c], and of the product column c,
// rows 8 (r / 4) + 4 h + r % 4, r = 0..15.  Products are arranged so that a probability is already where the next product wants
// it: S^T = K Q^T gives P^T as the B operand of O^T = V^T P^T (key slot (h, e) of a 16-key step bound to key 8 (e / 4) + 4 h +
// e % 4, the order the accumulator has), and likewise S = Q K^T gives P, dS as B operands of dV^T = dO^T P, dK^T = Q^T dS.  The
// transposed A operands come from row-major tiles through ds_read_b64_tr_b16.
//
// LDS tiles hold 16-byte chunks at chunk ^ f(row): with f below, the 16 rows of a 128-bit fragment read and the 4 rows of a
// transposing read fall on different banks without padding.
#include "adk_common.hpp"

namespace adk {

typedef _Float16 at_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 at_f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_bf16x4 __attribute__((ext_vector_type(4)));
typedef float at_f32x16 __attribute__((ext_vector_type(16)));
typedef float at_f32x4 __attribute__((ext_vector_type(4)));
typedef short at_s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int at_u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct AtEl;
template <> struct AtEl<_Float16> {
    typedef at_f16x8 x8;
    typedef at_f16x4 x4;
    static __device__ __forceinline__ at_f32x16 mfma(x8 a, x8 b, at_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct AtEl<__bf16> {
    typedef at_bf16x8 x8;
    typedef at_bf16x4 x4;
    static __device__ __forceinline__ at_f32x16 mfma(x8 a, x8 b, at_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

struct AttendArgs {
    const void *q, *k, *v, *out_in, *dout;
    void *out, *dq, *dk, *dv;
    float* lse;             // [B, H, Nq]
    float* delta;           // [B, H, Nq]
    float* part_o;          // [splits, B, Hk, G Nq, D] (splits > 1)
    float* part_ml;         // [splits, B, Hk, G Nq, 2]
    float* amax;            // largest |dout| of each block of at_delta_kernel
    const int* key_lengths; // [B] or null
    const uint8_t* mask;    // or null
    int B, H, Hk, G, Nq, Nk, D, splits, causal, mask_by_key;
    int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn, g_sb, g_sh, g_sn; // element strides: batch, head, token
    int64_t dq_sb, dq_sh, dq_sn, dk_sb, dk_sh, dk_sn, dv_sb, dv_sh, dv_sn;
    int64_t m_sb, m_sh, m_sq, m_sk;
    float scale, scale_log2e;
};

#define AT_ROWS 128 // rows (or keys) that a workgroup owns: 4 waves of 32
#define AT_TILE 64  // keys (or rows) of a staged tile

template <int DP> __device__ __forceinline__ int at_swz(int row) {
    return DP == 64 ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : (((row & 3) << 2) | ((row >> 2) & 3));
}
template <int DP> __device__ __forceinline__ int at_off(int row, int chunk) { return row * DP + ((chunk ^ at_swz<DP>(row)) << 3); }

__device__ __forceinline__ float at_max3(float x, float y, float z) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x, y), z); // one v_maximum3_f32; keeps a NaN
}
__device__ __forceinline__ float at_other_half(float v) { // the value of lane ^ 32
    typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? sw.x : sw.y);
}
__device__ __forceinline__ int at_wave_max(int v) {
    for (int o = 32; o; o >>= 1) v = max(v, __shfl_xor(v, o));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int at_wave_min(int v) {
    for (int o = 32; o; o >>= 1) v = min(v, __shfl_xor(v, o));
    return __builtin_amdgcn_readfirstlane(v);
}

// Fragment of a row-major LDS tile as the A operand: row r0 + c, elements 16 ks + 8 h .. + 7.
template <typename T, int DP> __device__ __forceinline__ typename AtEl<T>::x8 at_rowfrag(const T* tile, int r0, int ks, int lane) {
    return *reinterpret_cast<const typename AtEl<T>::x8*>(tile + at_off<DP>(r0 + (lane & 31), 2 * ks + (lane >> 5)));
}
// Fragment of its transpose as the A operand: row d = 32 db + c; slot (h, e) is tile row r0 + 8 (e / 4) + 4 h + e % 4.
// Inside 16 lanes ds_read_b64_tr_b16 gives lane i element j the element i & 3 of the 8 bytes that lane 4 j + (i >> 2) addresses.
template <typename T, int DP> __device__ __forceinline__ typename AtEl<T>::x8 at_colfrag(const T* tile, int r0, int db, int lane) {
    typedef __attribute__((address_space(3))) at_s16x4 lds_s16x4;
    const int h = lane >> 5, i = lane & 15, row = r0 + 4 * h + (i >> 2), chunk = 4 * db + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1), sub = 4 * (i & 1);
    const at_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + at_off<DP>(row, chunk) + sub));
    const at_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + at_off<DP>(row + 8, chunk) + sub));
    return __builtin_shufflevector(__builtin_bit_cast(typename AtEl<T>::x4, lo), __builtin_bit_cast(typename AtEl<T>::x4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
}

// A tile of AT_TILE rows goes from memory to LDS without passing through registers: each wave instruction moves 64 chunks of 16 bytes
// to consecutive LDS addresses, so the swizzle is in which chunk a lane asks for.  In asm because the compiler waits for the
// builtin's loads before any LDS read; the waits are at_landed() before the barrier that hands a tile over.  The address is a
// uniform base and a 32-bit byte offset (token strides are below 2^24 elements).
__device__ __forceinline__ void at_lds16(uint32_t lds, const void* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void at_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <typename T, int DP> struct AtTile {
    static constexpr int CH = DP / 8, IT = AT_TILE * CH / 256;
    // rows from base on; those past the `rows` (>= 1) that there are repeat the last (they are hidden in the scores, and what lies
    // there is never read); chunks past D are left as they are
    static __device__ __forceinline__ void load(T* tile, const T* base, int sn, int rows, int D) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)tile;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int row = (4 * i + wave) * (64 / CH) + lane / CH, chunk = (lane % CH) ^ at_swz<DP>(row);
            const uint32_t off = (uint32_t)min(row, rows - 1) * (uint32_t)sn * 2u + chunk * 16;
            if (DP == D || chunk * 8 < D) at_lds16(lds + (4 * i + wave) * 1024, base, off);
        }
    }
    // a mask that is the same for every query hides a key altogether: zeros, whatever stands there (by the lanes that loaded it)
    static __device__ __forceinline__ void hide(T* tile, const uint8_t* mask, int64_t sk, int rows) {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int row = (4 * i + wave) * (64 / CH) + lane / CH;
            if (!mask[(int64_t)min(row, rows - 1) * sk]) *reinterpret_cast<at_u32x4*>(tile + (4 * i + wave) * 512 + lane * 8) = at_u32x4{0, 0, 0, 0};
        }
    }
    // zeros in the chunks past D of `tiles` tiles, which no load touches
    static __device__ __forceinline__ void pad(T* first, int tiles, int D) {
        if (D == DP) return;
        for (int n = threadIdx.x; n < tiles * AT_TILE * CH; n += 256)
            if (((n % CH) ^ at_swz<DP>(n / CH % AT_TILE)) * 8 >= D) *reinterpret_cast<at_u32x4*>(first + n * 8) = at_u32x4{0, 0, 0, 0};
    }
};

template <typename T> __device__ __forceinline__ typename AtEl<T>::x8 at_global_frag(const T* row, int ks, int lane, int D) {
    const int col = 16 * ks + 8 * (lane >> 5);
    typename AtEl<T>::x8 z = {};
    return col < D ? *reinterpret_cast<const typename AtEl<T>::x8*>(row + col) : z;
}

// Which of a row's keys k0 + 8 (r / 4) + r % 4 a mask shows, as bit r.  Bytes are read at keys of the tensor (`last` repeats); where 4
// keys lie side by side in memory and the whole range is inside, four at a time.
struct __attribute__((packed, aligned(1))) AtFour { uint32_t x; };
__device__ __forceinline__ uint32_t at_mask_bits(const uint8_t* row, int64_t sk, int k0, int last, bool four) {
    uint32_t bits = 0;
    if (four) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const uint32_t x = reinterpret_cast<const AtFour*>(row + k0 + 8 * r4)->x;
#pragma unroll
            for (int e = 0; e < 4; ++e) bits |= ((x >> (8 * e)) & 255u ? 1u : 0u) << (4 * r4 + e);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) bits |= (row[(int64_t)min(k0 + 8 * (r >> 2) + (r & 3), last) * sk] ? 1u : 0u) << r;
    }
    return bits;
}
// Hiding is by selects on such bits: with a branch around the byte's load hipcc 7.2 lost the hiding of an accumulator's element 0.
// Bits r of the keys k0 + 8 (r / 4) + r % 4 that lie below lim.
__device__ __forceinline__ uint32_t at_below_bits(int k0, int lim) {
    uint32_t bits = 0;
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) bits |= ((1u << min(max(lim - k0 - 8 * r4, 0), 4)) - 1u) << (4 * r4);
    return bits;
}

// A workgroup's LDS.  The tiles come first: the loads' 16-bit LDS base has to reach them.
template <typename T, int DP> struct AtShared {
    T tiles[2][2][AT_TILE * DP];
    int tops[4];
    float unit4[4];
};
template <typename T, int DP, bool MASKED> struct AtSharedKeys {
    T tiles[2][2][AT_TILE * DP];
    float lse[2][AT_TILE], delta[2][AT_TILE];
    int lim[2][AT_TILE];
    int64_t mask[MASKED ? 2 : 1][MASKED ? AT_TILE : 1];
    float unit4[4];
};

// ------------------------------------------------------------------------------------------------------------------- forward
template <typename T, int DP, bool MASKED>
__global__ __launch_bounds__(256, 2) void at_fwd_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x8 x8;
    typedef typename AtEl<T>::x4 x4;
    __shared__ __attribute__((aligned(16))) AtShared<T, DP> sh;
    auto& smem = sh.tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int R = a.G * a.Nq, tiles = (R + AT_ROWS - 1) / AT_ROWS;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tile = a.causal ? tiles - 1 - id % tiles : id % tiles; // the long rows of a causal call first
    id /= tiles;
    const int split = id % a.splits;
    id /= a.splits;
    const int kh = id % a.Hk, b = id / a.Hk;

    const int len = a.key_lengths ? min(max(a.key_lengths[b], 0), a.Nk) : a.Nk;
    const int row = tile * AT_ROWS + wave * 32 + c, rowc = min(row, R - 1), g = rowc / a.Nq, i = rowc - g * a.Nq;
    const int head = kh * a.G + g;
    const int lim = row >= R ? 0 : a.causal ? min(len, max(0, i + a.Nk - a.Nq + 1)) : len; // this row sees keys below lim
    const int wave_top = at_wave_max(lim), wave_low = at_wave_min(row < R ? lim : 0x7fffffff);
    int* const tops = sh.tops;
    if (lane == 0) tops[wave] = wave_top;
    __syncthreads();
    const int top = __builtin_amdgcn_readfirstlane(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    const int all = (top + AT_TILE - 1) / AT_TILE, per = (all + a.splits - 1) / a.splits;
    const int t0 = split * per, t1 = min(all, t0 + per);

    const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.k_sb + (int64_t)kh * a.k_sh;
    const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.v_sb + (int64_t)kh * a.v_sh;
    const uint8_t* mrow = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)head * a.m_sh + (int64_t)i * a.m_sq : nullptr;
    const uint8_t* mkey = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)kh * a.G * a.m_sh : nullptr;

    x8 qf[DP / 16];
    {
        const T* qp = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh + (int64_t)i * a.q_sn;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) qf[ks] = at_global_frag<T>(qp, ks, lane, a.D);
    }
    at_f32x16 ot[DP / 32] = {};
    float m_run = -INFINITY, l_run = 0.f; // running maximum (raw scores), this lane's share of the sum

    auto load = [&](int t, int buf) {
        AtTile<T, DP>::load(smem[buf][0], kb + (int64_t)t * AT_TILE * a.k_sn, (int)a.k_sn, len - t * AT_TILE, a.D);
        AtTile<T, DP>::load(smem[buf][1], vb + (int64_t)t * AT_TILE * a.v_sn, (int)a.v_sn, len - t * AT_TILE, a.D);
    };
    AtTile<T, DP>::pad(smem[0][0], 4, a.D);
    if (t0 < t1) load(t0, 0);
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        at_landed();
        if (MASKED && a.mask_by_key) {
            AtTile<T, DP>::hide(smem[buf][0], mkey + (int64_t)t * AT_TILE * a.m_sk, a.m_sk, len - t * AT_TILE);
            AtTile<T, DP>::hide(smem[buf][1], mkey + (int64_t)t * AT_TILE * a.m_sk, a.m_sk, len - t * AT_TILE);
        }
        __syncthreads(); // tile t is in place, and nobody reads the other buffer any more
        const T *tk = smem[buf][0], *tv = smem[buf][1];
        if (t + 1 < t1) load(t + 1, buf ^ 1);
        if (t * AT_TILE < wave_top) {
            at_f32x16 st[2] = {};
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
                for (int n = 0; n < 2; ++n) st[n] = AtEl<T>::mfma(at_rowfrag<T, DP>(tk, 32 * n, ks, lane), qf[ks], st[n]);
            if (MASKED || (t + 1) * AT_TILE > wave_low) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int k0 = t * AT_TILE + 32 * n + 4 * h;
                    uint32_t see = at_below_bits(k0, lim);
                    if (MASKED) see &= at_mask_bits(mrow, a.m_sk, k0, a.Nk - 1, a.m_sk == 1 && (t + 1) * AT_TILE <= a.Nk);
#pragma unroll
                    for (int r = 0; r < 16; ++r) st[n][r] = (see >> r) & 1u ? st[n][r] : -INFINITY;
                }
            }
            float top0 = m_run, top1 = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                top0 = at_max3(top0, st[0][r], st[0][r + 1]);
                top1 = at_max3(top1, st[1][r], st[1][r + 1]);
            }
            top0 = fmaxf(top0, top1);
            const float m_new = fmaxf(top0, at_other_half(top0));
            const float m_use = m_new == -INFINITY ? 0.f : m_new, neg_m = -m_use * a.scale_log2e;
            if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0ull) { // no row's maximum rose: the factor is 1
                const float alpha = __builtin_amdgcn_exp2f((m_run - m_use) * a.scale_log2e);
                l_run *= alpha;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) ot[db] *= alpha;
            }
            m_run = m_new;
            float ps[4] = {0.f, 0.f, 0.f, 0.f};
            x8 pf[2][2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[n][r], a.scale_log2e, neg_m));
                    ps[r & 3] += p;
                    pf[n][r >> 3][r & 7] = (T)p; // rounded to the operands' type for the second product; the sum keeps 32 bits
                }
            l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) ot[db] = AtEl<T>::mfma(at_colfrag<T, DP>(tv, 32 * n + 16 * s, db, lane), pf[n][s], ot[db]);
        }
    }

    const float l = l_run + at_other_half(l_run);
    if (row >= R) return;
    const int64_t at = ((int64_t)b * a.Hk + kh) * R + row; // = (b H + head) Nq + i
    if (a.splits > 1) {
        const int64_t slot = (int64_t)split * a.B * a.Hk * R + at;
        if (h == 0) { a.part_ml[2 * slot] = m_run; a.part_ml[2 * slot + 1] = l; }
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int d = 32 * db + 2 * r + 4 * h;
                if (d < a.D) *reinterpret_cast<at_f32x4*>(a.part_o + slot * a.D + d) = at_f32x4{ot[db][r], ot[db][r + 1], ot[db][r + 2], ot[db][r + 3]};
            }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (h == 0) a.lse[at] = l == 0.f ? -INFINITY : m_run * a.scale + logf(l);
    T* op = static_cast<T*>(a.out) + (((int64_t)b * a.Nq + i) * a.H + head) * a.D;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * db + 2 * r + 4 * h;
            x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (T)(ot[db][r + e] * inv);
            if (d < a.D) *reinterpret_cast<x4*>(op + d) = o;
        }
}

// Joins the parts of a row that several workgroups computed: 32 lanes a row, 4 elements a lane.
template <typename T>
__global__ __launch_bounds__(256) void at_join_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x4 x4;
    const int64_t rows = (int64_t)a.B * a.H * a.Nq, at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (at >= rows) return;
    const int d = (threadIdx.x & 31) * 4;
    float m = -INFINITY;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[2 * (s * rows + at)]);
    const float m_use = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    at_f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const float w = __builtin_amdgcn_exp2f((a.part_ml[2 * (s * rows + at)] - m_use) * a.scale_log2e);
        l += w * a.part_ml[2 * (s * rows + at) + 1];
        if (d < a.D) o += w * *reinterpret_cast<const at_f32x4*>(a.part_o + (s * rows + at) * a.D + d);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (d == 0) a.lse[at] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
    if (d >= a.D) return;
    const int64_t bh = at / a.Nq;
    const int i = (int)(at - bh * a.Nq), head = (int)(bh % a.H);
    x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(o[e] * inv);
    *reinterpret_cast<x4*>(static_cast<T*>(a.out) + (((bh / a.H) * a.Nq + i) * a.H + head) * a.D + d) = y;
}

// ------------------------------------------------------------------------------------------------------------------ backward
// delta_i = <dO_i, o_i>, 16 lanes a row; and the largest |dO| of each block of 16 rows, from which the fp16 kernels take the
// power of two that brings dS into fp16's range.
#define AT_DELTA_ROWS 16
template <typename T>
__global__ __launch_bounds__(256) void at_delta_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x8 x8;
    const int64_t rows = (int64_t)a.B * a.H * a.Nq, at = (int64_t)blockIdx.x * AT_DELTA_ROWS + (threadIdx.x >> 4);
    const int d = (threadIdx.x & 15) * 8;
    float sum = 0.f, top = 0.f;
    if (at < rows && d < a.D) {
        const int64_t bh = at / a.Nq, i = at - bh * a.Nq, head = bh % a.H, b = bh / a.H;
        const x8 o = *reinterpret_cast<const x8*>(static_cast<const T*>(a.out_in) + ((b * a.Nq + i) * a.H + head) * a.D + d);
        const x8 g = *reinterpret_cast<const x8*>(static_cast<const T*>(a.dout) + b * a.g_sb + head * a.g_sh + i * a.g_sn + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) { sum += (float)o[e] * (float)g[e]; top = fmaxf(top, fabsf((float)g[e])); }
    }
    for (int o = 8; o; o >>= 1) { sum += __shfl_xor(sum, o); top = fmaxf(top, __shfl_xor(top, o)); }
    if (at < rows && (threadIdx.x & 15) == 0) a.delta[at] = sum;
    __shared__ float tops[AT_DELTA_ROWS];
    if ((threadIdx.x & 15) == 0) tops[threadIdx.x >> 4] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < AT_DELTA_ROWS; ++i) top = fmaxf(top, tops[i]);
        a.amax[blockIdx.x] = top;
    }
}

// fp16 only: 2^e with 2^e max|dO| in [1, 2), over the rows of this key head.  dS = P (dP - delta) of a small gradient would fall
// below fp16's normal range (6e-5), of a scaled loss leave it; both are linear in dO.  bf16 has fp32's range and needs none.
template <typename T> __device__ __forceinline__ float at_grad_unit(const AttendArgs& a, int b, int kh, float* shared4) {
    if (sizeof(T) == 2 && !__is_same(T, _Float16)) return 1.f;
    const int64_t R = (int64_t)a.G * a.Nq, first = ((int64_t)b * a.Hk + kh) * R;
    if (R == 0) return 1.f;
    float top = 0.f;
    for (int64_t n = first / AT_DELTA_ROWS + threadIdx.x; n <= (first + R - 1) / AT_DELTA_ROWS; n += 256) top = fmaxf(top, a.amax[n]);
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) shared4[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(shared4[0], shared4[1]), fmaxf(shared4[2], shared4[3]));
    if (!(top > 0.f) || top == INFINITY) return 1.f;
    return __uint_as_float((254u - (__float_as_uint(top) >> 23)) << 23);
}

// dQ: a wave owns 32 rows and walks the keys that they see.
template <typename T, int DP, bool MASKED>
__global__ __launch_bounds__(256, 2) void at_bwd_rows_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x8 x8;
    typedef typename AtEl<T>::x4 x4;
    __shared__ __attribute__((aligned(16))) AtShared<T, DP> sh;
    auto& smem = sh.tiles;
    int* const tops = sh.tops;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int R = a.G * a.Nq, tiles = (R + AT_ROWS - 1) / AT_ROWS;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tile = a.causal ? tiles - 1 - id % tiles : id % tiles;
    id /= tiles;
    const int kh = id % a.Hk, b = id / a.Hk;
    const float unit = at_grad_unit<T>(a, b, kh, sh.unit4);

    const int len = a.key_lengths ? min(max(a.key_lengths[b], 0), a.Nk) : a.Nk;
    const int row = tile * AT_ROWS + wave * 32 + c, rowc = min(row, R - 1), g = rowc / a.Nq, i = rowc - g * a.Nq;
    const int head = kh * a.G + g;
    const int lim = row >= R ? 0 : a.causal ? min(len, max(0, i + a.Nk - a.Nq + 1)) : len;
    const int wave_top = at_wave_max(lim), wave_low = at_wave_min(row < R ? lim : 0x7fffffff);
    if (lane == 0) tops[wave] = wave_top;
    __syncthreads();
    const int t1 = (__builtin_amdgcn_readfirstlane(max(max(tops[0], tops[1]), max(tops[2], tops[3]))) + AT_TILE - 1) / AT_TILE;

    const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.k_sb + (int64_t)kh * a.k_sh;
    const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.v_sb + (int64_t)kh * a.v_sh;
    const uint8_t* mrow = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)head * a.m_sh + (int64_t)i * a.m_sq : nullptr;
    const uint8_t* mkey = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)kh * a.G * a.m_sh : nullptr;
    x8 qf[DP / 16], gf[DP / 16];
    {
        const T* qp = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh + (int64_t)i * a.q_sn;
        const T* gp = static_cast<const T*>(a.dout) + (int64_t)b * a.g_sb + (int64_t)head * a.g_sh + (int64_t)i * a.g_sn;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) { qf[ks] = at_global_frag<T>(qp, ks, lane, a.D); gf[ks] = at_global_frag<T>(gp, ks, lane, a.D); }
    }
    const int64_t at = ((int64_t)b * a.Hk + kh) * R + rowc;
    const float lse = a.lse[at], neg_lse = lse == -INFINITY ? -INFINITY : -lse * 1.4426950408889634f, neg_delta = -a.delta[at] * unit;
    at_f32x16 acc[DP / 32] = {};

    auto load = [&](int t, int buf) {
        AtTile<T, DP>::load(smem[buf][0], kb + (int64_t)t * AT_TILE * a.k_sn, (int)a.k_sn, len - t * AT_TILE, a.D);
        AtTile<T, DP>::load(smem[buf][1], vb + (int64_t)t * AT_TILE * a.v_sn, (int)a.v_sn, len - t * AT_TILE, a.D);
    };
    AtTile<T, DP>::pad(smem[0][0], 4, a.D);
    if (t1 > 0) load(0, 0);
    for (int t = 0; t < t1; ++t) {
        const int buf = t & 1;
        at_landed();
        if (MASKED && a.mask_by_key) {
            AtTile<T, DP>::hide(smem[buf][0], mkey + (int64_t)t * AT_TILE * a.m_sk, a.m_sk, len - t * AT_TILE);
            AtTile<T, DP>::hide(smem[buf][1], mkey + (int64_t)t * AT_TILE * a.m_sk, a.m_sk, len - t * AT_TILE);
        }
        __syncthreads(); // tile t is in place, and nobody reads the other buffer any more
        const T *tk = smem[buf][0], *tv = smem[buf][1];
        if (t + 1 < t1) load(t + 1, buf ^ 1);
        if (t * AT_TILE < wave_top) {
            at_f32x16 st[2] = {}, dp[2] = {};
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    st[n] = AtEl<T>::mfma(at_rowfrag<T, DP>(tk, 32 * n, ks, lane), qf[ks], st[n]);
                    dp[n] = AtEl<T>::mfma(at_rowfrag<T, DP>(tv, 32 * n, ks, lane), gf[ks], dp[n]);
                }
            if (MASKED || (t + 1) * AT_TILE > wave_low) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int k0 = t * AT_TILE + 32 * n + 4 * h;
                    uint32_t see = at_below_bits(k0, lim);
                    if (MASKED) see &= at_mask_bits(mrow, a.m_sk, k0, a.Nk - 1, a.m_sk == 1 && (t + 1) * AT_TILE <= a.Nk);
#pragma unroll
                    for (int r = 0; r < 16; ++r) st[n][r] = (see >> r) & 1u ? st[n][r] : -INFINITY;
                }
            }
            x8 ds[2][2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[n][r], a.scale_log2e, neg_lse));
                    ds[n][r >> 3][r & 7] = (T)(p * fmaf(dp[n][r], unit, neg_delta));
                }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) acc[db] = AtEl<T>::mfma(at_colfrag<T, DP>(tk, 32 * n + 16 * s, db, lane), ds[n][s], acc[db]);
        }
    }
    if (row >= R) return;
    const float f = a.scale / unit;
    T* op = static_cast<T*>(a.dq) + (int64_t)b * a.dq_sb + (int64_t)head * a.dq_sh + (int64_t)i * a.dq_sn;
    const bool blind = lse == -INFINITY; // sees nothing: a gradient of zero whatever the (unread) products gave
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * db + 2 * r + 4 * h;
            x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = blind ? (T)0.f : (T)(acc[db][r + e] * f);
            if (d < a.D) *reinterpret_cast<x4*>(op + d) = o;
        }
}

// dK, dV: a wave owns 32 keys and walks the rows that may see them.
template <typename T, int DP, bool MASKED>
__global__ __launch_bounds__(256, DP == 64 ? 2 : 1) void at_bwd_keys_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x8 x8;
    typedef typename AtEl<T>::x4 x4;
    __shared__ __attribute__((aligned(16))) AtSharedKeys<T, DP, MASKED> sh;
    auto& smem = sh.tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int R = a.G * a.Nq, tiles = (a.Nk + AT_ROWS - 1) / AT_ROWS, off = a.Nk - a.Nq;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tile = id % tiles; // causal: the first keys are seen by most rows, the long ones come first as they are
    id /= tiles;
    const int kh = id % a.Hk, b = id / a.Hk;
    const float unit = at_grad_unit<T>(a, b, kh, sh.unit4);
    const int len = a.key_lengths ? min(max(a.key_lengths[b], 0), a.Nk) : a.Nk;
    const int k0 = tile * AT_ROWS, wave_k0 = k0 + __builtin_amdgcn_readfirstlane(wave) * 32, key = wave_k0 + c;

    at_f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
    if (k0 < len) {
        x8 kf[DP / 16], vf[DP / 16];
        const int keyc = min(key, len - 1);
        {
            const T* kp = static_cast<const T*>(a.k) + (int64_t)b * a.k_sb + (int64_t)kh * a.k_sh + (int64_t)keyc * a.k_sn;
            const T* vp = static_cast<const T*>(a.v) + (int64_t)b * a.v_sb + (int64_t)kh * a.v_sh + (int64_t)keyc * a.v_sn;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) { kf[ks] = at_global_frag<T>(kp, ks, lane, a.D); vf[ks] = at_global_frag<T>(vp, ks, lane, a.D); }
        }
        const T* qb = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)kh * a.G * a.q_sh;
        const T* gb = static_cast<const T*>(a.dout) + (int64_t)b * a.g_sb + (int64_t)kh * a.G * a.g_sh;
        const int64_t at0 = ((int64_t)b * a.Hk + kh) * R;
        const uint8_t* mkey = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)kh * a.G * a.m_sh + (int64_t)keyc * a.m_sk : nullptr;
        if (MASKED && a.mask_by_key && !mkey[0]) {
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) { kf[ks] = x8{}; vf[ks] = x8{}; }
        }
        // the tiles: head by head, from the first query that sees a key of this workgroup
        const int i_first = a.causal ? max(0, k0 - off) : 0, per_head = a.Nq > i_first ? (a.Nq - i_first + AT_TILE - 1) / AT_TILE : 0, t1 = a.G * per_head;
        int g_next = 0, i_next = i_first;
        float n_lse = 0.f, n_delta = 0.f;
        int n_lim = -1;
        int64_t n_mask = 0;
        auto load = [&](int buf) { // tile (g_next, i_next)
            AtTile<T, DP>::load(smem[buf][0], qb + (int64_t)g_next * a.q_sh + (int64_t)i_next * a.q_sn, (int)a.q_sn, a.Nq - i_next, a.D);
            AtTile<T, DP>::load(smem[buf][1], gb + (int64_t)g_next * a.g_sh + (int64_t)i_next * a.g_sn, (int)a.g_sn, a.Nq - i_next, a.D);
            if (threadIdx.x < AT_TILE) {
                const int i = i_next + threadIdx.x, ic = min(i, a.Nq - 1);
                const int64_t at = at0 + (int64_t)g_next * a.Nq + ic;
                n_lse = a.lse[at]; // as they are: worked on in note(), when they have long arrived
                n_delta = a.delta[at];
                n_lim = i >= a.Nq ? -1 : a.causal ? min(len - 1, i + off) : len - 1; // the last key that the row sees
                if (MASKED) n_mask = (int64_t)g_next * a.m_sh + (int64_t)ic * a.m_sq;
            }
        };
        auto note = [&](int buf) {
            if (threadIdx.x < AT_TILE) {
                sh.lse[buf][threadIdx.x] = n_lse == -INFINITY ? -INFINITY : -n_lse * 1.4426950408889634f;
                sh.delta[buf][threadIdx.x] = -n_delta * unit;
                sh.lim[buf][threadIdx.x] = n_lim;
                if (MASKED) sh.mask[buf][threadIdx.x] = n_mask;
            }
        };
        AtTile<T, DP>::pad(smem[0][0], 4, a.D);
        if (t1 > 0) { load(0); note(0); }
        for (int t = 0; t < t1; ++t) {
            const int buf = t & 1, i0 = i_next;
            i_next += AT_TILE;
            if (i_next >= a.Nq) { i_next = i_first; ++g_next; }
            at_landed();
            __syncthreads();
            const T *tq = smem[buf][0], *tg = smem[buf][1];
            if (t + 1 < t1) load(buf ^ 1);
            // unless every row of the tile sees every key of the wave
            const bool edge = MASKED || i0 + AT_TILE > a.Nq || wave_k0 + 32 > len || (a.causal && i0 + off < wave_k0 + 31);
            at_f32x16 st[2] = {}, dp[2] = {};
            x8 pf[2][2], df[2][2], gt[2][DP / 32], qt[2][DP / 32];
            auto scores = [&](int n) {
                x8 qa[DP / 16], ga[DP / 16];
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) { qa[ks] = at_rowfrag<T, DP>(tq, 32 * n, ks, lane); ga[ks] = at_rowfrag<T, DP>(tg, 32 * n, ks, lane); }
                if (DP == 128) __builtin_amdgcn_sched_barrier(0); // all reads under way before the first product
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) {
                    st[n] = AtEl<T>::mfma(qa[ks], kf[ks], st[n]);
                    dp[n] = AtEl<T>::mfma(ga[ks], vf[ks], dp[n]);
                }
            };
            auto hide = [&](int n) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int q = 32 * n + 8 * (r >> 2) + 4 * h + (r & 3);
                    bool on = key <= sh.lim[buf][q];
                    if (MASKED) on = on & (mkey[sh.mask[buf][q]] != 0);
                    st[n][r] = on ? st[n][r] : -INFINITY;
                }
            };
            auto probs = [&](int n) {
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int q0 = 32 * n + 8 * r4 + 4 * h;
                    const at_f32x4 nl = *reinterpret_cast<const at_f32x4*>(&sh.lse[buf][q0]), nd = *reinterpret_cast<const at_f32x4*>(&sh.delta[buf][q0]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * r4 + e;
                        const float p = __builtin_amdgcn_exp2f(fmaf(st[n][r], a.scale_log2e, nl[e]));
                        pf[n][r >> 3][r & 7] = (T)p;
                        df[n][r >> 3][r & 7] = (T)(p * fmaf(dp[n][r], unit, nd[e]));
                    }
                }
            };
            auto columns = [&](int n) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) {
                        gt[s][db] = at_colfrag<T, DP>(tg, 32 * n + 16 * s, db, lane);
                        qt[s][db] = at_colfrag<T, DP>(tq, 32 * n + 16 * s, db, lane);
                    }
            };
            auto gradients = [&](int n) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) {
                        dv[db] = AtEl<T>::mfma(gt[s][db], pf[n][s], dv[db]);
                        dk[db] = AtEl<T>::mfma(qt[s][db], df[n][s], dk[db]);
                    }
            };
            if (DP == 128) {
                // 128 accumulators and 64 registers of K and V leave one wave a SIMD, whose own products have to cover its arithmetic:
                // the scores of the second 32 rows run while the probabilities of the first are worked out, and so on.  4096 tokens x
                // 16 heads: 594 -> 520 us for the whole backward pass against one step after the other.
                scores(0);
                if (edge) hide(0);
                __builtin_amdgcn_sched_barrier(0);
                scores(1);
                probs(0);
                columns(0);
                if (edge) hide(1);
                __builtin_amdgcn_sched_barrier(0);
                gradients(0);
                probs(1);
                columns(1);
                __builtin_amdgcn_sched_barrier(0);
                gradients(1);
            } else { // three waves a SIMD cover each other; the order above costs registers and one of them (1070 -> 1258 us at 8192 x 16)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    scores(n);
                    if (edge) hide(n);
                    probs(n);
                    columns(n);
                    gradients(n);
                }
            }
            if (t + 1 < t1) note(buf ^ 1);
        }
    }
    if (key >= a.Nk) return;
    const float f = a.scale / unit;
    T* kp = static_cast<T*>(a.dk) + (int64_t)b * a.dk_sb + (int64_t)kh * a.dk_sh + (int64_t)key * a.dk_sn;
    T* vp = static_cast<T*>(a.dv) + (int64_t)b * a.dv_sb + (int64_t)kh * a.dv_sh + (int64_t)key * a.dv_sn;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * db + 2 * r + 4 * h;
            x4 x, y;
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[e] = (T)(dk[db][r + e] * f); y[e] = (T)dv[db][r + e]; }
            if (d < a.D) { *reinterpret_cast<x4*>(kp + d) = x; *reinterpret_cast<x4*>(vp + d) = y; }
        }
}

// -------------------------------------------------------------------------------------------------------------------- launches
// Parts that a row's keys are cut into: enough workgroups for two on each of the 256 CUs, at least two tiles of keys a part.
static int at_splits(int64_t B, int Hk, int64_t R, int Nk) {
    const int64_t groups = B * Hk * ceil_div(R, AT_ROWS);
    const int64_t tiles = ceil_div(Nk, AT_TILE);
    int64_t s = ceil_div(512, groups);
    if (s > tiles / 2) s = tiles / 2;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

static int at_check(int dtype, int B, int H, int Hk, int Nq, int Nk, int D, float scale) {
    if (dtype != 0 && dtype != 2) return ADK_EUNSUPPORTED;
    if (B < 0 || H < 1 || Hk < 1 || H % Hk || Nq < 0 || Nk < 0) return ADK_EINVAL;
    if (D < 8 || D > 128 || (D & 7)) return ADK_EUNSUPPORTED;
    if (!(scale > 0.f) || !(scale < INFINITY)) return ADK_EINVAL;
    const int64_t R = (int64_t)(H / Hk) * Nq; // row and key numbers, and a grid, in 31 bits
    if (R > 0x7fffff00ll || Nk > 0x7fffff00 || (int64_t)B * Hk * ceil_div(R > Nk ? R : Nk, AT_ROWS) > 0x1ffffff) return ADK_EUNSUPPORTED;
    if ((int64_t)B * H * Nq > 0x7fffff00ll * 8) return ADK_EUNSUPPORTED;
    return 0;
}

// s: strides (batch, head, token)
static int at_tensor(const void* p, const int64_t* s) {
    if (!p || ((uintptr_t)p & 15) || ((s[0] | s[1] | s[2]) & 7)) return ADK_EINVAL;
    return s[2] < 0 || s[2] >= (1 << 24) ? ADK_EUNSUPPORTED : 0; // 64 rows of a tile in 32-bit byte offsets
}

#define AT_LAUNCH3(KERNEL, T, GRID)                                                                                             \
    do {                                                                                                                        \
        if (a.D <= 64) {                                                                                                        \
            if (a.mask) hipLaunchKernelGGL((KERNEL<T, 64, true>), dim3(GRID), dim3(256), 0, stream, a);                         \
            else hipLaunchKernelGGL((KERNEL<T, 64, false>), dim3(GRID), dim3(256), 0, stream, a);                               \
        } else {                                                                                                                \
            if (a.mask) hipLaunchKernelGGL((KERNEL<T, 128, true>), dim3(GRID), dim3(256), 0, stream, a);                        \
            else hipLaunchKernelGGL((KERNEL<T, 128, false>), dim3(GRID), dim3(256), 0, stream, a);                              \
        }                                                                                                                       \
    } while (0)

template <typename T> static int at_fwd(const AttendArgs& a, hipStream_t stream) {
    const int64_t R = (int64_t)a.G * a.Nq;
    AT_LAUNCH3(at_fwd_kernel, T, (unsigned)(ceil_div(R, AT_ROWS) * a.B * a.Hk * a.splits));
    if (a.splits > 1) hipLaunchKernelGGL((at_join_kernel<T>), dim3((unsigned)ceil_div((int64_t)a.B * a.H * a.Nq, 8)), dim3(256), 0, stream, a);
    ADK_RETURN_LAST_ERROR();
}

template <typename T> static int at_bwd(const AttendArgs& a, hipStream_t stream) {
    const int64_t R = (int64_t)a.G * a.Nq, rows = (int64_t)a.B * a.H * a.Nq;
    if (rows) {
        hipLaunchKernelGGL((at_delta_kernel<T>), dim3((unsigned)ceil_div(rows, AT_DELTA_ROWS)), dim3(256), 0, stream, a);
        AT_LAUNCH3(at_bwd_rows_kernel, T, (unsigned)(ceil_div(R, AT_ROWS) * a.B * a.Hk));
    }
    if (a.Nk) AT_LAUNCH3(at_bwd_keys_kernel, T, (unsigned)(ceil_div(a.Nk, AT_ROWS) * a.B * a.Hk));
    ADK_RETURN_LAST_ERROR();
}

// s: strides of q, k, v (batch, head, token each), then of the mask (batch, head, query, key)
static void at_fill(AttendArgs& a, const void* q, const void* k, const void* v, const float* lse, const int* key_lengths, const uint8_t* mask, int B, int H, int Hk,
                    int Nq, int Nk, int D, const int64_t* s, float scale, int causal) {
    a.q = q; a.k = k; a.v = v; a.lse = const_cast<float*>(lse);
    a.key_lengths = key_lengths; a.mask = Nq && Nk ? mask : nullptr;
    a.B = B; a.H = H; a.Hk = Hk; a.G = H / Hk; a.Nq = Nq; a.Nk = Nk; a.D = D; a.splits = 1; a.causal = causal;
    a.q_sb = s[0]; a.q_sh = s[1]; a.q_sn = s[2];
    a.k_sb = s[3]; a.k_sh = s[4]; a.k_sn = s[5];
    a.v_sb = s[6]; a.v_sh = s[7]; a.v_sn = s[8];
    if (mask) { a.m_sb = s[9]; a.m_sh = s[10]; a.m_sq = s[11]; a.m_sk = s[12]; }
    a.mask_by_key = a.mask && a.m_sq == 0 && (a.m_sh == 0 || a.G == 1);
    a.scale = scale; a.scale_log2e = scale * 1.4426950408889634f;
}

} // namespace adk

extern "C" int64_t adk_attend_fwd_workspace_bytes(int B, int H, int Hk, int Nq, int Nk, int D)
{
    const int e = adk::at_check(0, B, H, Hk, Nq, Nk, D, 1.f);
    if (e) return e;
    const int64_t rows = (int64_t)B * H * Nq;
    const int s = rows ? adk::at_splits(B, Hk, (int64_t)(H / Hk) * Nq, Nk) : 1;
    return s > 1 ? s * rows * (D + 2) * 4 : 0;
}

extern "C" int adk_attend_fwd(const void* q, const void* k, const void* v, void* out, float* lse, const int32_t* key_lengths, const uint8_t* mask, int dtype, int B, int H,
                              int Hk, int Nq, int Nk, int D, const int64_t* strides, float scale, int causal, void* ws, int64_t ws_bytes, hipStream_t stream)
{
    int e = adk::at_check(dtype, B, H, Hk, Nq, Nk, D, scale);
    if (e) return e;
    if ((int64_t)B * Nq == 0) return 0;
    if (!strides || !out || ((uintptr_t)out & 7) || !lse) return ADK_EINVAL;
    if ((e = adk::at_tensor(q, strides)) || (Nk && ((e = adk::at_tensor(k, strides + 3)) || (e = adk::at_tensor(v, strides + 6))))) return e;
    adk::AttendArgs a = {};
    adk::at_fill(a, q, k, v, lse, key_lengths, mask, B, H, Hk, Nq, Nk, D, strides, scale, causal);
    a.out = out;
    const int64_t need = adk_attend_fwd_workspace_bytes(B, H, Hk, Nq, Nk, D);
    if (need > 0) {
        if (!ws || ws_bytes < need || ((uintptr_t)ws & 15)) return ADK_EWORKSPACE;
        a.splits = adk::at_splits(B, Hk, (int64_t)a.G * Nq, Nk);
        a.part_o = static_cast<float*>(ws);
        a.part_ml = a.part_o + (int64_t)a.splits * B * H * Nq * D;
    }
    return dtype == 0 ? adk::at_fwd<_Float16>(a, stream) : adk::at_fwd<__bf16>(a, stream);
}

extern "C" int64_t adk_attend_bwd_workspace_bytes(int B, int H, int Hk, int Nq, int Nk, int D)
{
    const int e = adk::at_check(0, B, H, Hk, Nq, Nk, D, 1.f);
    if (e) return e;
    const int64_t rows = (int64_t)B * H * Nq;
    return 4 * (rows + adk::ceil_div(rows, AT_DELTA_ROWS));
}

extern "C" int adk_attend_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse, const int32_t* key_lengths,
                              const uint8_t* mask, int dtype, int B, int H, int Hk, int Nq, int Nk, int D, const int64_t* strides, float scale, int causal, void* dq,
                              void* dk, void* dv, void* ws, int64_t ws_bytes, hipStream_t stream)
{
    int e = adk::at_check(dtype, B, H, Hk, Nq, Nk, D, scale);
    if (e) return e;
    if (B == 0 || (Nq == 0 && Nk == 0)) return 0;
    if (!strides) return ADK_EINVAL;
    const int64_t* s = strides + 13; // of dout, dq, dk, dv
    if (Nq && (!out || ((uintptr_t)out & 15) || !lse)) return ADK_EINVAL;
    if (Nq && ((e = adk::at_tensor(q, strides)) || (e = adk::at_tensor(dout, s)) || (e = adk::at_tensor(dq, s + 3)))) return e;
    if (Nk && ((e = adk::at_tensor(k, strides + 3)) || (e = adk::at_tensor(v, strides + 6)) || (e = adk::at_tensor(dk, s + 6)) || (e = adk::at_tensor(dv, s + 9)))) return e;
    adk::AttendArgs a = {};
    adk::at_fill(a, q, k, v, lse, key_lengths, mask, B, H, Hk, Nq, Nk, D, strides, scale, causal);
    a.dout = dout; a.out_in = out; a.dq = dq; a.dk = dk; a.dv = dv;
    a.g_sb = s[0]; a.g_sh = s[1]; a.g_sn = s[2];
    a.dq_sb = s[3]; a.dq_sh = s[4]; a.dq_sn = s[5];
    a.dk_sb = s[6]; a.dk_sh = s[7]; a.dk_sn = s[8];
    a.dv_sb = s[9]; a.dv_sh = s[10]; a.dv_sn = s[11];
    const int64_t rows = (int64_t)B * H * Nq;
    if (rows) {
        if (!ws || ws_bytes < adk_attend_bwd_workspace_bytes(B, H, Hk, Nq, Nk, D) || ((uintptr_t)ws & 15)) return ADK_EWORKSPACE;
        a.delta = static_cast<float*>(ws);
        a.amax = a.delta + rows;
    }
    return dtype == 0 ? adk::at_bwd<_Float16>(a, stream) : adk::at_bwd<__bf16>(a, stream);
}
