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
// Three shapes.  Wide: a workgroup owns 128 rows (or keys), 32 a wave, and its four waves share tiles of 64 keys (or rows).  Narrow, for
// calls too small to fill the chip so: a workgroup owns 32, and each wave walks every fourth tile of 32 with LDS tiles of its own and
// no barrier; the four partial results are joined through LDS at the end, in a fixed order.  Half, for the backward pass between the two: it
// owns 64, two waves share every second tile of 32, and two partial results are joined; its tiles are small enough for two workgroups a CU.
// Where even these are few for what they walk (a token over a long cache, a few keys that thousands of queries read), the walk is cut
// into parts whose 32-bit results a last launch adds in their order.
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
    uint32_t* tops;         // fp16: from each block of at_delta_kernel, as at_top_word has them
    float *part_dq, *part_dk, *part_dv; // [row_splits, B, H, Nq, D], [key_splits, B, Hk, Nk, D] where there are several
    uint32_t *by_row, *by_key; // the mask's bits, as at_mask_bits writes them
    const int* key_lengths; // [B] or null
    const uint8_t* mask;    // or null
    int B, H, Hk, G, Nq, Nk, D, splits, causal, mask_by_key, mask_rows, delta_blocks, unit_blocks, row_splits, key_splits;
    int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn, g_sb, g_sh, g_sn; // element strides: batch, head, token
    int64_t dq_sb, dq_sh, dq_sn, dk_sb, dk_sh, dk_sn, dv_sb, dv_sh, dv_sn;
    int64_t m_sb, m_sh, m_sq, m_sk;
    float scale, scale_log2e;
};

// A shape's numbers.
enum { AT_WIDE = 0, AT_NARROW = 1, AT_HALF = 2 };
template <int SHAPE> struct AtShape {
    static constexpr int WAVES = SHAPE == AT_WIDE ? 4 : SHAPE == AT_HALF ? 2 : 1; // waves that share a tile
    static constexpr int STREAMS = 4 / WAVES;                                     // tiles in work at once
    static constexpr int OWN = 32 * WAVES;                                        // rows (or keys) that a workgroup owns
    static constexpr int TILE = SHAPE == AT_WIDE ? 64 : 32;                       // keys (or rows) of a staged tile
};

template <int DP> __device__ __forceinline__ int at_swz(int row) {
    if (DP == 96) return (row >> 2) & 3; // rows of 192 bytes: 4 of them lie on different quarters of the 64 banks as they are
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

// A tile goes from memory to LDS without passing through registers: each wave instruction moves 64 chunks of 16 bytes
// to consecutive LDS addresses, so the swizzle is in which chunk a lane asks for.  In asm because the compiler waits for the
// builtin's loads before any LDS read; the waits are at_landed() before a tile is read.  The address is a
// uniform base and a 32-bit byte offset (token strides are below 2^24 elements).
__device__ __forceinline__ void at_lds16(uint32_t lds, const void* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
// the wave's tiles are in LDS (all but its last `later` loads), and its reads of earlier ones are done, so that what it loads next
// may take their place
template <int later = 0> __device__ __forceinline__ void at_landed() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(later) : "memory"); }

template <typename T, int DP, int SHAPE> struct AtTile {
    static constexpr int TILE = AtShape<SHAPE>::TILE, WAVES = AtShape<SHAPE>::WAVES, CH = DP / 8, IT = TILE * CH / (64 * WAVES);
    // rows from base on; those past the `rows` (>= 1) that there are repeat the last (they are hidden in the scores, and what lies
    // there is never read); chunks past D are left as they are
    static __device__ __forceinline__ void load(T* tile, const T* base, int sn, int rows, int D) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WAVES, lane = threadIdx.x & 63;
        const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)tile;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (WAVES * i + wave) * 64 + lane, row = at / CH, chunk = (at % CH) ^ at_swz<DP>(row);
            const uint32_t off = (uint32_t)min(row, rows - 1) * (uint32_t)sn * 2u + chunk * 16;
            if (DP == D || chunk * 8 < D) at_lds16(lds + (WAVES * i + wave) * 1024, base, off);
        }
    }
    // a mask that is the same for every query hides a key altogether: zeros, whatever stands there (by the lanes that loaded it)
    static __device__ __forceinline__ void hide(T* tile, const uint8_t* mask, int64_t sk, int rows) {
        const int wave = (threadIdx.x >> 6) % WAVES, lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int row = ((WAVES * i + wave) * 64 + lane) / CH;
            if (!mask[(int64_t)min(row, rows - 1) * sk]) *reinterpret_cast<at_u32x4*>(tile + (WAVES * i + wave) * 512 + lane * 8) = at_u32x4{0, 0, 0, 0};
        }
    }
    // zeros in the chunks past D of the workgroup's tiles, which no load touches
    static __device__ __forceinline__ void pad(T* first, int bufs, int D) {
        if (D == DP) return;
        for (int n = threadIdx.x; n < AtShape<SHAPE>::STREAMS * 2 * bufs * TILE * CH; n += 256)
            if (((n % CH) ^ at_swz<DP>(n / CH % TILE)) * 8 >= D) *reinterpret_cast<at_u32x4*>(first + n * 8) = at_u32x4{0, 0, 0, 0};
        __syncthreads(); // narrow: a wave's tiles are its own from here on
    }
};

template <typename T> __device__ __forceinline__ typename AtEl<T>::x8 at_global_frag(const T* row, int ks, int lane, int D) {
    const int col = 16 * ks + 8 * (lane >> 5);
    typename AtEl<T>::x8 z = {};
    return col < D ? *reinterpret_cast<const typename AtEl<T>::x8*>(row + col) : z;
}

// Which of 32 keys a row sees, bit k for key k0 + k, alike in lanes c and c + 32.  Asked for a tile ahead: lane (h, c) brings the bytes
// of its 16 keys from k0 + 16 h on.  In the wide shape they stay on their way until bits() wants them; in the narrow one the wait for the
// tile's V, which is for all loads, waits for them too.  Where keys lie side by side in memory and all 32
// are inside the tensor that is one load; otherwise bytes, at keys of the tensor (`last` repeats).  (4 loads of 4 bytes in the accumulator's
// order ask for 4 times the cache lines: 517 x 1031 x 12/4 heads, D 80, 43.3 us against 40.6.  Bits packed by a launch before, as for the
// backward pass: 42.0; 16 heads of 4096 x 4096, D 64: 131 against 123.)
struct __attribute__((packed, aligned(1))) AtSixteen { uint32_t x[4]; };
struct AtMask32 {
    uint32_t x[4];
    __device__ __forceinline__ void ask(const uint8_t* row, int64_t sk, int k0, int last, bool together) { // k0: of this lane's 16
        if (together) {
            const AtSixteen v = *reinterpret_cast<const AtSixteen*>(row + k0);
#pragma unroll
            for (int n = 0; n < 4; ++n) x[n] = v.x[n];
        } else {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                x[n] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n] |= (uint32_t)row[(int64_t)min(k0 + 4 * n + e, last) * sk] << (8 * e);
            }
        }
    }
    // 128 for a byte that is not 0: a boolean tensor may be a view of any bytes, of 0 and 255 say (2 % of a masked call: 517 x 1031 x 12/4 heads,
    // D 80, 42.9 -> 43.9 us)
    static __device__ __forceinline__ uint32_t shown(uint32_t x) { return (((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u; }
    __device__ __forceinline__ uint32_t bits() const { // sums of powers of two, times 128
        typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
        const uint32_t lo = __builtin_amdgcn_udot4(shown(x[1]), 0x80402010u, __builtin_amdgcn_udot4(shown(x[0]), 0x08040201u, 0u, false), false);
        const uint32_t hi = __builtin_amdgcn_udot4(shown(x[3]), 0x80402010u, __builtin_amdgcn_udot4(shown(x[2]), 0x08040201u, 0u, false), false);
        const uint32_t mine = lo >> 7 | hi << 1;
        const u32x2 both = __builtin_amdgcn_permlane32_swap(mine, mine, false, false); // lane c's and lane c + 32's
        return both.x | both.y << 16;
    }
};
// Hiding is by selects on such bits: with a branch around the byte's load hipcc 7.2 lost the hiding of an accumulator's element 0.
__device__ __forceinline__ float at_hidden_unless(uint32_t bits, int n, float s) { // s if bit n is set, else -inf
    const uint32_t on = (uint32_t)__builtin_amdgcn_sbfe((int)bits, n, 1);
    return __uint_as_float((__float_as_uint(s) & on) | (0xff800000u & ~on));
}
__device__ __forceinline__ int at_key(int r) { return 8 * (r >> 2) + (r & 3); } // accumulator element r of lane half h has key at_key(r) + 4 h
// Bits k of the 32 numbers k0 + k that lie below lim.
__device__ __forceinline__ uint32_t at_below_bits(int k0, int lim) {
    const int n = lim - k0;
    return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1u;
}

// A workgroup's LDS.  Narrow: when the tiles are done with, their place takes the waves' partial results, 64 lanes a register.
template <typename T, int DP, int SHAPE, int BUFS = 2> struct AtShared {
    T tiles[AtShape<SHAPE>::STREAMS][BUFS][2][AtShape<SHAPE>::TILE * DP]; // stream, buffer, tensor
    int tops[4];
    uint32_t top4[4];
    float m[4][32], l[4][32];
};
template <typename T, int DP, int SHAPE> struct AtSharedKeys {
    static constexpr int S = AtShape<SHAPE>::STREAMS, TILE = AtShape<SHAPE>::TILE;
    T tiles[S][2][2][TILE * DP];
    float lse[S][2][TILE], delta[S][2][TILE];
    uint32_t top4[4];
};

// The sum of `regs` values a lane over the streams' waves that own the same rows (or keys); the wave of stream n gets the values
// n regs / streams + 0 .. regs / streams - 1.
template <int REGS, int SHAPE> __device__ __forceinline__ void at_sum_streams(const float* mine, float* room, float* sum) {
    constexpr int WAVES = AtShape<SHAPE>::WAVES, STREAMS = AtShape<SHAPE>::STREAMS;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < REGS; ++r) room[(wave * REGS + r) * 64 + lane] = mine[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < REGS / STREAMS; ++r) {
        const float* p = room + (wave % WAVES * REGS + wave / WAVES * (REGS / STREAMS) + r) * 64 + lane;
        sum[r] = p[0] + p[WAVES * REGS * 64];
        if (STREAMS == 4) sum[r] += p[2 * REGS * 64] + p[3 * REGS * 64];
    }
}
// The first channel of the four that accumulator values 4 n .. 4 n + 3 hold.
__device__ __forceinline__ int at_channel(int n, int h) { return 32 * (n >> 2) + 8 * (n & 3) + 4 * h; }

// Which tile, part, key head and sequence workgroup `id` of a launch has.  Tiles lie side by side, so that the workgroups of one XCD
// (a consecutive range, by xcd_remap) share K and V in its L2; with lengths the sequences do, because a range of its own would leave the
// XCDs of short ones idle (lengths 1031, 637, 243, 0: as long as with four of 1031).
struct AtWhere { int tile, split, kh, b; };
__device__ __forceinline__ AtWhere at_where(const AttendArgs& a, int id, int tiles, int splits) {
    AtWhere w;
    if (a.key_lengths) { w.b = id % a.B; id /= a.B; }
    w.tile = id % tiles; id /= tiles;
    w.split = id % splits; id /= splits;
    w.kh = id % a.Hk; id /= a.Hk;
    if (!a.key_lengths) w.b = id;
    return w;
}

// ------------------------------------------------------------------------------------------------------------------- forward
template <typename T, int DP, bool MASKED, int SHAPE>
__global__ __launch_bounds__(256, 2) void at_fwd_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x8 x8;
    typedef typename AtEl<T>::x4 x4;
    typedef AtTile<T, DP, SHAPE> Tile;
    constexpr int OWN = AtShape<SHAPE>::OWN, TILE = AtShape<SHAPE>::TILE, STREAMS = AtShape<SHAPE>::STREAMS, SUBS = TILE / 32, BUFS = SHAPE == AT_NARROW ? 1 : 2;
    constexpr bool NARROW = SHAPE == AT_NARROW;
    static_assert(SHAPE != AT_HALF, "the forward has two shapes");
    __shared__ __attribute__((aligned(16))) AtShared<T, DP, SHAPE, BUFS> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31, stream = wave / AtShape<SHAPE>::WAVES, sub = wave % AtShape<SHAPE>::WAVES;
    const int R = a.G * a.Nq, tiles = (R + OWN - 1) / OWN;
    const AtWhere where = at_where(a, xcd_remap(blockIdx.x, gridDim.x), tiles, a.splits);
    const int tile = a.causal ? tiles - 1 - where.tile : where.tile, split = where.split, kh = where.kh, b = where.b; // the long rows of a causal call first

    const int len = a.key_lengths ? min(max(a.key_lengths[b], 0), a.Nk) : a.Nk;
    const int row = tile * OWN + sub * 32 + c, rowc = min(row, R - 1), g = rowc / a.Nq, i = rowc - g * a.Nq;
    const int head = kh * a.G + g;
    const int lim = row >= R ? 0 : a.causal ? min(len, max(0, i + a.Nk - a.Nq + 1)) : len; // this row sees keys below lim
    const int wave_top = at_wave_max(lim), wave_low = at_wave_min(row < R ? lim : 0x7fffffff);
    int top = wave_top;
    if (!NARROW) {
        if (lane == 0) sh.tops[wave] = wave_top;
        __syncthreads();
        top = __builtin_amdgcn_readfirstlane(max(max(sh.tops[0], sh.tops[1]), max(sh.tops[2], sh.tops[3])));
    }
    // parts are cut by the tensor's length, not the sequence's: a short one has fewer of the same size
    const int all = (top + TILE - 1) / TILE, per = ((a.Nk + TILE - 1) / TILE + a.splits - 1) / a.splits;
    const int t0 = split * per, t1 = min(all, t0 + per);
    if (a.splits > 1 && t0 >= t1) { // nothing of these rows' keys: a part that weighs nothing, its sums are not read
        const int r = tile * OWN + threadIdx.x;
        if (threadIdx.x < OWN && r < R) {
            float* ml = a.part_ml + 2 * (((int64_t)split * a.B * a.Hk + (int64_t)b * a.Hk + kh) * R + r);
            ml[0] = -INFINITY;
            ml[1] = 0.f;
        }
        return;
    }

    const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.k_sb + (int64_t)kh * a.k_sh;
    const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.v_sb + (int64_t)kh * a.v_sh;
    const uint8_t* mrow = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)head * a.m_sh + (int64_t)i * a.m_sq : nullptr;
    const uint8_t* mkey = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)kh * a.G * a.m_sh : nullptr;

    auto load_k = [&](int t, int buf) { Tile::load(sh.tiles[stream][buf][0], kb + (int64_t)t * TILE * a.k_sn, (int)a.k_sn, len - t * TILE, a.D); };
    auto load_v = [&](int t, int buf) { Tile::load(sh.tiles[stream][buf][1], vb + (int64_t)t * TILE * a.v_sn, (int)a.v_sn, len - t * TILE, a.D); };
    auto hide = [&](int t, T* tile) {
        if (MASKED && a.mask_by_key) Tile::hide(tile, mkey + (int64_t)t * TILE * a.m_sk, a.m_sk, len - t * TILE);
    };
    AtMask32 raw[MASKED ? SUBS : 1];
    auto ask = [&](int t) {
        if (MASKED)
#pragma unroll
            for (int n = 0; n < SUBS; ++n) raw[n].ask(mrow, a.m_sk, t * TILE + 32 * n + 16 * h, a.Nk - 1, a.m_sk == 1 && (t + 1) * TILE <= a.Nk);
    };
    Tile::pad(sh.tiles[0][0][0], BUFS, a.D);
    if (t0 + stream < t1) { load_k(t0 + stream, 0); load_v(t0 + stream, 0); ask(t0 + stream); }
    x8 qf[DP / 16];
    {
        const T* qp = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh + (int64_t)i * a.q_sn;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) qf[ks] = at_global_frag<T>(qp, ks, lane, a.D);
    }
    at_f32x16 ot[DP / 32] = {};
    float m_run = -INFINITY, l_run = 0.f; // running maximum (raw scores), this lane's share of the sum

    int buf = 0;
    for (int t = t0 + stream; t < t1; t += STREAMS, buf ^= BUFS - 1) {
        T *tk = sh.tiles[stream][buf][0], *tv = sh.tiles[stream][buf][1];
        if (NARROW) { // K is there; V's loads, the last, may still be under way
            at_landed<Tile::IT>();
            hide(t, tk);
        } else {
            at_landed();
            hide(t, tk);
            hide(t, tv);
            __syncthreads(); // tile t is in place, and nobody reads the other buffer any more
        }
        uint32_t seen[SUBS];
#pragma unroll
        for (int n = 0; n < SUBS; ++n) seen[n] = MASKED ? raw[n].bits() : 0;
        if (!NARROW && t + 1 < t1) { load_k(t + 1, buf ^ 1); load_v(t + 1, buf ^ 1); }
        if (t + STREAMS < t1) ask(t + STREAMS);
        if (!NARROW && t * TILE >= wave_top) continue;
        at_f32x16 st[SUBS] = {};
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
            for (int n = 0; n < SUBS; ++n) st[n] = AtEl<T>::mfma(at_rowfrag<T, DP>(tk, 32 * n, ks, lane), qf[ks], st[n]);
        if (MASKED || (t + 1) * TILE > wave_low) {
#pragma unroll
            for (int n = 0; n < SUBS; ++n) {
                uint32_t see = at_below_bits(t * TILE + 32 * n, lim);
                if (MASKED) see &= seen[n];
                see >>= 4 * h;
#pragma unroll
                for (int r = 0; r < 16; ++r) st[n][r] = at_hidden_unless(see, at_key(r), st[n][r]);
            }
        }
        if (NARROW) { // one buffer: K's next tile as soon as this one is read, V's at the end; half the LDS, so twice the waves
            at_landed();
            if (t + STREAMS < t1) load_k(t + STREAMS, 0);
            hide(t, tv);
        }
        float tops[SUBS];
#pragma unroll
        for (int n = 0; n < SUBS; ++n) {
            tops[n] = n ? -INFINITY : m_run;
#pragma unroll
            for (int r = 0; r < 16; r += 2) tops[n] = at_max3(tops[n], st[n][r], st[n][r + 1]);
        }
        const float most = SUBS > 1 ? fmaxf(tops[0], tops[SUBS - 1]) : tops[0];
        const float m_new = fmaxf(most, at_other_half(most));
        const float m_use = m_new == -INFINITY ? 0.f : m_new, neg_m = -m_use * a.scale_log2e;
        if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0ull) { // no row's maximum rose: the factor is 1
            const float alpha = __builtin_amdgcn_exp2f((m_run - m_use) * a.scale_log2e);
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) ot[db] *= alpha;
        }
        m_run = m_new;
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
        x8 pf[SUBS][2];
#pragma unroll
        for (int n = 0; n < SUBS; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = __builtin_amdgcn_exp2f(fmaf(st[n][r], a.scale_log2e, neg_m));
                ps[r & 3] += p;
                pf[n][r >> 3][r & 7] = (T)p; // rounded to the operands' type for the second product; the sum keeps 32 bits
            }
        l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
        for (int n = 0; n < SUBS; ++n)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) ot[db] = AtEl<T>::mfma(at_colfrag<T, DP>(tv, 32 * n + 16 * s, db, lane), pf[n][s], ot[db]);
        if (NARROW && t + STREAMS < t1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load_v(t + STREAMS, 0);
        }
    }

    float l = l_run + at_other_half(l_run), m = m_run;
    const int64_t at = ((int64_t)b * a.Hk + kh) * R + row; // = (b H + head) Nq + i
    const int64_t slot = (int64_t)split * a.B * a.Hk * R + at;
    auto statistics = [&]() {
        if (a.splits > 1) { a.part_ml[2 * slot] = m; a.part_ml[2 * slot + 1] = l; }
        else a.lse[at] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
    };
    auto store = [&](int n, const float* o, float inv) { // four values, n as at_channel's
        const int d = at_channel(n, h);
        if (d >= a.D) return;
        if (a.splits > 1) { *reinterpret_cast<at_f32x4*>(a.part_o + slot * a.D + d) = at_f32x4{o[0], o[1], o[2], o[3]}; return; }
        x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)(o[e] * inv);
        *reinterpret_cast<x4*>(static_cast<T*>(a.out) + (((int64_t)b * a.Nq + i) * a.H + head) * a.D + d) = y;
    };
    float flat[DP / 2];
#pragma unroll
    for (int r = 0; r < DP / 2; ++r) flat[r] = ot[r >> 4][r & 15];
    if (NARROW) {
        if (h == 0) { sh.m[wave][c] = m; sh.l[wave][c] = l; }
        __syncthreads(); // and every wave is done with its tiles
        const float m_own = m;
        m = fmaxf(fmaxf(sh.m[0][c], sh.m[1][c]), fmaxf(sh.m[2][c], sh.m[3][c]));
        const float m_use = m == -INFINITY ? 0.f : m;
        l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l += sh.l[w][c] * __builtin_amdgcn_exp2f((sh.m[w][c] - m_use) * a.scale_log2e);
        const float weight = __builtin_amdgcn_exp2f((m_own - m_use) * a.scale_log2e);
#pragma unroll
        for (int r = 0; r < DP / 2; ++r) flat[r] *= weight;
        float sum[DP / 8];
        at_sum_streams<DP / 2, SHAPE>(flat, reinterpret_cast<float*>(sh.tiles), sum);
        if (row >= R) return;
        if (wave == 0 && h == 0) statistics();
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) store(wave * (DP / 32) + n, sum + 4 * n, inv);
        return;
    }
    if (row >= R) return;
    if (h == 0) statistics();
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) store(n, flat + 4 * n, inv);
}

// Joins the parts of a row that several workgroups computed: 32 lanes a row, 4 elements a lane; lane s brings the statistics of parts s and s + 32.
template <typename T>
__global__ __launch_bounds__(256) void at_join_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x4 x4;
    const int64_t rows = (int64_t)a.B * a.H * a.Nq, at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), atc = at < rows ? at : rows - 1;
    const int s32 = threadIdx.x & 31, d = s32 * 4;
    float ms[2], ls[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int s = s32 + 32 * k;
        ms[k] = s < a.splits ? a.part_ml[2 * (s * rows + atc)] : -INFINITY;
        ls[k] = s < a.splits ? a.part_ml[2 * (s * rows + atc) + 1] : 0.f;
    }
    float m = fmaxf(ms[0], ms[1]);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float m_use = m == -INFINITY ? 0.f : m;
    const float w0 = __builtin_amdgcn_exp2f((ms[0] - m_use) * a.scale_log2e), w1 = __builtin_amdgcn_exp2f((ms[1] - m_use) * a.scale_log2e);
    float l = ls[0] * w0 + ls[1] * w1;
    for (int o = 16; o; o >>= 1) l += __shfl_xor(l, o);
    at_f32x4 o = {0.f, 0.f, 0.f, 0.f};
    const float* p = a.part_o + atc * a.D + (d < a.D ? d : 0);
    for (int s0 = 0; s0 < a.splits; s0 += 4) { // four parts' loads under way at a time; a part past the last weighs 0
        at_f32x4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const at_f32x4*>(p + min(s0 + k, a.splits - 1) * rows * a.D);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float w = __shfl(s0 < 32 ? w0 : w1, (s0 + k) & 31, 32);
            if (s0 + k < a.splits && w != 0.f) o += w * x[k]; // (a part without keys has no sums)
        }
    }
    if (at >= rows) return;
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
// The mask as bits: by row, word (set, n, i) the keys 32 n + k of row i; by key, word (set, n, j) the rows 32 n + r that show key j.  A set
// is a sequence's or a head's mask, one for all of them where it is broadcast; a mask that is the same for every query has one row, and its
// words by key say so for 32.  The owners of rows and of keys then ask for one word each, side by side in memory, where the bytes of a
// tile of 32 rows lie in 32 cache lines: 517 x 1031 x 12/4 heads, D 80, 101 us with bytes, 73 with bits.
__host__ __device__ __forceinline__ int at_words(int n) { return (n + 31) / 32; }
__host__ __device__ __forceinline__ int64_t at_mask_set(const AttendArgs& a, int b, int head) {
    return (int64_t)(a.m_sb ? b : 0) * (a.m_sh ? a.H : 1) + (a.m_sh ? head : 0);
}
__host__ __device__ __forceinline__ int64_t at_mask_waves(const AttendArgs& a) { // one for 32 rows x 64 keys
    return (at_mask_set(a, a.B - 1, a.H - 1) + 1) * at_words(a.mask_rows) * ((a.Nk + 63) / 64);
}
static __device__ __forceinline__ void at_mask_bits(const AttendArgs& a, int64_t id) {
    if (id >= at_mask_waves(a)) return;
    const int lane = threadIdx.x & 63, rt = at_words(a.mask_rows), kt = at_words(a.Nk), pairs = (a.Nk + 63) / 64;
    const int pair = (int)(id % pairs), n = (int)(id / pairs % rt);
    const int64_t set = id / pairs / rt, b = a.m_sh ? set / a.H : set, head = a.m_sh ? set % a.H : 0;
    const int key = 64 * pair + lane;
    const uint8_t* p = a.mask + b * a.m_sb + head * a.m_sh + (int64_t)min(key, a.Nk - 1) * a.m_sk;
    uint32_t rows = 0, keys = 0; // of this lane's key; of row 32 n + lane % 32, keys 64 pair + 32 (lane / 32) ..
#pragma unroll
    for (int r = 0; r < 32; ++r) {
        const bool on = p[(int64_t)min(32 * n + r, a.mask_rows - 1) * a.m_sq] != 0 && key < a.Nk && 32 * n + r < a.mask_rows;
        const uint64_t all = __builtin_amdgcn_ballot_w64(on);
        rows |= (uint32_t)on << r;
        if ((lane & 31) == r) keys = lane < 32 ? (uint32_t)all : (uint32_t)(all >> 32);
    }
    if (a.mask_rows == 1) rows = rows ? 0xffffffffu : 0u;
    if (key < a.Nk) a.by_key[(set * rt + n) * a.Nk + key] = rows;
    const int row = 32 * n + (lane & 31), word = 2 * pair + (lane >> 5);
    if (row < a.mask_rows && word < kt) a.by_row[(set * kt + word) * a.mask_rows + row] = keys;
}

// delta_i = <dO_i, o_i>, 16 lanes a row.  Its last workgroups pack the mask.
//
// fp16 holds dS = P (dP - delta) in a power of two that the launch also prepares: |dP - delta| is at most 2 |dO_i| |v_j| (2-norms; o is a mean
// of the v), P at most 1, so the unit takes twice the largest |dO| times the largest |v| of a key head to 2^15 and nothing can leave fp16's
// range.  An even softmax over 8192 keys then has its dS around 2^15 / 8192 / sqrt(D), about 2^-2, twelve binary places above the end of
// fp16's normal range.  (For dQ the unit is the row's own, at_bwd_rows.)  Both norms are of the key head's own rows and keys, so what a sequence
// gets does not depend on its neighbours in the batch; rows that see no key, keys behind the length or hidden by a mask over keys, and
// what is not finite do not count.  (What a free mask hides from every query does: values there of more than some thousand times the
// others' size cost those bits.)  bf16 has fp32's range and needs none.  The pass over V: 8 x 768 x 16 heads, D 64, 9.7 -> 13.0 us, 38 MB
// where it had been 25; where V is most of what there is, one query for each of 64 x 8 heads of 512 keys, the whole backward pass 57 -> 63 us.
#define AT_DELTA_ROWS 16
#define AT_DELTA_KEYS 64
typedef unsigned short at_u16x2 __attribute__((ext_vector_type(2))); // exponents (biased) of the largest |dO|^2 and |v|^2
__device__ __forceinline__ at_u16x2 at_top_word(uint32_t w) { return __builtin_bit_cast(at_u16x2, w); }
__device__ __forceinline__ unsigned short at_exponent(float square) { return square < INFINITY ? (unsigned short)(__float_as_uint(square) >> 23) : (unsigned short)0; }
__device__ __forceinline__ at_u16x2 at_larger(at_u16x2 t, uint32_t w) { return __builtin_elementwise_max(t, at_top_word(w)); }
template <int FROM> __device__ __forceinline__ at_u16x2 at_lanes_top(at_u16x2 t) { // of lanes FROM apart and more
    for (int o = 32; o >= FROM; o >>= 1) t = at_larger(t, (uint32_t)__shfl_xor((int)__builtin_bit_cast(uint32_t, t), o));
    return t;
}
// 2^(15 - x) with 2 |dO| |v| < 2^x
__device__ __forceinline__ float at_unit(int grad, int value) {
    if (grad == 0 || value == 0) return 1.f; // dP - delta is 0
    return __uint_as_float((uint32_t)(127 + 14 - ((grad + value - 252 + 1) >> 1)) << 23);
}

template <typename T, bool WIDE> // WIDE: head sizes above 64, 16 lanes a key; else 8
__global__ __launch_bounds__(256) void at_delta_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x8 x8;
    constexpr bool UNIT = __is_same(T, _Float16);
    constexpr int LANES = WIDE ? 16 : 8, KEYS = UNIT ? AT_DELTA_KEYS * LANES / 256 : 0; // keys a thread has a chunk of
    if ((int)blockIdx.x >= a.delta_blocks) {
        at_mask_bits(a, 4 * (int64_t)(blockIdx.x - a.delta_blocks) + (threadIdx.x >> 6));
        return;
    }
    // fp16: a block's rows and keys are of one key head; otherwise rows of all of them.  (Rows are numbered in 30 bits.)
    const uint32_t R = UNIT ? a.G * a.Nq : a.B * a.H * a.Nq;
    const uint32_t part = UNIT ? blockIdx.x % a.unit_blocks : blockIdx.x, bkh = UNIT ? blockIdx.x / a.unit_blocks : 0, ub = bkh / a.Hk, ukh = bkh - ub * a.Hk;
    const uint32_t in = part * AT_DELTA_ROWS + (threadIdx.x >> 4), list = in / a.Nq, i = in - list * a.Nq;
    const uint32_t b = UNIT ? ub : list / a.H, head = UNIT ? ukh * a.G + list : list - b * a.H;
    const int d = (threadIdx.x & 15) * 8;
    x8 v[KEYS ? KEYS : 1] = {}; // asked for first: all loads are under way together
    if constexpr (UNIT) {
        const int len = a.key_lengths ? min(max(a.key_lengths[ub], 0), a.Nk) : a.Nk, dv = (threadIdx.x % LANES) * 8;
        const T* vb = static_cast<const T*>(a.v) + (int64_t)ub * a.v_sb + (int64_t)ukh * a.v_sh;
        const uint8_t* mkey = a.mask_by_key ? a.mask + (int64_t)ub * a.m_sb + (int64_t)ukh * a.G * a.m_sh : nullptr;
#pragma unroll
        for (int n = 0; n < KEYS; ++n) {
            const int key = (int)part * AT_DELTA_KEYS + n * (256 / LANES) + threadIdx.x / LANES;
            if (key < len && dv < a.D && !(mkey && !mkey[key * a.m_sk])) v[n] = *reinterpret_cast<const x8*>(vb + key * a.v_sn + dv);
        }
    }
    const uint32_t at = bkh * R + in;
    float sum = 0.f, size = 0.f;
    if (in < R && d < a.D) {
        const x8 o = *reinterpret_cast<const x8*>(static_cast<const T*>(a.out_in) + (((int64_t)b * a.Nq + i) * a.H + head) * a.D + d);
        const x8 g = *reinterpret_cast<const x8*>(static_cast<const T*>(a.dout) + b * a.g_sb + head * a.g_sh + i * a.g_sn + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) { sum += (float)o[e] * (float)g[e]; size += (float)g[e] * (float)g[e]; }
    }
    for (int o = 8; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (in < R && (threadIdx.x & 15) == 0) a.delta[at] = sum;
    if constexpr (UNIT) {
        for (int o = 8; o; o >>= 1) size += __shfl_xor(size, o);
        at_u16x2 top = {in < R && a.lse[at] != -INFINITY ? at_exponent(size) : (unsigned short)0, 0};
#pragma unroll
        for (int n = 0; n < KEYS; ++n) {
            float square = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) square += (float)v[n][e] * (float)v[n][e];
            for (int o = LANES / 2; o; o >>= 1) square += __shfl_xor(square, o);
            top.y = max(top.y, at_exponent(square));
        }
        __shared__ uint32_t tops[4];
        top = at_lanes_top<8>(top);
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = __builtin_bit_cast(uint32_t, top);
        __syncthreads();
        if (threadIdx.x == 0) a.tops[blockIdx.x] = __builtin_bit_cast(uint32_t, at_larger(at_larger(at_larger(top, tops[1]), tops[2]), tops[3]));
    }
}

// The exponents of this key head.
template <typename T> __device__ __forceinline__ at_u16x2 at_head_top(const AttendArgs& a, int b, int kh, uint32_t* shared4) {
    if (!__is_same(T, _Float16) || a.Nq == 0) return at_u16x2{0, 0};
    const uint32_t* words = a.tops + ((int64_t)b * a.Hk + kh) * a.unit_blocks;
    at_u16x2 top = {0, 0};
    for (int n = threadIdx.x; n < a.unit_blocks; n += 256) top = at_larger(top, words[n]);
    top = at_lanes_top<1>(top);
    if ((threadIdx.x & 63) == 0) shared4[threadIdx.x >> 6] = __builtin_bit_cast(uint32_t, top);
    __syncthreads();
    top = at_larger(at_larger(at_larger(at_top_word(shared4[0]), shared4[1]), shared4[2]), shared4[3]);
    return at_top_word((uint32_t)__builtin_amdgcn_readfirstlane((int)__builtin_bit_cast(uint32_t, top)));
}
// The exponent of |dO|^2 of the row whose fragments the two lanes c and c + 32 hold.
template <typename T, int DP> __device__ __forceinline__ int at_row_exponent(const typename AtEl<T>::x8* frag) {
    float square = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) square += (float)frag[ks][e] * (float)frag[ks][e];
    return at_exponent(square + at_other_half(square));
}

// dQ: a wave owns 32 rows and walks the keys that they see.
template <typename T, int DP, bool MASKED, int SHAPE, bool SPLIT> __device__ __forceinline__ void at_bwd_rows(const AttendArgs& a, AtShared<T, DP, SHAPE>& sh, int id)
{
    typedef typename AtEl<T>::x8 x8;
    typedef typename AtEl<T>::x4 x4;
    typedef AtTile<T, DP, SHAPE> Tile;
    constexpr int OWN = AtShape<SHAPE>::OWN, TILE = AtShape<SHAPE>::TILE, STREAMS = AtShape<SHAPE>::STREAMS, SUBS = TILE / 32;
    constexpr bool NARROW = SHAPE == AT_NARROW;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31, stream = wave / AtShape<SHAPE>::WAVES, sub = wave % AtShape<SHAPE>::WAVES;
    const int R = a.G * a.Nq, tiles = (R + OWN - 1) / OWN;
    const AtWhere where = at_where(a, id, tiles, SPLIT ? a.row_splits : 1);
    const int tile = a.causal ? tiles - 1 - where.tile : where.tile, kh = where.kh, b = where.b;
    const int value_top = at_head_top<T>(a, b, kh, sh.top4).y;

    const int len = a.key_lengths ? min(max(a.key_lengths[b], 0), a.Nk) : a.Nk;
    const int row = tile * OWN + sub * 32 + c, rowc = min(row, R - 1), g = rowc / a.Nq, i = rowc - g * a.Nq;
    const int head = kh * a.G + g;
    const int lim = row >= R ? 0 : a.causal ? min(len, max(0, i + a.Nk - a.Nq + 1)) : len;
    const int wave_top = at_wave_max(lim), wave_low = at_wave_min(row < R ? lim : 0x7fffffff);
    int top = wave_top;
    if (!NARROW) {
        if (lane == 0) sh.tops[wave] = wave_top;
        __syncthreads();
        top = __builtin_amdgcn_readfirstlane(max(max(sh.tops[0], sh.tops[1]), max(sh.tops[2], sh.tops[3])));
    }
    int t0 = 0, t1 = (top + TILE - 1) / TILE;
    if (SPLIT) {
        const int per = ((a.Nk + TILE - 1) / TILE + a.row_splits - 1) / a.row_splits;
        t0 = where.split * per;
        t1 = min(t1, t0 + per);
    }

    const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.k_sb + (int64_t)kh * a.k_sh;
    const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.v_sb + (int64_t)kh * a.v_sh;
    const uint32_t* words = MASKED ? a.by_row + at_mask_set(a, b, head) * at_words(a.Nk) * a.mask_rows + (a.mask_rows > 1 ? i : 0) : nullptr; // this row's
    const uint8_t* mkey = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)kh * a.G * a.m_sh : nullptr;
    auto load = [&](int t, int buf) {
        Tile::load(sh.tiles[stream][buf][0], kb + (int64_t)t * TILE * a.k_sn, (int)a.k_sn, len - t * TILE, a.D);
        Tile::load(sh.tiles[stream][buf][1], vb + (int64_t)t * TILE * a.v_sn, (int)a.v_sn, len - t * TILE, a.D);
    };
    uint32_t coming[MASKED ? SUBS : 1];
    auto ask = [&](int t) { // a tile ahead
        if (MASKED)
#pragma unroll
            for (int n = 0; n < SUBS; ++n) coming[n] = words[(int64_t)min(t * SUBS + n, at_words(a.Nk) - 1) * a.mask_rows];
    };
    Tile::pad(sh.tiles[0][0][0], 2, a.D);
    if (t0 + stream < t1) { load(t0 + stream, 0); ask(t0 + stream); }
    x8 qf[DP / 16], gf[DP / 16];
    {
        const T* qp = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh + (int64_t)i * a.q_sn;
        const T* gp = static_cast<const T*>(a.dout) + (int64_t)b * a.g_sb + (int64_t)head * a.g_sh + (int64_t)i * a.g_sn;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) { qf[ks] = at_global_frag<T>(qp, ks, lane, a.D); gf[ks] = at_global_frag<T>(gp, ks, lane, a.D); }
    }
    const int64_t at = ((int64_t)b * a.Hk + kh) * R + rowc;
    // a row's dQ depends on no other row: its unit is its own (one for the key head cost the rows beside one 3e5 times as large 3 % of their
    // dQ at 8192 keys)
    const float unit = __is_same(T, _Float16) ? at_unit(at_row_exponent<T, DP>(gf), value_top) : 1.f;
    const float lse = a.lse[at], neg_lse = lse == -INFINITY ? -INFINITY : -lse * 1.4426950408889634f, neg_delta = -a.delta[at] * unit;
    at_f32x16 acc[DP / 32] = {};

    int buf = 0;
    for (int t = t0 + stream; NARROW ? t < t1 : t - stream < t1; t += STREAMS, buf ^= 1) { // streams that share barriers take as many turns
        T *tk = sh.tiles[stream][buf][0], *tv = sh.tiles[stream][buf][1];
        at_landed();
        if (MASKED && a.mask_by_key && t < t1) {
            Tile::hide(tk, mkey + (int64_t)t * TILE * a.m_sk, a.m_sk, len - t * TILE);
            Tile::hide(tv, mkey + (int64_t)t * TILE * a.m_sk, a.m_sk, len - t * TILE);
        }
        if (!NARROW) __syncthreads();
        uint32_t seen[SUBS];
#pragma unroll
        for (int n = 0; n < SUBS; ++n) seen[n] = MASKED ? coming[n] : 0;
        if (t + STREAMS < t1) { load(t + STREAMS, buf ^ 1); ask(t + STREAMS); }
        if (t >= t1 || t * TILE >= wave_top) continue;
        at_f32x16 st[SUBS] = {}, dp[SUBS] = {};
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
            for (int n = 0; n < SUBS; ++n) {
                st[n] = AtEl<T>::mfma(at_rowfrag<T, DP>(tk, 32 * n, ks, lane), qf[ks], st[n]);
                dp[n] = AtEl<T>::mfma(at_rowfrag<T, DP>(tv, 32 * n, ks, lane), gf[ks], dp[n]);
            }
        if (MASKED || (t + 1) * TILE > wave_low) {
#pragma unroll
            for (int n = 0; n < SUBS; ++n) {
                uint32_t see = at_below_bits(t * TILE + 32 * n, lim);
                if (MASKED) see &= seen[n];
                see >>= 4 * h;
#pragma unroll
                for (int r = 0; r < 16; ++r) st[n][r] = at_hidden_unless(see, at_key(r), st[n][r]);
            }
        }
        x8 ds[SUBS][2];
#pragma unroll
        for (int n = 0; n < SUBS; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = __builtin_amdgcn_exp2f(fmaf(st[n][r], a.scale_log2e, neg_lse));
                ds[n][r >> 3][r & 7] = (T)(p * fmaf(dp[n][r], unit, neg_delta));
            }
#pragma unroll
        for (int n = 0; n < SUBS; ++n)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) acc[db] = AtEl<T>::mfma(at_colfrag<T, DP>(tk, 32 * n + 16 * s, db, lane), ds[n][s], acc[db]);
    }
    const float f = 1.f / unit; // the unit is taken off first: scale / unit could be infinite
    const bool blind = lse == -INFINITY; // sees nothing: a gradient of zero whatever the (unread) products gave
    auto store = [&](int n, const float* o) {
        const int d = at_channel(n, h);
        if (SPLIT && a.row_splits > 1) {
            if (d < a.D) *reinterpret_cast<at_f32x4*>(a.part_dq + (((int64_t)(where.split * a.B + b) * a.Hk + kh) * R + row) * a.D + d) = blind ? at_f32x4{0.f, 0.f, 0.f, 0.f} : at_f32x4{o[0] * f * a.scale, o[1] * f * a.scale, o[2] * f * a.scale, o[3] * f * a.scale};
            return;
        }
        x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = blind ? (T)0.f : (T)(o[e] * f * a.scale);
        if (d < a.D) *reinterpret_cast<x4*>(static_cast<T*>(a.dq) + (int64_t)b * a.dq_sb + (int64_t)head * a.dq_sh + (int64_t)i * a.dq_sn + d) = y;
    };
    float flat[DP / 2];
#pragma unroll
    for (int r = 0; r < DP / 2; ++r) flat[r] = acc[r >> 4][r & 15];
    if (STREAMS > 1) {
        float sum[DP / 2 / STREAMS];
        __syncthreads(); // every wave is done with its tiles
        at_sum_streams<DP / 2, SHAPE>(flat, reinterpret_cast<float*>(sh.tiles), sum);
        if (row >= R) return;
#pragma unroll
        for (int n = 0; n < DP / 8 / STREAMS; ++n) store(stream * (DP / 8 / STREAMS) + n, sum + 4 * n);
        return;
    }
    if (row >= R) return;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) store(n, flat + 4 * n);
}

// dK, dV: a wave owns 32 keys and walks the rows that may see them.
template <typename T, int DP, bool MASKED, int SHAPE, bool SPLIT> __device__ __forceinline__ void at_bwd_keys(const AttendArgs& a, AtSharedKeys<T, DP, SHAPE>& sh, int id)
{
    typedef typename AtEl<T>::x8 x8;
    typedef typename AtEl<T>::x4 x4;
    typedef AtTile<T, DP, SHAPE> Tile;
    constexpr int OWN = AtShape<SHAPE>::OWN, TILE = AtShape<SHAPE>::TILE, STREAMS = AtShape<SHAPE>::STREAMS, SUBS = TILE / 32;
    constexpr bool NARROW = SHAPE == AT_NARROW;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31, stream = wave / AtShape<SHAPE>::WAVES, sub = wave % AtShape<SHAPE>::WAVES;
    const int R = a.G * a.Nq, tiles = (a.Nk + OWN - 1) / OWN, off = a.Nk - a.Nq;
    const AtWhere where = at_where(a, id, tiles, SPLIT ? a.key_splits : 1);
    const int tile = where.tile, kh = where.kh, b = where.b; // causal: the first keys are seen by most rows, the long ones come first as they are
    const at_u16x2 top = at_head_top<T>(a, b, kh, sh.top4);
    // fp16 holds P for dV times 2^14: an even softmax over 16384 keys ends fp16's normal range, and P is at most 1
    constexpr float P_SHIFT = __is_same(T, _Float16) ? 14.f : 0.f, P_UNIT = __is_same(T, _Float16) ? 16384.f : 1.f;
    const float unit = at_unit(top.x, top.y), unit_p = unit / P_UNIT; // P carries its own unit into dS
    const int len = a.key_lengths ? min(max(a.key_lengths[b], 0), a.Nk) : a.Nk;
    const int k0 = tile * OWN, wave_k0 = k0 + sub * 32, key = wave_k0 + c;

    at_f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
    if (k0 < len) {
        const int keyc = min(key, len - 1);
        const T* qb = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)kh * a.G * a.q_sh;
        const T* gb = static_cast<const T*>(a.dout) + (int64_t)b * a.g_sb + (int64_t)kh * a.G * a.g_sh;
        const int64_t at0 = ((int64_t)b * a.Hk + kh) * R;
        const uint8_t* mkey = MASKED ? a.mask + (int64_t)b * a.m_sb + (int64_t)kh * a.G * a.m_sh + (int64_t)keyc * a.m_sk : nullptr;
        // the tiles: head by head, from the first query that sees a key of this workgroup (where there is a mask, of its word's rows)
        const int i_first = a.causal ? MASKED ? max(0, k0 - off) & ~31 : max(0, k0 - off) : 0, per_head = a.Nq > i_first ? (a.Nq - i_first + TILE - 1) / TILE : 0;
        int t0 = 0, t1 = a.G * per_head, g_next = 0, j_next = stream; // the next tile: head and number in it
        const int slot = threadIdx.x & (TILE - 1);                       // the row whose numbers this thread brings
        const bool brings = sub == 0 && lane < TILE;
        float n_lse = 0.f, n_delta = 0.f;
        uint32_t coming[MASKED ? SUBS : 1];
        if (SPLIT && t1) {
            const int per = (t1 + a.key_splits - 1) / a.key_splits;
            t0 = where.split * per;
            t1 = min(t1, t0 + per);
            g_next = t0 / per_head;
            j_next = t0 - g_next * per_head + stream;
        }
        while (j_next >= per_head && g_next < a.G) { j_next -= per_head; ++g_next; }
        auto load = [&](int buf) { // returns the first row of the tile
            const int g = g_next, i0 = i_first + j_next * TILE;
            j_next += STREAMS;
            while (j_next >= per_head) { j_next -= per_head; ++g_next; }
            Tile::load(sh.tiles[stream][buf][0], qb + (int64_t)g * a.q_sh + (int64_t)i0 * a.q_sn, (int)a.q_sn, a.Nq - i0, a.D);
            Tile::load(sh.tiles[stream][buf][1], gb + (int64_t)g * a.g_sh + (int64_t)i0 * a.g_sn, (int)a.g_sn, a.Nq - i0, a.D);
            if (brings) {
                const int64_t at = at0 + (int64_t)g * a.Nq + min(i0 + slot, a.Nq - 1);
                n_lse = a.lse[at]; // as they are: worked on in note(), when they have long arrived
                n_delta = a.delta[at];
            }
            if (MASKED)
#pragma unroll
                for (int n = 0; n < SUBS; ++n)
                    coming[n] = a.by_key[(at_mask_set(a, b, kh * a.G + g) * at_words(a.mask_rows) + min(i0 / 32 + n, at_words(a.mask_rows) - 1)) * a.Nk + keyc];
            return i0;
        };
        auto note = [&](int buf) {
            if (brings) {
                sh.lse[stream][buf][slot] = n_lse == -INFINITY ? -INFINITY : fmaf(-n_lse, 1.4426950408889634f, P_SHIFT);
                sh.delta[stream][buf][slot] = -n_delta * unit_p;
            }
        };
        Tile::pad(sh.tiles[0][0][0], 2, a.D);
        int i0 = 0, i0_next = 0;
        if (t0 + stream < t1) { i0_next = load(0); note(0); }
        x8 kf[DP / 16], vf[DP / 16];
        {
            const T* kp = static_cast<const T*>(a.k) + (int64_t)b * a.k_sb + (int64_t)kh * a.k_sh + (int64_t)keyc * a.k_sn;
            const T* vp = static_cast<const T*>(a.v) + (int64_t)b * a.v_sb + (int64_t)kh * a.v_sh + (int64_t)keyc * a.v_sn;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) { kf[ks] = at_global_frag<T>(kp, ks, lane, a.D); vf[ks] = at_global_frag<T>(vp, ks, lane, a.D); }
        }
        if (MASKED && a.mask_by_key && !mkey[0]) {
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) { kf[ks] = x8{}; vf[ks] = x8{}; }
        }
        int buf = 0;
        for (int t = t0 + stream; NARROW ? t < t1 : t - stream < t1; t += STREAMS, buf ^= 1) {
            const T *tq = sh.tiles[stream][buf][0], *tg = sh.tiles[stream][buf][1];
            at_landed();
            if (!NARROW) __syncthreads();
            i0 = i0_next;
            uint32_t seen[SUBS];
#pragma unroll
            for (int n = 0; n < SUBS; ++n) seen[n] = MASKED ? coming[n] : 0;
            if (t + STREAMS < t1) i0_next = load(buf ^ 1);
            if (STREAMS > 1 && t >= t1) continue;
            // unless every row of the tile sees every key of the wave
            const bool edge = MASKED || i0 + TILE > a.Nq || wave_k0 + 32 > len || (a.causal && i0 + off < wave_k0 + 31);
            at_f32x16 st[SUBS] = {}, dp[SUBS] = {};
            x8 pf[SUBS][2], df[SUBS][2], gt[2][DP / 32], qt[2][DP / 32];
            auto scores = [&](int n) {
                x8 qa[DP / 16], ga[DP / 16];
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) { qa[ks] = at_rowfrag<T, DP>(tq, 32 * n, ks, lane); ga[ks] = at_rowfrag<T, DP>(tg, 32 * n, ks, lane); }
                if (DP >= 96) __builtin_amdgcn_sched_barrier(0); // all reads under way before the first product
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) {
                    st[n] = AtEl<T>::mfma(qa[ks], kf[ks], st[n]);
                    dp[n] = AtEl<T>::mfma(ga[ks], vf[ks], dp[n]);
                }
            };
            auto hide = [&](int n) {
                uint32_t see = key < len ? at_below_bits(i0 + 32 * n, a.Nq) : 0; // which rows see this lane's key
                if (a.causal) see &= ~at_below_bits(i0 + 32 * n, key - off);
                if (MASKED) see &= seen[n];
                see >>= 4 * h;
#pragma unroll
                for (int r = 0; r < 16; ++r) st[n][r] = at_hidden_unless(see, at_key(r), st[n][r]);
            };
            auto probs = [&](int n) {
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int q0 = 32 * n + 8 * r4 + 4 * h;
                    const at_f32x4 nl = *reinterpret_cast<const at_f32x4*>(&sh.lse[stream][buf][q0]), nd = *reinterpret_cast<const at_f32x4*>(&sh.delta[stream][buf][q0]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * r4 + e;
                        const float p = __builtin_amdgcn_exp2f(fmaf(st[n][r], a.scale_log2e, nl[e]));
                        pf[n][r >> 3][r & 7] = (T)p;
                        df[n][r >> 3][r & 7] = (T)(p * fmaf(dp[n][r], unit_p, nd[e]));
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
            if constexpr (DP == 128 && SUBS == 2) {
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
                for (int n = 0; n < SUBS; ++n) {
                    scores(n);
                    if (edge) hide(n);
                    probs(n);
                    columns(n);
                    gradients(n);
                }
            }
            if (t + STREAMS < t1) note(buf ^ 1);
        }
    }
    const float f = 1.f / unit;
    auto store = [&](int n, const float* x, const float* y) {
        const int d = at_channel(n, h);
        if (SPLIT && a.key_splits > 1) {
            const int64_t to = (((int64_t)(where.split * a.B + b) * a.Hk + kh) * a.Nk + key) * a.D + d;
            if (d < a.D) {
                *reinterpret_cast<at_f32x4*>(a.part_dk + to) = at_f32x4{x[0] * f * a.scale, x[1] * f * a.scale, x[2] * f * a.scale, x[3] * f * a.scale};
                *reinterpret_cast<at_f32x4*>(a.part_dv + to) = at_f32x4{y[0] / P_UNIT, y[1] / P_UNIT, y[2] / P_UNIT, y[3] / P_UNIT};
            }
            return;
        }
        x4 k4, v4;
#pragma unroll
        for (int e = 0; e < 4; ++e) { k4[e] = (T)(x[e] * f * a.scale); v4[e] = (T)(y[e] / P_UNIT); }
        if (d < a.D) {
            *reinterpret_cast<x4*>(static_cast<T*>(a.dk) + (int64_t)b * a.dk_sb + (int64_t)kh * a.dk_sh + (int64_t)key * a.dk_sn + d) = k4;
            *reinterpret_cast<x4*>(static_cast<T*>(a.dv) + (int64_t)b * a.dv_sb + (int64_t)kh * a.dv_sh + (int64_t)key * a.dv_sn + d) = v4;
        }
    };
    float fk[DP / 2], fv[DP / 2];
#pragma unroll
    for (int r = 0; r < DP / 2; ++r) { fk[r] = dk[r >> 4][r & 15]; fv[r] = dv[r >> 4][r & 15]; }
    if (STREAMS > 1) {
        float sk[DP / 2 / STREAMS], sv[DP / 2 / STREAMS];
        __syncthreads(); // every wave is done with its tiles
        at_sum_streams<DP / 2, SHAPE>(fk, reinterpret_cast<float*>(sh.tiles), sk);
        __syncthreads();
        at_sum_streams<DP / 2, SHAPE>(fv, reinterpret_cast<float*>(sh.tiles), sv);
        if (key >= a.Nk) return;
#pragma unroll
        for (int n = 0; n < DP / 8 / STREAMS; ++n) store(stream * (DP / 8 / STREAMS) + n, sk + 4 * n, sv + 4 * n);
        return;
    }
    if (key >= a.Nk) return;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) store(n, fk + 4 * n, fv + 4 * n);
}

// PART 1: the rows' workgroups, 2: the keys', 3: both in one launch, the keys' first (they are the longer ones).
template <typename T, int DP, bool MASKED, int SHAPE, int PART, bool SPLIT>
__global__ __launch_bounds__(256, (DP == 128 && PART > 1) || (DP > 64 && SHAPE == AT_NARROW) ? 1 : 2) void at_bwd_kernel(AttendArgs a)
{
    union Shared {
        AtShared<T, DP, SHAPE> rows;
        AtSharedKeys<T, DP, SHAPE> keys;
    };
    if constexpr (PART == 1) {
        __shared__ __attribute__((aligned(16))) AtShared<T, DP, SHAPE> sh;
        at_bwd_rows<T, DP, MASKED, SHAPE, SPLIT>(a, sh, xcd_remap(blockIdx.x, gridDim.x));
    } else if constexpr (PART == 2) {
        __shared__ __attribute__((aligned(16))) AtSharedKeys<T, DP, SHAPE> sh;
        at_bwd_keys<T, DP, MASKED, SHAPE, SPLIT>(a, sh, xcd_remap(blockIdx.x, gridDim.x));
    } else {
        __shared__ __attribute__((aligned(16))) char raw[sizeof(Shared)];
        Shared& sh = *reinterpret_cast<Shared*>(raw);
        const int first = (a.Nk + AtShape<SHAPE>::OWN - 1) / AtShape<SHAPE>::OWN * a.B * a.Hk * (SPLIT ? a.key_splits : 1), id = blockIdx.x;
        if (id < first) at_bwd_keys<T, DP, MASKED, SHAPE, SPLIT>(a, sh.keys, xcd_remap(id, first));
        else at_bwd_rows<T, DP, MASKED, SHAPE, SPLIT>(a, sh.rows, xcd_remap(id - first, gridDim.x - first));
    }
}

// The parts of a gradient, added in their order: four channels a thread, the rows' before the keys'.
template <typename T> __global__ __launch_bounds__(256) void at_bwd_join_kernel(AttendArgs a)
{
    typedef typename AtEl<T>::x4 x4;
    const int q4 = a.D / 4;
    const int64_t rows = a.row_splits > 1 ? (int64_t)a.B * a.H * a.Nq * q4 : 0, keys = a.key_splits > 1 ? (int64_t)a.B * a.Hk * a.Nk * q4 : 0;
    int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= rows + 2 * keys) return;
    const bool is_q = at < rows, is_k = at - rows < keys;
    at -= is_q ? 0 : is_k ? rows : rows + keys;
    const float* p = (is_q ? a.part_dq : is_k ? a.part_dk : a.part_dv) + at * 4;
    const int64_t part = 4 * (is_q ? rows : keys);
    at_f32x4 sum = *reinterpret_cast<const at_f32x4*>(p);
    for (int n = 1; n < (is_q ? a.row_splits : a.key_splits); ++n) sum += *reinterpret_cast<const at_f32x4*>(p + n * part);
    const int d = (int)(at % q4) * 4, heads = is_q ? a.H : a.Hk, count = is_q ? a.Nq : a.Nk;
    const int64_t i = at / q4 % count, head = at / q4 / count % heads, b = at / q4 / count / heads;
    const int64_t to = is_q ? b * a.dq_sb + head * a.dq_sh + i * a.dq_sn : is_k ? b * a.dk_sb + head * a.dk_sh + i * a.dk_sn : b * a.dv_sb + head * a.dv_sh + i * a.dv_sn;
    x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)sum[e];
    *reinterpret_cast<x4*>(static_cast<T*>(is_q ? a.dq : is_k ? a.dk : a.dv) + to + d) = y;
}

// -------------------------------------------------------------------------------------------------------------------- launches
// Which shape, by the workgroups of 128 rows (or keys) that the wide one would have on the 256 CUs.
// Forward, us, narrow | wide, at D 64; 80; 128:  768 keys, 96 workgroups 11 | 18; 14 | 24; 16 | 23.  192: 15 | 19; 20 | 25; 25 | 24.  288: 20 | 25;
//   30 | 32; 39 | 34.  384: 25 | 26; 37 | 34; 45 | 37.  480: 33 | 28; 45 | 34; 57 | 38.  2048 keys, 384: 49 | 55; 73 | 71; 90 | 73.  8192 keys, 256: 109 |
//   146; 176 | 221; 199 | 210.  384: 163 | 198; 244 | 238; 299 | 256.  512: 210 | 195; 320 | 238; 391 | 284.  Causal (half the work, uneven), 2048 keys, 512: 40 |
//   55; 57 | 70; 72 | 71.  8192 keys, 768: 185 | 212; 289 | 280; 339 | 280.  1024: 212 | 232; 330 | 297; 410 | 297; but 512 keys, 512: 20 | 18; 31 | 24; 39 | 26.
//   Up to 32 rows (token by token in a large batch) three of the wide shape's four waves would have none: 4 rows, 2048 keys, 1024 key heads 116 | 116;
//   124 | 161; 197 | 201.  (A half shape, as the backward has, gained at most 5 % at any of these.)
// Backward, us, narrow | half | wide, at D 64; 80; 128, as many workgroups for rows as for keys:  768 x 768, 24: 13 | 19 | 26; 19 | 26 | 56; 19 |
//   28 | 64.  48: 16 | 19 | 26; 32 | 26 | 57; 34 | 29 | 65.  96: 24 | 22 | 27; 48 | 28 | 58; 50 | 47 | 66.  144: 34 | 35 | 30; 77 | 47 | 59; 83 | 67 | 69.
//   192: 39 | 38 | 31; 95 | 49 | 60; 101 | 75 | 71.  384: 75 | 60 | 54; 191 | 82 | 81; 198 | 139 | 122.  8192 x 8192, 128: 173 | 155 | 217; 513 | 210 |
//   454; 549 | 352 | 534.  256: 328 | 289 | 248; 1052 | 405 | 468; 1059 | 702 | 541.
static int64_t at_groups(int64_t bh, int64_t owned) { return bh * ceil_div(owned, 128); }
static bool at_narrow_fwd(int64_t bh, int64_t R, int Nk, int D, int causal) {
    const int64_t g = at_groups(bh, R) / (causal && Nk >= 1024 ? 2 : 1);
    if (R <= 32) return true;
    return D <= 64 ? g <= 448 : D <= 96 ? g <= 320 : g <= 128 || (g <= 256 && Nk >= 4096);
}
// A causal call has half the work, unevenly spread, so its workgroups count half (16 heads of 2048 x 2048, backward, us, narrow | half | wide at
// D 64; 80; 128: 60 | 60 | 63; 158 | 80 | 126; 175 | 123 | 149).
static int at_shape_bwd(int64_t bh, int64_t owned, int D, int causal) {
    const int64_t g = at_groups(bh, owned) / (causal ? 2 : 1);
    if (g < (D <= 64 ? 60 : 36)) return AT_NARROW;
    return g < (D <= 64 ? 140 : D <= 96 ? 384 : 200) ? AT_HALF : AT_WIDE;
}
// Parts that a row's keys are cut into where even the narrow shape's workgroups are few.  A single tile of rows (token by token) is bound
// by memory: four workgroups a CU, so that sequences of different lengths even out (16 caches of 0 to 8192: 75.3 us with two, 71.5, 72.7 with
// eight, 84.1 with sixteen); more rows: two, as the parts have to be joined.  At
// least 256 keys a part.
static int at_splits(int64_t bh, int64_t R, int Nk, int D) {
    if (!at_narrow_fwd(bh, R, Nk, D, 0)) return 1; // whatever the order, so that the workspace is the same
    int64_t s = R <= 32 ? 1024 / bh : 512 / (bh * ceil_div(R, 32));
    if (s > Nk / 256) s = Nk / 256;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

// The backward pass's launches: shapes of the keys' and the rows' owners, and the parts that their walks are cut into (by the sizes alone, so
// that the workspace is the same for a causal call).  Cut, whole, us, D 64: 8192 keys x 16 queries x 4 heads 24, 69; 33 keys x 4096 queries x 16/2
// heads 49, 330; 7 keys x 5000 x 8/1 41, 389.
struct AtBwdPlan { int keys, rows, key_splits, row_splits; };
static AtBwdPlan at_plan_bwd(int64_t bh, int64_t R, int64_t Nk, int D, int causal) {
    AtBwdPlan p = {at_shape_bwd(bh, Nk, D, 0), at_shape_bwd(bh, R, D, 0), 1, 1};
    const int64_t wr = bh * ceil_div(R, 32), wk = bh * ceil_div(Nk, 32);
    if (!wr || !wk) return p;
    auto parts = [](int64_t s, int64_t walked) { // of 512 at least: four waves' four tiles
        s = s < walked / 512 ? s : walked / 512;
        return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    };
    if (p.keys != p.rows && Nk > R) { // launches of their own, each to fill the chip four times
        p.key_splits = parts(1024 / wk, R); // 128 x 4096 x 4 x 16 heads, D 64; 128, us, rows whole: 107; 201.  In 2: 86; 171.  4: 77; 165
        p.row_splits = parts(1024 / wr, Nk);
    } else { // together: none is to walk much further than a 512th of the whole, where that is worth the join (1024 x 1024 x 4 heads, D 64; 128:
             // whole 16; 24 us, in 2 20; 38.  512 x 512 x 64/8 causal: 42; 64, in 2 36; 73.  6708 queries x 81 keys x 4 x 96/12, D 80; 128: 1910;
             // 2220, in 2 1598; 1860)
        const int64_t fair = ceil_div(wr * Nk + wk * R, 512), join = D <= 64 ? 1100 : 2100; // what the join costs, in rows (or keys) walked
        auto worth = [&](int64_t walked) { return walked > fair + join ? parts(walked >= 2 * fair ? walked / fair : 2, walked) : 1; };
        p.key_splits = worth(R);
        p.row_splits = worth(Nk);
    }
    p.keys = at_shape_bwd(bh, Nk, D, causal);
    p.rows = at_shape_bwd(bh, R, D, causal);
    // keys that are fewer than the rows walk far: their shape for both, in one launch; unless their walk is cut and the rows' is short (rows x
    // keys x heads / key heads, us together | apart, at D 64; 80; 128:  4096 x 33 x 16/2: 53 | 49; 101 | 56; 96 | 61.  8192 x 256 x 8: 56 | 62;
    // 123 | 69; 117 | 74.  1200 x 700 x 8/2: 29 | 34; 49 | 44; 55 | 49.  2048 x 2048 x 8/2, causal: 46 | 76; 89 | 97; 97 | 109)
    if (Nk <= R && p.row_splits == 1 && (p.key_splits == 1 || Nk > (D <= 64 ? 192 : 1024))) p.rows = p.keys;
    if (p.key_splits > 1 && p.keys == AT_WIDE) p.keys = AT_HALF;
    if (p.row_splits > 1 && p.rows == AT_WIDE) p.rows = AT_HALF;
    return p;
}

static int at_check(int dtype, int B, int H, int Hk, int Nq, int Nk, int D, float scale) {
    if (dtype != 0 && dtype != 2) return ADK_EUNSUPPORTED;
    if (B < 0 || H < 1 || Hk < 1 || H % Hk || Nq < 0 || Nk < 0) return ADK_EINVAL;
    if (D < 8 || D > 128 || (D & 7)) return ADK_EUNSUPPORTED;
    if (!(scale > 0.f) || !(scale < 1e37f)) return ADK_EINVAL; // and scale log2 e a number
    const int64_t R = (int64_t)(H / Hk) * Nq; // row and key numbers, and a grid, in 31 bits
    if (R > 0x7fffff00ll || Nk > 0x7fffff00 || (int64_t)B * Hk * ceil_div(R + Nk, 32) > 0xffffff) return ADK_EUNSUPPORTED;
    if ((int64_t)B * H * Nq > 0x7fffff00ll * 8) return ADK_EUNSUPPORTED;
    return 0;
}

// Blocks of at_delta_kernel that a key head has in fp16.
static int at_unit_blocks(int64_t R, int64_t Nk) {
    const int64_t rows = ceil_div(R, AT_DELTA_ROWS), keys = ceil_div(Nk, AT_DELTA_KEYS);
    return (int)(rows > keys ? rows : keys);
}

// s: strides (batch, head, token)
static int at_tensor(const void* p, const int64_t* s) {
    if (!p || ((uintptr_t)p & 15) || ((s[0] | s[1] | s[2]) & 7)) return ADK_EINVAL;
    return s[2] < 0 || s[2] >= (1 << 24) ? ADK_EUNSUPPORTED : 0; // 64 rows of a tile in 32-bit byte offsets
}

template <typename T, int DP, bool MASKED> static void at_launch_fwd(const AttendArgs& a, hipStream_t stream) {
    const int64_t R = (int64_t)a.G * a.Nq;
    if (at_narrow_fwd((int64_t)a.B * a.Hk, R, a.Nk, a.D, a.causal)) hipLaunchKernelGGL((at_fwd_kernel<T, DP, MASKED, AT_NARROW>), dim3((unsigned)(ceil_div(R, 32) * a.B * a.Hk * a.splits)), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((at_fwd_kernel<T, DP, MASKED, AT_WIDE>), dim3((unsigned)(ceil_div(R, 128) * a.B * a.Hk)), dim3(256), 0, stream, a);
}
template <typename T, int DP, bool MASKED> static void at_launch_bwd(const AttendArgs& a, hipStream_t stream) {
    const int64_t R = (int64_t)a.G * a.Nq, bh = (int64_t)a.B * a.Hk;
    const AtBwdPlan plan = at_plan_bwd(bh, R, a.Nk, a.D, a.causal);
    const int sk = plan.keys, sr = plan.rows, own[3] = {AtShape<AT_WIDE>::OWN, AtShape<AT_NARROW>::OWN, AtShape<AT_HALF>::OWN};
    const int64_t gk = ceil_div(a.Nk, own[sk]) * bh * a.key_splits, gr = ceil_div(R, own[sr]) * bh * a.row_splits;
#define AT_BWD(SHAPE, PART, SPLIT, GROUPS) hipLaunchKernelGGL((at_bwd_kernel<T, DP, MASKED, SHAPE, PART, SPLIT>), dim3((unsigned)(GROUPS)), dim3(256), 0, stream, a)
#define AT_BWD_CUT(SHAPE, PART, SPLITS, GROUPS) if ((SPLITS) > 1) AT_BWD(SHAPE, PART, true, GROUPS); else AT_BWD(SHAPE, PART, false, GROUPS)
    if (sk == sr && sk == AT_NARROW) { AT_BWD_CUT(AT_NARROW, 3, a.key_splits * a.row_splits, gk + gr); return; }
    if (sk == sr && sk == AT_HALF) { AT_BWD_CUT(AT_HALF, 3, a.key_splits * a.row_splits, gk + gr); return; }
    if constexpr (DP == 64) // 8 a CU: below, the tails of two launches cost more than the rows' third wave a SIMD brings
        if (sk == sr && gk + gr < 2048) { AT_BWD(AT_WIDE, 3, false, gk + gr); return; }
    if (gk) {
        if (sk == AT_NARROW) AT_BWD(AT_NARROW, 2, true, gk); // few keys in a launch of their own: their walk is cut
        else if (sk == AT_HALF) { AT_BWD_CUT(AT_HALF, 2, a.key_splits, gk); }
        else AT_BWD(AT_WIDE, 2, false, gk);
    }
    if (gr) {
        if (sr == AT_NARROW) { AT_BWD_CUT(AT_NARROW, 1, a.row_splits, gr); }
        else if (sr == AT_HALF) { AT_BWD_CUT(AT_HALF, 1, a.row_splits, gr); }
        else AT_BWD(AT_WIDE, 1, false, gr);
    }
#undef AT_BWD_CUT
#undef AT_BWD
}

template <typename T> static int at_fwd(const AttendArgs& a, hipStream_t stream) {
    if (a.D <= 64) { if (a.mask) at_launch_fwd<T, 64, true>(a, stream); else at_launch_fwd<T, 64, false>(a, stream); }
    else if (a.D <= 96) { if (a.mask) at_launch_fwd<T, 96, true>(a, stream); else at_launch_fwd<T, 96, false>(a, stream); }
    else { if (a.mask) at_launch_fwd<T, 128, true>(a, stream); else at_launch_fwd<T, 128, false>(a, stream); }
    if (a.splits > 1) hipLaunchKernelGGL((at_join_kernel<T>), dim3((unsigned)ceil_div((int64_t)a.B * a.H * a.Nq, 8)), dim3(256), 0, stream, a);
    ADK_RETURN_LAST_ERROR();
}

template <typename T> static int at_bwd(const AttendArgs& a, hipStream_t stream) {
    const int64_t blocks = a.delta_blocks + (a.mask ? ceil_div(at_mask_waves(a), 4) : 0);
    if (blocks && a.D > 64) hipLaunchKernelGGL((at_delta_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    else if (blocks) hipLaunchKernelGGL((at_delta_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    if (a.D <= 64) { if (a.mask) at_launch_bwd<T, 64, true>(a, stream); else at_launch_bwd<T, 64, false>(a, stream); }
    else if (a.D <= 96) { if (a.mask) at_launch_bwd<T, 96, true>(a, stream); else at_launch_bwd<T, 96, false>(a, stream); }
    else { if (a.mask) at_launch_bwd<T, 128, true>(a, stream); else at_launch_bwd<T, 128, false>(a, stream); }
    const int64_t parts = ((a.row_splits > 1 ? (int64_t)a.B * a.H * a.Nq : 0) + (a.key_splits > 1 ? 2 * (int64_t)a.B * a.Hk * a.Nk : 0)) * (a.D / 4);
    if (parts) hipLaunchKernelGGL((at_bwd_join_kernel<T>), dim3((unsigned)ceil_div(parts, 256)), dim3(256), 0, stream, a);
    ADK_RETURN_LAST_ERROR();
}

// s: strides of q, k, v (batch, head, token each), then of the mask (batch, head, query, key)
static void at_fill(AttendArgs& a, const void* q, const void* k, const void* v, const float* lse, const int* key_lengths, const uint8_t* mask, int B, int H, int Hk,
                    int Nq, int Nk, int D, const int64_t* s, float scale, int causal) {
    a.q = q; a.k = k; a.v = v; a.lse = const_cast<float*>(lse);
    a.key_lengths = key_lengths; a.mask = Nq && Nk ? mask : nullptr;
    a.B = B; a.H = H; a.Hk = Hk; a.G = H / Hk; a.Nq = Nq; a.Nk = Nk; a.D = D; a.splits = a.row_splits = a.key_splits = 1; a.causal = causal;
    a.q_sb = s[0]; a.q_sh = s[1]; a.q_sn = s[2];
    a.k_sb = s[3]; a.k_sh = s[4]; a.k_sn = s[5];
    a.v_sb = s[6]; a.v_sh = s[7]; a.v_sn = s[8];
    if (mask) { a.m_sb = s[9]; a.m_sh = s[10]; a.m_sq = s[11]; a.m_sk = s[12]; }
    a.mask_rows = a.m_sq ? Nq : 1;
    a.mask_by_key = a.mask && a.m_sq == 0 && (a.m_sh == 0 || a.G == 1);
    a.scale = scale; a.scale_log2e = scale * 1.4426950408889634f;
}

} // namespace adk

extern "C" int64_t adk_attend_fwd_workspace_bytes(int B, int H, int Hk, int Nq, int Nk, int D)
{
    const int e = adk::at_check(0, B, H, Hk, Nq, Nk, D, 1.f);
    if (e) return e;
    const int64_t rows = (int64_t)B * H * Nq;
    const int s = rows ? adk::at_splits((int64_t)B * Hk, (int64_t)(H / Hk) * Nq, Nk, D) : 1;
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
        a.splits = adk::at_splits((int64_t)B * Hk, (int64_t)a.G * Nq, Nk, D);
        a.part_o = static_cast<float*>(ws);
        a.part_ml = a.part_o + (int64_t)a.splits * B * H * Nq * D;
    }
    return dtype == 0 ? adk::at_fwd<_Float16>(a, stream) : adk::at_fwd<__bf16>(a, stream);
}

extern "C" int64_t adk_attend_bwd_workspace_bytes(int B, int H, int Hk, int Nq, int Nk, int D)
{
    const int e = adk::at_check(0, B, H, Hk, Nq, Nk, D, 1.f);
    if (e) return e;
    const int64_t rows = (int64_t)B * H * Nq, keys = (int64_t)B * Hk * Nk, R = (int64_t)(H / Hk) * Nq;
    const adk::AtBwdPlan p = adk::at_plan_bwd((int64_t)B * Hk, R, Nk, D, 0);
    const int rs = p.row_splits, ks = p.key_splits;
    const int64_t parts = (rs > 1 ? rs * rows * D : 0) + (ks > 1 ? 2 * ks * keys * D : 0);
    return 4 * (parts + rows + (rows ? (int64_t)B * Hk * adk::at_unit_blocks(R, Nk) : 0));
}

extern "C" int64_t adk_attend_mask_bytes(int B, int H, int Nq, int Nk, const int64_t* strides)
{
    if (B < 1 || H < 1 || Nq < 1 || Nk < 1) return 0;
    if (!strides) return ADK_EINVAL;
    const int64_t sets = (int64_t)(strides[0] ? B : 1) * (strides[1] ? H : 1), rows = strides[2] ? Nq : 1;
    return 4 * sets * (adk::at_words(Nk) * rows + adk::at_words((int)rows) * (int64_t)Nk);
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
        int64_t need = adk_attend_bwd_workspace_bytes(B, H, Hk, Nq, Nk, D);
        const adk::AtBwdPlan p = adk::at_plan_bwd((int64_t)B * Hk, (int64_t)a.G * Nq, Nk, D, causal);
        a.row_splits = p.row_splits;
        a.key_splits = p.key_splits;
        a.part_dq = static_cast<float*>(ws); // first: 16-byte aligned
        a.part_dk = a.part_dq + (a.row_splits > 1 ? a.row_splits * rows * D : 0);
        a.part_dv = a.part_dk + (a.key_splits > 1 ? a.key_splits * (int64_t)B * Hk * Nk * D : 0);
        a.delta = a.part_dv + (a.key_splits > 1 ? a.key_splits * (int64_t)B * Hk * Nk * D : 0);
        a.tops = reinterpret_cast<uint32_t*>(a.delta + rows);
        a.unit_blocks = adk::at_unit_blocks((int64_t)a.G * Nq, Nk);
        a.delta_blocks = dtype == 0 ? B * Hk * a.unit_blocks : (int)adk::ceil_div(rows, AT_DELTA_ROWS);
        if (a.delta_blocks + (a.mask ? adk::ceil_div(adk::at_mask_waves(a), 4) : 0) > 0xffffff) return ADK_EUNSUPPORTED; // a launch has fewer than 2^32 threads
        if (a.mask) {
            a.by_row = a.tops + (int64_t)B * Hk * a.unit_blocks;
            a.by_key = a.by_row + (adk::at_mask_set(a, B - 1, H - 1) + 1) * adk::at_words(Nk) * a.mask_rows;
            need += adk_attend_mask_bytes(B, H, Nq, Nk, strides + 9);
        }
        if (!ws || ws_bytes < need || ((uintptr_t)ws & 15)) return ADK_EWORKSPACE;
    }
    return dtype == 0 ? adk::at_bwd<_Float16>(a, stream) : adk::at_bwd<__bf16>(a, stream);
}
