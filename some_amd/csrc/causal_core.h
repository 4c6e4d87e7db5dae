// Shared pieces of the causal attention kernels over packed clips (causal_fwd.hip, causal_bwd.hip, attention_step.hip): element types, the
// LDS tile format with its two fragment reads, the global -> LDS copy and the block -> (clip, tile, head) map.
//
// All matrix products are 32 x 32 tiles with a contraction of 16 (v_mfma_f32_32x32x16 for f16 / bf16; for f32 eight v_mfma_f32_32x32x2_f32 on the
// same fragments).  Lane l = (l31 = l & 31, hi = l >> 5):
//     A / B fragment: 8 values, row (column) l31, contraction slots 8 hi + j          C / D register r: column l31, row crow(r, hi)
// A contraction may run in any order as long as both operands agree, so the C registers 8 s .. 8 s + 7 of one product ARE the B fragment of the
// next one when its A fragment takes the rows 16 s + (j & 3) + 8 (j >> 2) + 4 hi in slot j: probabilities never leave their registers.
#pragma once
#include "internal.h"

namespace causal {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct Frag { typedef s16x8 type; };
template <> struct Frag<float> { typedef f32x8 type; };

__device__ __forceinline__ int crow(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }

// (plain functions: hipcc drops the host stub of a kernel template that holds these builtins in a dependent context)
__device__ __forceinline__ f32x16 mma_bf16(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma_f16(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma_f32(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
template <typename T> __device__ __forceinline__ f32x16 mma(typename Frag<T>::type a, typename Frag<T>::type b, f32x16 c) {
    if constexpr (sizeof(T) == 4) return mma_f32(a, b, c);
    else if constexpr (__is_same(T, bf16_t)) return mma_bf16(a, b, c);
    else return mma_f16(a, b, c);
}
__device__ __forceinline__ s16x4 tr_read(const char* p) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)p);
}
__device__ __forceinline__ void dma16(const char* src, char* lds_dst) {
    typedef __attribute__((address_space(3))) void lds_void;
    __builtin_amdgcn_global_load_lds(src, (lds_void*)(uintptr_t)lds_dst, 16, 0, 0);
}
__device__ __forceinline__ void dma4(const char* src, char* lds_dst) {
    typedef __attribute__((address_space(3))) void lds_void;
    __builtin_amdgcn_global_load_lds(src, (lds_void*)(uintptr_t)lds_dst, 4, 0, 0);
}
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }
// a value and its counterpart in the other half of the wave (the same pair in both halves, so both compute the same bits)
__device__ __forceinline__ f32x2 both_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return (f32x2){__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
__device__ __forceinline__ float halves_max(float x) { const f32x2 b = both_halves(x); return fmaxf(b[0], b[1]); }
__device__ __forceinline__ float halves_sum(float x) { const f32x2 b = both_halves(x); return b[0] + b[1]; }
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

// Around a run of products: the wave goes before the others of its SIMD, whose exponentials then fill the gaps between the products instead of delaying them.
// us without and with: 8 x 2584 frames, 8/2 heads of 64: dK/dV bf16 146, 142, f16 189, 174, dQ 108.8, 108.3 and 119.9, 115.8; forward, 3 clips up to 8191, 16/4
// heads of 128, bf16: 305, 286; 4 x 4096 frames, 8/2 heads of 64, f32: forward 661, 597, dQ 903, 845.  Not so the 16-bit forward at heads of 64 (bf16 87.6, 88.5,
// f16 85.9, 87.6) and dK/dV in f32 (1212, 1270): those go without.
__device__ __forceinline__ void products_first() { __builtin_amdgcn_s_setprio(1); }
__device__ __forceinline__ void products_done() { __builtin_amdgcn_s_setprio(0); }

// Instruction order inside a basic block.  Left alone, hipcc places every LDS read directly before the matrix instruction that needs it and waits for it
// there, one read in flight at a time.  A sequence of these calls at the end of a block asks for `N` instructions of one kind after the other instead:
// reads some products ahead.
template <int N> __device__ __forceinline__ void order_mfma() { __builtin_amdgcn_sched_group_barrier(0x008, N, 0); }
template <int N> __device__ __forceinline__ void order_lds() { __builtin_amdgcn_sched_group_barrier(0x100, N, 0); }
// MFMAS products, each with READS LDS reads of its own, the reads AHEAD products early
template <int MFMAS, int READS, int AHEAD> __device__ __forceinline__ void order_products() {
    order_lds<READS * AHEAD>();
#pragma unroll
    for (int i = 0; i < MFMAS - AHEAD; ++i) {
        order_mfma<1>();
        order_lds<READS>();
    }
    order_mfma<AHEAD>();
}

// registers 8 s .. 8 s + 7 of a product as a fragment, rounded to the operand type (16-bit: half a step, 2^-8 or 2^-11 of the value)
template <typename T> __device__ __forceinline__ typename Frag<T>::type pack8(const f32x16& x, int s) {
    typename Frag<T>::type f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = x[8 * s + j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __builtin_bit_cast(short, (T)x[8 * s + j]);
    }
    return f;
}
template <typename T> __device__ __forceinline__ float to_f32(T x) { return (float)x; }

// 8 consecutive values of a row in global memory as a fragment
template <typename T> __device__ __forceinline__ typename Frag<T>::type load8(const T* p) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return *reinterpret_cast<const s16x8*>(p);
    }
}

// four neighbouring values of a row, rounded to the type once
template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(p) = (f32x4){a, b, c, d};
    } else {
        *reinterpret_cast<s16x4*>(p) = (s16x4){__builtin_bit_cast(short, (T)a), __builtin_bit_cast(short, (T)b), __builtin_bit_cast(short, (T)c), __builtin_bit_cast(short, (T)d)};
    }
}

// What a 16-bit type loses of x, to be kept in a second value of that type (f16: times 2^10, as it would be subnormal otherwise; never beyond x in size).
// D = rowsum(dO O) needs it: every key of a row gets D's error, and where a row sees few keys dP - D is far smaller than its terms - with D from the rounded
// O alone the gradients of clips of two frames are off by 5.6e-3 in bf16, with the rest by 2.4e-3, of which dS's own rounding is 2.3e-3.
template <typename T> constexpr float kRestScale = __is_same(T, f16_t) ? 1024.f : 1.f;
template <typename T> __device__ __forceinline__ float rest_of(float x) {
    const float r = x - (float)(T)x;
    return r - r == 0.f ? r * kRestScale<T> : 0.f;           // (x not finite: nothing)
}
template <typename T> __device__ __forceinline__ void store4_rest(T* p, float a, float b, float c, float d) {
    store4<T>(p, rest_of<T>(a), rest_of<T>(b), rest_of<T>(c), rest_of<T>(d));
}

// ---- LDS tiles: ROWS rows of D values, row pitch D sizeof(T) bytes, 16-byte chunk c of row r stored at chunk c ^ swz(r) --------------------
// The copy global -> LDS writes lane-linear chunks, so the permutation is applied to its per-lane source address.  swz is chosen so that both
// reads touch every LDS bank equally often: row fragments (32 rows, one chunk) and column fragments (ds_read_b64_tr_b16: 8 rows x 64 bytes; f32:
// rows r and r + 4 x 128 bytes).
template <typename T, int D> struct Tile {
    static constexpr int PITCH = D * (int)sizeof(T);
    static constexpr int CHUNKS = PITCH / 16;

    static __device__ __forceinline__ int swz(int r) {
        if constexpr (sizeof(T) == 4) return ((r & 4) << 1) | ((r & 3) << 1) | ((r >> 3) & 1);
        else if constexpr (CHUNKS == 8) return ((r & 2) << 1) | ((r >> 1) & 2) | ((r >> 3) & 1);
        else return ((r & 3) << 2) | ((r >> 2) & 3);
    }
    // fragment of row `row` (any row = 32 n + l31): values 16 ks + 8 hi .. + 7
    static __device__ __forceinline__ typename Frag<T>::type row_frag(const char* tile, int row, int ks, int hi) {
        const char* p = tile + row * PITCH;
        const int x = swz(row);
        if constexpr (sizeof(T) == 4) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p + (((4 * ks + 2 * hi) ^ x) << 4));
            const f32x4 b = *reinterpret_cast<const f32x4*>(p + (((4 * ks + 2 * hi + 1) ^ x) << 4));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<const s16x8*>(p + (((2 * ks + hi) ^ x) << 4));
        }
    }
    // fragment of column 32 db + l31: slot j holds row r0 + (j & 3) + 8 (j >> 2) + 4 hi (r0 a multiple of 16)
    static __device__ __forceinline__ typename Frag<T>::type col_frag(const char* tile, int r0, int db, int lane) {
        const int hi = lane >> 5;
        typename Frag<T>::type f;
        if constexpr (sizeof(T) == 4) {
            const int c = 8 * db + ((lane & 31) >> 2);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = r0 + (j & 3) + 8 * (j >> 2) + 4 * hi;
                f[j] = *reinterpret_cast<const float*>(tile + row * PITCH + ((c ^ swz(row)) << 4) + (lane & 3) * 4);
            }
        } else {
            // 16 lanes read a 4 x 16 block transposed: lane i supplies 4 values of row i >> 2, receives column i
            const int row = r0 + 4 * hi + ((lane & 15) >> 2), c = 4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            const s16x4 a = tr_read(tile + row * PITCH + ((c ^ swz(row)) << 4) + (lane & 1) * 8);
            const s16x4 b = tr_read(tile + (row + 8) * PITCH + ((c ^ swz(row + 8)) << 4) + (lane & 1) * 8);
            f = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return f;
    }
};

// Copy of ROWS consecutive rows (one tile) global -> LDS by NT threads.  The tile's first row is a wave-uniform pointer, a lane's place in the tile
// a 32-bit offset that never changes (the host refuses row strides whose tile would not fit 31 bits).  Rows at or past `rows` are copies of the
// last real one: finite or not, whoever reads them masks them, and no address leaves the matrix.
template <typename T, int D, int ROWS, int NT> struct Copier {
    typedef Tile<T, D> TL;
    static constexpr int PASSES = ROWS * TL::CHUNKS / NT;
    static_assert(PASSES * NT == ROWS * TL::CHUNKS, "whole passes");
    uint32_t off[PASSES];
    uint32_t row_bytes;

    __device__ __forceinline__ void init(int64_t stride_bytes, int tid) {
        row_bytes = (uint32_t)stride_bytes;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) off[p] = place(p * NT + tid, ROWS);
    }
    __device__ __forceinline__ uint32_t place(int L, int rows) const {
        const int row = L / TL::CHUNKS, slot = L % TL::CHUNKS;
        return (uint32_t)min(row, rows - 1) * row_bytes + (uint32_t)((slot ^ TL::swz(row)) << 4);
    }
    __device__ __forceinline__ void run(char* tile, const char* first, int rows, int tid) const {
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const uint32_t o = rows >= ROWS ? off[p] : place(p * NT + tid, rows);
            dma16(first + o, tile + (p * NT + wave * 64) * 16);
        }
    }
};

// ---- the softmax's running maximum -----------------------------------------------------------------------------------------------------------
// The running maximum only has to keep the exponentials in range, so it follows the true one lazily: it moves when a score passes it by 2^8.  P then
// reaches 256, far inside every operand type, and the accumulators are rescaled once or twice per row instead of at every new maximum.
constexpr float kSlack = 8.f;
constexpr float kDrop = 11.f;                    // (f16: row_base)

// What the exponentials of a row are taken relative to: P = exp2(s c2 - row_base(m)).  In f16 the base lies 2^7 below the maximum, so that P runs from 2^15 (the
// slack included) down to subnormals of 2^-24, and the running maximum follows the true one of a tile DOWN as well when that lies 2^11 below: with the row's
// maximum and a largest P of 1, the level tail of a peaked row - 16 384 keys 17.4 nats below one - was rounded away altogether.  A weight is off by at most 2^-21
// of its tile's largest that way (and by 2^-32 of it where that is the row's).  Scores of 2^20 and more, whose base has no digits behind the point left to spare,
// do without the 2^7: there P needs the room above.
template <typename T> __device__ __forceinline__ float row_base(float m, float c2) {
    const float x = m * c2;
    if constexpr (__is_same(T, f16_t)) return x - (__builtin_fabsf(x) < 0x1p20f ? 7.f : 0.f);
    else return x;
}
// a distance of exponents in units of the raw products; finite for scales next to nought too, or the first key would not pass it
__device__ __forceinline__ float score_units(float x, float c2) { return x / fmaxf(c2, 0x1p-120f); }
// whether a tile of maximum mx moves the running maximum m (the first visible key passes -inf; a sum m + slack would round up where scores are huge), and where to
template <typename T> __device__ __forceinline__ bool max_moves(float mx, float m, float slack, float drop) {
    if constexpr (__is_same(T, f16_t)) return __builtin_fabsf(mx - m + 0.5f * (drop - slack)) > 0.5f * (drop + slack);
    else return mx - m > slack;
}
template <typename T> __device__ __forceinline__ float max_moved(float mx, float m, float l, float c2, float slack, float drop) {
    float mn = mx - m > slack ? mx : m;
    if constexpr (__is_same(T, f16_t)) {                     // down: as far as the row's sum, and with it O, keeps inside f32's range
        const float room = fmaxf(100.f - log2_(halves_max(l)), 0.f) / c2;
        if (mx - m < -drop && mx > -INFINITY) mn = fmaxf(mx, m - room);
    }
    return mn;
}

// f32: acc[d] += the tile's 32 rows from r0 on, transposed, times x.  These products add one row after the other, so a block's are summed by themselves, one
// sum in registers at a time: added to a long sum one by one, equal terms all round the same way (65 536 of them: off by 7e-4).
template <typename T, int D> __device__ __forceinline__ void add_block(f32x16 (&acc)[D / 32], const char* tile, int r0, const f32x16& x, int lane) {
    typedef Tile<T, D> TL;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
        acc[d] += mma<T>(TL::col_frag(tile, r0 + 16, d, lane), pack8<T>(x, 1), mma<T>(TL::col_frag(tile, r0, d, lane), pack8<T>(x, 0), zero16()));
        __builtin_amdgcn_sched_barrier(0);
    }
}

// ---- not-a-number and infinities in masked places ----------------------------------------------------------------------------------------------
// A masked weight is 0, and 0 * inf would reach the sum.  Only a 32 x 32 block on the diagonal (or at a clip's end) mixes masked and visible places.
// If the 32 tile rows such a block contracts over hold a value that is not finite, the wave remembers it and, when its loop is done, computes its
// 32 columns anew one by one over the visible rows alone (solo_column).  The check is a few LDS reads per such block; the redo is slow and rare, and
// stands behind the loop where its registers cost nothing.
template <typename T, int D> __device__ __forceinline__ bool block_not_finite(const char* tile, int r0) {
    typedef Tile<T, D> TL;
    const int lane = threadIdx.x & 63;
    bool bad = false;
    for (int i = lane; i < 32 * TL::CHUNKS; i += 64) {
        const uint4 w = *reinterpret_cast<const uint4*>(tile + (r0 + i / TL::CHUNKS) * TL::PITCH + (i % TL::CHUNKS) * 16);
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(T) == 4) bad |= (x[k] & 0x7f800000u) == 0x7f800000u;
            else {
                constexpr uint32_t E = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
                bad |= (x[k] & E) == E || ((x[k] >> 16) & E) == E;
            }
        }
    }
    return __any(bad);
}
template <typename T, int D> __device__ __forceinline__ float dot_rows(const T* x, const T* y) {
    float s = 0.f;
    for (int d = 0; d < D; ++d) s = fmaf(to_f32(x[d]), to_f32(y[d]), s);
    return s;
}
// acc[e] (+)= sum over rows r in [r0, r1) of weight(r) * m[r][lane + 64 e]; the wave's lanes compute 64 weights side by side, then share them
template <typename T, int D, typename Weight>
__device__ __forceinline__ void solo_column(float (&acc)[(D + 63) / 64], int r0, int r1, const T* m, int64_t stride, Weight weight) {
    const int lane = threadIdx.x & 63;
    for (int base = r0; base < r1; base += 64) {
        const float w = base + lane < r1 ? weight(base + lane) : 0.f;
        float part[(D + 63) / 64] = {};                      // (64 rows by themselves: equal terms added one by one all round the same way)
        for (int j = 0; j < min(64, r1 - base); ++j) {
            const float wj = __shfl(w, j, 64);
#pragma unroll
            for (int e = 0; e < (D + 63) / 64; ++e) part[e] = fmaf(wj, to_f32(m[(int64_t)(base + j) * stride + lane + 64 * e]), part[e]);
        }
#pragma unroll
        for (int e = 0; e < (D + 63) / 64; ++e) acc[e] += part[e];
    }
}

template <typename T> __device__ __forceinline__ float dot8(typename Frag<T>::type x, typename Frag<T>::type y) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (sizeof(T) == 4) s = fmaf(x[j], y[j], s);
        else s = fmaf((float)__builtin_bit_cast(T, (short)x[j]), (float)__builtin_bit_cast(T, (short)y[j]), s);
    }
    return s;
}

// ---- block map ------------------------------------------------------------------------------------------------------------------------
// Rows are packed: clip b owns rows [off[b], off[b + 1]) of the queries and of the keys.  The heads of a group share keys, so a query tile holds TR / group
// frames with all their heads: query n of a clip is frame n / group, head n % group.  A launch has a position for every tile of TR queries (keys) the clips
// can have (`rows / TR + B` of them cover any lengths); a block finds its clip and tile from its position and the offsets alone, without a table.
struct Clip { int b, tile, qf, Tq, kf, Tk; };             // b < 0: no such tile

// sum over the wave of the lanes up to this one (lane 63: of all)
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);      // row_shr 1, 2, 4, 8: within 16 lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);      // row_bcast 15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);      // row_bcast 31 into rows 2 and 3
    return x;
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// Up to 64 clips: positions run through the tiles of all clips by falling work - the keys a query tile sees, or (KEYS) the queries that see a key tile -
// so the longest blocks start first whichever clip they belong to and the launch ends evenly.  A lane holds a clip; a clip's tiles in falling order of
// work are its last query tile first (its first key tile first), `at_least(x)` of them with a work of x units of TR or more; a bisection finds the
// level position p falls into.  More clips: clip after clip (each is then a small part of the launch), found by counting the clips that begin before.
// (Query tiles count in units of TR / group keys, so that a clip's next tile sees one unit more.)
template <bool KEYS, int TR>
__device__ __forceinline__ Clip find_clip(const int32_t* __restrict__ q_off, const int32_t* __restrict__ k_off, int B, bool causal, int group, int p) {
    const int lane = threadIdx.x & 63;
    Clip c;
    if (B <= 64) {
        const int b0 = min(lane, B - 1);
        const int qf = q_off[b0], Tq = q_off[b0 + 1] - qf, kf = k_off[b0], Tk = k_off[b0 + 1] - kf;
        const int mul = KEYS ? 1 : group;
        const int nq = (int)(((int64_t)Tq * mul + TR - 1) / TR), nk = (int)(((int64_t)Tk * mul + TR - 1) / TR);
        const int n = lane < B ? (KEYS ? nk : nq) : 0;
        const int past = max(0, nk - nq);                                // key tiles every query tile sees (and query levels below nought are all alike)
        const int top = KEYS ? nq : nk;
        const auto at_least = [&](int x) {
            if (!causal) return top >= x ? n : 0;
            return top >= x ? min(n, top - x + 1 + (KEYS ? past : 0)) : 0;
        };
        if (p >= wave_total(n)) return {-1, 0, 0, 0, 0, 0};
        int lo = -(1 << 22), hi = 1 << 22;                               // at_least(lo) counts everything, at_least(hi) nothing
        {
            int mx = lane < B ? top : 0;                                 // tighten: levels lie in (top - n, top]
            int mn = lane < B ? top - n - 1 : 0;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                mx = max(mx, __shfl_xor(mx, o, 64));
                mn = min(mn, __shfl_xor(mn, o, 64));
            }
            hi = __builtin_amdgcn_readfirstlane(mx) + 1;
            lo = __builtin_amdgcn_readfirstlane(mn);
        }
        while (hi - lo > 1) {                                            // the largest level with more than p tiles at or above it
            const int mid = (lo + hi) >> 1;
            if (wave_total(at_least(mid)) > p) lo = mid;
            else hi = mid;
        }
        const int above = at_least(lo + 1), here = at_least(lo) - above, upto = wave_scan(here);
        const int r = p - wave_total(above);                             // the r-th tile of this level
        const int b = __ffsll((unsigned long long)__ballot(upto > r)) - 1;
        const int k = __builtin_amdgcn_readlane(above, b) + r - (__builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(here, b));
        c.b = b;
        c.tile = KEYS ? k : __builtin_amdgcn_readlane(nq, b) - 1 - k;
        c.qf = __builtin_amdgcn_readlane(qf, b);
        c.Tq = __builtin_amdgcn_readlane(Tq, b);
        c.kf = __builtin_amdgcn_readlane(kf, b);
        c.Tk = __builtin_amdgcn_readlane(Tk, b);
        return c;
    }
    const int32_t* off = KEYS ? k_off : q_off;
    const int64_t mul = KEYS ? 1 : group;
    int n = 0;
    for (int base = 0; base < B; base += 64) {
        const int b = base + lane;
        const int m = __popcll(__ballot(b < B && off[b] * mul / TR + b <= p));
        n += m;
        if (m < 64) break;
    }
    c.b = __builtin_amdgcn_readfirstlane(n > 0 ? n - 1 : 0);
    c.qf = q_off[c.b]; c.Tq = q_off[c.b + 1] - c.qf;
    c.kf = k_off[c.b]; c.Tk = k_off[c.b + 1] - c.kf;
    c.tile = __builtin_amdgcn_readfirstlane(p - (int)(off[c.b] * mul / TR + c.b));
    if ((int64_t)c.tile * TR >= (KEYS ? c.Tk : c.Tq) * mul) c.b = -1;
    return c;
}
// blockIdx -> (kv head, position, head of the group and part): the blocks of one kv head run on as few of the 8 XCDs as balance allows (they read the same
// K and V through that XCD's L2), neighbouring positions at the same time.
struct Work { int kvh, pos, g; };
inline int work_subs(int kv_heads) { return (kv_heads & 1) ? 8 : (kv_heads & 2) ? 4 : (kv_heads & 4) ? 2 : 1; }
inline int64_t work_blocks(int kv_heads, int per_pos, int positions) {
    const int nsub = work_subs(kv_heads);
    return 8ll * (kv_heads * nsub / 8) * per_pos * ((positions + nsub - 1) / nsub);
}
__device__ __forceinline__ Work find_work(int kv_heads, int nsub, int per_pos) {
    const int xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
    const int upx = kv_heads * nsub / 8;
    const int g = j % per_pos, t = j / per_pos;
    const int u = (t % upx) * 8 + xcd;
    return {u / nsub, (t / upx) * nsub + u % nsub, g};
}

}  // namespace causal
