// Causal attention over packed clips, backward (causal_fwd.hip's mask, groups and layouts).  With s2 = scale log2(e) q.k, P = exp2(s2 - lse) is recomputed
// tile by tile:
//     D_i = sum_d dO O (kept negated),   dV = P^T dO,   dP = dO V^T,   dS = P (dP - D),   dQ = scale dS K,   dK = scale dS^T Q     (dK, dV summed over a group's heads)
// Two kernels, no atomics, so the gradients do not depend on the order blocks run in:
//   causal_dq_kernel   a wave owns 32 queries (a lane's column is a query), loops over the keys they see; writes D on the way in
//   causal_dkv_kernel  a wave owns 32 keys of one kv head (a lane's column is a key), loops over the group's heads and the queries that see them
// In both, the recomputed tile's registers are the B operand of the products that follow (causal_core.h).  Nine products of a pair instead of the formula's seven
// are the price of the order.  8 x 2584 frames, 8/2 heads of 64, bf16: 104 + 135 us, 800 TF/s of what they compute (VALU 51 and 42 % busy, products 36 %);
// 3 clips up to 8191, 16/4 heads of 128: 411 + 613 us, 950 TF/s, products 48 and 40 % busy at the clock the power limit leaves.
#include "causal_core.h"

namespace {
using namespace causal;

// f16 only: dS has the gradient's scale, which may lie far below (or above) f16's range.  A column's values (in units of `unit`) are multiplied by a power of two F of
// its own - constant over the contraction, so the accumulators simply carry it - that is lowered (accumulators rescaled) when a block would pass 2^14.
__device__ __forceinline__ float block_max(const f32x16& x) {
    float mx = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, __builtin_fabsf(x[r]));
    return halves_max(mx);
}
template <int DB> __device__ __forceinline__ void fit_column(const f32x16& ds, float unit, float& F, f32x16 (&acc)[DB]) {
    const float mx = block_max(ds) * unit;
    if (__any(mx * F > 16384.f)) {
        if (mx * F > 16384.f) {
            const float f = __builtin_ldexpf(1.f, min(100, max(-126, 5 - __builtin_amdgcn_frexp_expf(mx))));
            const float ratio = f / F;
            F = f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= ratio;
        }
    }
}
constexpr float kFitStart = 0x1p100f;
// f16 only: a key's weights may all lie far below f16's range as well, or those of the queries that count may (a key that one row alone looks at).  They too carry a
// power of two, which follows a block's largest weight down and up, at most 2^80: weights are 1 at most, so the accumulators stay inside f32's range.  It is set where
// that weight leaves [2^-4, 2^14], to 2^11 or more: a weight is off by at most 2^-21 of its block's largest, and by 2^-36 of the largest that set it.
constexpr float kProbStart = 80.f;
template <int DB> __device__ __forceinline__ void fit_probs(f32x16& p, f32x16& ds, float& log2f, f32x16 (&acc)[DB]) {
    const float mx = block_max(p);
    const bool off = mx > 16384.f || (mx < 0.0625f && mx > 0.f && log2f < kProbStart);
    if (__any(off)) {
        const float by = off ? fminf((float)(12 - __builtin_amdgcn_frexp_expf(mx)), kProbStart - log2f) : 0.f, ratio = exp2_(by);
        log2f += by;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            p[r] *= ratio;
            ds[r] *= ratio;
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= ratio;
    }
}

// ---- dQ (and D) ----------------------------------------------------------------------------------------------------------------------------
constexpr int QB = 128;                          // queries per workgroup
template <typename T, int D> struct DqShape {
    static constexpr int KT = (sizeof(T) == 4 && D == 128) ? 32 : 64;
    static constexpr int TILE_B = KT * D * (int)sizeof(T);
    static constexpr int LDS_B = 2 * 2 * TILE_B;
};

template <typename T, int D>
__global__ __launch_bounds__(256, (D == 64 ? (sizeof(T) == 2 ? 4 : 2) : sizeof(T) == 2 ? 2 : 1)) void causal_dq_kernel(CausalBwdArgs b, int nsub, int positions) {
    constexpr int KT = DqShape<T, D>::KT, NB = KT / 32, KS = D / 16, DB = D / 32, TILE_B = DqShape<T, D>::TILE_B;
    constexpr bool F16 = __is_same(T, f16_t);
    typedef Tile<T, D> TL;
    typedef typename Frag<T>::type frag;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const CausalArgs& a = b.f;

    const Work w = find_work(a.kv_heads, nsub, a.parts);
    if (w.pos >= positions) return;
    const Clip clip = find_clip<false, QB>(a.q_offsets, a.k_offsets, a.B, a.causal, a.group, w.pos);
    if (clip.b < 0) return;
    const int qf = clip.qf, Tq = clip.Tq, kf = clip.kf, Tk = clip.Tk, q0 = clip.tile * QB;
    const int shift = a.causal ? Tk - Tq : 0x3fffffff;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const int G = a.group, N = Tq * G, qw = q0 + wave * 32;  // queries: frame n / G, head n % G
    const unsigned n_lane = (unsigned)min(qw + l31, N - 1);
    const int q = (int)(n_lane / (unsigned)G), head = w.kvh * G + (int)(n_lane % (unsigned)G);
    const bool mine = qw + l31 < N;
    const int64_t qr = qf + q;
    const T* qrow = static_cast<const T*>(a.q.p) + qr * a.q.row + (int64_t)head * a.q.head + 8 * hi;
    const T* grow = static_cast<const T*>(b.dout.p) + qr * b.dout.row + (int64_t)head * b.dout.head + 8 * hi;
    const T* orow = static_cast<const T*>(a.out.p) + qr * a.out.row + (int64_t)head * a.out.head + 8 * hi;
    frag qfr[KS], gfr[KS];
    float dsum = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qfr[ks] = load8<T>(qrow + 16 * ks);
        gfr[ks] = load8<T>(grow + 16 * ks);
        dsum += dot8<T>(gfr[ks], load8<T>(orow + 16 * ks));
    }
    if constexpr (sizeof(T) == 2) {
        if (a.rest) {
            const T* rrow = static_cast<const T*>(a.rest) + (qr * a.kv_heads * G + head) * D + 8 * hi;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dsum = fmaf(dot8<T>(gfr[ks], load8<T>(rrow + 16 * ks)), 1.f / kRestScale<T>, dsum);
        }
    }
    dsum = halves_sum(dsum);
    const float lse = a.lse[(int64_t)head * a.q_rows + qr];
    if (w.g == 0 && mine && hi == 0) b.dsum[(int64_t)head * a.q_rows + qr] = -dsum;

    const int last_q = (int)((unsigned)(min(q0 + QB, N) - 1) / (unsigned)G);
    const int nkeys = min(Tk, max(0, last_q + shift + 1));
    const int ntiles = (nkeys + KT - 1) / KT;
    const int t_begin = (int)((int64_t)ntiles * w.g / a.parts), t_end = (int)((int64_t)ntiles * (w.g + 1) / a.parts);      // this part's tiles
    const int seen_w = qw < N ? min(Tk, max(0, (int)((unsigned)min(qw + 31, N - 1) / (unsigned)G) + shift + 1)) : 0;
    const int limit = min(q + shift, Tk - 1);
    const int full_w = min(Tk, max(0, (int)((unsigned)qw / (unsigned)G) + shift + 1));

    const char* kbase = reinterpret_cast<const char*>(static_cast<const T*>(a.k.p) + (int64_t)kf * a.k.row + (int64_t)w.kvh * a.k.head);
    const char* vbase = reinterpret_cast<const char*>(static_cast<const T*>(a.v.p) + (int64_t)kf * a.v.row + (int64_t)w.kvh * a.v.head);
    const int64_t kbytes = a.k.row * (int64_t)sizeof(T), vbytes = a.v.row * (int64_t)sizeof(T);
    Copier<T, D, KT, 256> ck, cv;
    ck.init(kbytes, tid);
    cv.init(vbytes, tid);
    auto fetch = [&](int t) {
        char* st = lds + (t & 1) * 2 * TILE_B;
        const int left = Tk - t * KT;
        ck.run(st, kbase + (int64_t)(t * KT) * kbytes, left, tid);
        cv.run(st + TILE_B, vbase + (int64_t)(t * KT) * vbytes, left, tid);
    };

    f32x16 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = zero16();
    float F = F16 ? kFitStart : 1.f;
    const float c2 = a.scale * 1.4426950408889634f;
    bool bad = false;

    if (t_begin < t_end) fetch(t_begin);
    for (int t = t_begin; t < t_end; ++t) {
        wait_vm<0>();
        __syncthreads();
        if (t + 1 < t_end) fetch(t + 1);
        const char* kt = lds + (t & 1) * 2 * TILE_B;
        const char* vt = kt + TILE_B;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int key0 = t * KT + nb * 32;
            if (key0 >= seen_w) break;
            f32x16 s = zero16(), dp = zero16();
            products_first();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = mma<T>(TL::row_frag(kt, nb * 32 + l31, ks, hi), qfr[ks], s);
                dp = mma<T>(TL::row_frag(vt, nb * 32 + l31, ks, hi), gfr[ks], dp);
            }
            products_done();
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = exp2_(fmaf(s[r], c2, -lse)) * (dp[r] - dsum);
            const bool edge = key0 + 32 > full_w;
            if (edge) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = key0 + crow(r, hi) <= limit ? s[r] : 0.f;
            }
            if constexpr (F16) {
                fit_column<DB>(s, 1.f, F, acc);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= F;
            }
            if (edge) bad |= block_not_finite<T, D>(kt, nb * 32);
            products_first();
            if constexpr (sizeof(T) == 4) {
                add_block<T, D>(acc, kt, nb * 32, s, lane);
            } else {
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const frag p = pack8<T>(s, s2);
#pragma unroll
                    for (int d = 0; d < DB; ++d) acc[d] = mma<T>(TL::col_frag(kt, nb * 32 + 16 * s2, d, lane), p, acc[d]);
                }
            }
            products_done();
        }
    }

    if (bad) {                                               // (wave-uniform; causal_core.h, "not-a-number and infinities")
        const T* kp = reinterpret_cast<const T*>(kbase);
        const T* vp = reinterpret_cast<const T*>(vbase);
        for (int n = 0; n < 32 && qw + n < N; ++n) {
            const int qn = (qw + n) / G, hd = w.kvh * G + (qw + n) % G;
            const int64_t row = qf + qn;
            const T* qp = static_cast<const T*>(a.q.p) + row * a.q.row + (int64_t)hd * a.q.head;
            const T* gp = static_cast<const T*>(b.dout.p) + row * b.dout.row + (int64_t)hd * b.dout.head;
            const float lse_n = __shfl(lse, n, 64), dsum_n = __shfl(dsum, n, 64);
            float x[(D + 63) / 64] = {};
            solo_column<T, D>(x, t_begin * KT, min(t_end * KT, min(qn + shift, Tk - 1) + 1), kp, a.k.row, [&](int j) {
                return exp2_(fmaf(dot_rows<T, D>(qp, kp + (int64_t)j * a.k.row), c2, -lse_n)) * (dot_rows<T, D>(gp, vp + (int64_t)j * a.v.row) - dsum_n);
            });
            T* dst = static_cast<T*>(b.dq.p) + row * b.dq.row + (int64_t)hd * b.dq.head;
            float* pdst = b.part_q + ((w.g * a.q_rows + row) * a.kv_heads * G + hd) * D;
#pragma unroll
            for (int e = 0; e < (D + 63) / 64; ++e) {
                if (a.parts > 1) pdst[lane + 64 * e] = x[e] * a.scale;
                else dst[lane + 64 * e] = (T)(x[e] * a.scale);
            }
        }
        return;
    }
    if (mine) {
        const float f = a.scale / F;
        T* dst = static_cast<T*>(b.dq.p) + qr * b.dq.row + (int64_t)head * b.dq.head + 4 * hi;
        float* pdst = b.part_q + ((w.g * a.q_rows + qr) * a.kv_heads * G + head) * D + 4 * hi;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const float x0 = acc[d][4 * r4] * f, x1 = acc[d][4 * r4 + 1] * f, x2 = acc[d][4 * r4 + 2] * f, x3 = acc[d][4 * r4 + 3] * f;
                if (a.parts > 1) store4<float>(pdst + 32 * d + 8 * r4, x0, x1, x2, x3);
                else store4<T>(dst + 32 * d + 8 * r4, x0, x1, x2, x3);
            }
    }
}

// ---- dK, dV --------------------------------------------------------------------------------------------------------------------------------
constexpr int KB = 128;                         // keys per workgroup
template <typename T, int D> struct DkvShape {
    // V fragments from LDS, not registers: at heads of 128 two waves share a SIMD, in f32 nothing spills (4 x 4096 frames, 8/2 heads of 64: 1270 us, with spills 1490)
    static constexpr bool V_LDS = D == 128 || sizeof(T) == 4;
    static constexpr int QT = V_LDS ? 32 : 64;                             // queries per tile
    static constexpr int TILE_B = QT * D * (int)sizeof(T);
    static constexpr int STAGE_B = 2 * TILE_B + 2 * 64 * 4;                // Q, dO, lse, D
    static constexpr int LDS_B = 2 * STAGE_B + (V_LDS ? KB * D * (int)sizeof(T) : 0);
};

template <typename T, int D>
__global__ __launch_bounds__(256, (D == 64 ? (sizeof(T) == 2 ? 3 : 2) : sizeof(T) == 2 ? 2 : 1)) void causal_dkv_kernel(CausalBwdArgs b, int nsub, int positions) {
    constexpr int QT = DkvShape<T, D>::QT, NB = QT / 32, KS = D / 16, DB = D / 32, TILE_B = DkvShape<T, D>::TILE_B, STAGE_B = DkvShape<T, D>::STAGE_B;
    constexpr bool F16 = __is_same(T, f16_t);
    typedef Tile<T, D> TL;
    typedef typename Frag<T>::type frag;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const CausalArgs& a = b.f;

    const Work w = find_work(a.kv_heads, nsub, b.parts);
    if (w.pos >= positions) return;
    const Clip clip = find_clip<true, KB>(a.q_offsets, a.k_offsets, a.B, a.causal, a.group, w.pos);
    if (clip.b < 0) return;
    const int qf = clip.qf, Tq = clip.Tq, kf = clip.kf, Tk = clip.Tk, k0 = clip.tile * KB;
    const int shift = a.causal ? Tk - Tq : 0x3fffffff;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const int kw = k0 + wave * 32, key = kw + l31;
    const int64_t kr = kf + min(key, Tk - 1);
    const T* krow = static_cast<const T*>(a.k.p) + kr * a.k.row + (int64_t)w.kvh * a.k.head + 8 * hi;
    const T* vrow = static_cast<const T*>(a.v.p) + kr * a.v.row + (int64_t)w.kvh * a.v.head + 8 * hi;
    // the first query that sees key k0 is k0 - shift
    const int t0 = max(0, k0 - shift) / QT, nt = max(0, (Tq + QT - 1) / QT - t0);
    const int total = nt * a.group;                          // (head, tile) pairs; this part's share of them:
    const int it0 = (int)((int64_t)total * w.g / b.parts), it1 = (int)((int64_t)total * (w.g + 1) / b.parts);
    constexpr bool V_LDS = DkvShape<T, D>::V_LDS;
    frag kfr[KS], vreg[V_LDS ? 1 : KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        kfr[ks] = load8<T>(krow + 16 * ks);
        if constexpr (!V_LDS) vreg[ks] = load8<T>(vrow + 16 * ks);
    }
    const char* vtile = lds + 2 * STAGE_B;
    if (V_LDS && it0 < it1) {                                // (its first iteration waits for the copy)
        Copier<T, D, KB, 256> cv;
        cv.init(a.v.row * (int64_t)sizeof(T), tid);
        cv.run(lds + 2 * STAGE_B, reinterpret_cast<const char*>(static_cast<const T*>(a.v.p) + (int64_t)(kf + k0) * a.v.row + (int64_t)w.kvh * a.v.head), Tk - k0, tid);
    }
    const auto vfr = [&](int ks) {
        if constexpr (V_LDS) return TL::row_frag(vtile, wave * 32 + l31, ks, hi);
        else return vreg[ks];
    };

    const int64_t qbytes = a.q.row * (int64_t)sizeof(T), gbytes = b.dout.row * (int64_t)sizeof(T);
    const char* qbase = reinterpret_cast<const char*>(static_cast<const T*>(a.q.p) + (int64_t)qf * a.q.row + (int64_t)w.kvh * a.group * a.q.head);
    const char* gbase = reinterpret_cast<const char*>(static_cast<const T*>(b.dout.p) + (int64_t)qf * b.dout.row + (int64_t)w.kvh * a.group * b.dout.head);
    const float* lbase = a.lse + (int64_t)w.kvh * a.group * a.q_rows + qf;
    const float* dbase = b.dsum + (int64_t)w.kvh * a.group * a.q_rows + qf;
    Copier<T, D, QT, 256> cq, cg;
    cq.init(qbytes, tid);
    cg.init(gbytes, tid);
    auto fetch = [&](int it, int g, int t) {
        char* st = lds + (it & 1) * STAGE_B;
        const int left = Tq - t * QT;
        cq.run(st, qbase + (int64_t)g * a.q.head * (int64_t)sizeof(T) + (int64_t)(t * QT) * qbytes, left, tid);
        cg.run(st + TILE_B, gbase + (int64_t)g * b.dout.head * (int64_t)sizeof(T) + (int64_t)(t * QT) * gbytes, left, tid);
        const int row = min(lane, left - 1);
        if (wave == 0) dma4(reinterpret_cast<const char*>(lbase + (int64_t)g * a.q_rows + t * QT + row), st + 2 * TILE_B);
        if (wave == 1) dma4(reinterpret_cast<const char*>(dbase + (int64_t)g * a.q_rows + t * QT + row), st + 2 * TILE_B + 64 * 4);
    };

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        dk[d] = zero16();
        dv[d] = zero16();
    }
    float F = F16 ? kFitStart : 1.f, log2p = F16 ? kProbStart : 0.f;       // dk's and dv's powers of two (f16)
    const float c2 = a.scale * 1.4426950408889634f;
    bool bad = false;

    int g = nt > 0 ? it0 / nt : 0, t = nt > 0 ? t0 + it0 % nt : 0;
    if (it0 < it1) fetch(it0, g, t);
    for (int it = it0; it < it1; ++it) {
        int gn = g, tn = t + 1;
        if (tn == t0 + nt) { tn = t0; ++gn; }
        wait_vm<0>();
        __syncthreads();
        if (it + 1 < it1) fetch(it + 1, gn, tn);
        const char* qt = lds + (it & 1) * STAGE_B;
        const char* gt = qt + TILE_B;
        const float* lt = reinterpret_cast<const float*>(qt + 2 * TILE_B);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int qb0 = t * QT + nb * 32;
            if (kw >= Tk || qb0 >= Tq || qb0 + 31 + shift < kw) continue;  // no key of the wave's, no query here, or none that sees its first key
            // 16-bit: the product dP starts from -D, which saves the subtraction (f32, bound by its matrix products: 80 -> 88 us at 8 x 520 frames)
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int r4 = 0; r4 < 4 && sizeof(T) == 2; ++r4) {
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(lt + 64 + nb * 32 + 8 * r4 + 4 * hi);
#pragma unroll
                for (int i = 0; i < 4; ++i) dp[4 * r4 + i] = d4[i];
            }
            if constexpr (sizeof(T) == 2) products_first();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = mma<T>(TL::row_frag(qt, nb * 32 + l31, ks, hi), kfr[ks], s);
                dp = mma<T>(TL::row_frag(gt, nb * 32 + l31, ks, hi), vfr(ks), dp);
            }
            if constexpr (sizeof(T) == 2) products_done();
            const bool edge = qb0 + shift < kw + 31 || qb0 + 32 > Tq || kw + 32 > Tk;
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const f32x4 lv = *reinterpret_cast<const f32x4*>(lt + nb * 32 + 8 * r4 + 4 * hi);
                f32x4 d4 = {0.f, 0.f, 0.f, 0.f};
                if constexpr (sizeof(T) == 4) d4 = *reinterpret_cast<const f32x4*>(lt + 64 + nb * 32 + 8 * r4 + 4 * hi);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 4 * r4 + i;
                    s[r] = exp2_(fmaf(s[r], c2, F16 ? log2p - lv[i] : -lv[i]));
                    dp[r] = s[r] * (sizeof(T) == 4 ? dp[r] + d4[i] : dp[r]);
                }
            }
            if (edge) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int qi = qb0 + crow(r, hi);
                    const bool see = qi < Tq && key < Tk && key <= qi + shift;
                    s[r] = see ? s[r] : 0.f;
                    dp[r] = see ? dp[r] : 0.f;
                }
                bad |= block_not_finite<T, D>(qt, nb * 32) || block_not_finite<T, D>(gt, nb * 32);
            }
            if constexpr (F16) {
                fit_probs<DB>(s, dp, log2p, dv);
                const float unit = exp2_(-log2p);
                fit_column<DB>(dp, unit, F, dk);
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= F * unit;
            }
            if constexpr (sizeof(T) == 2) products_first();
            if constexpr (sizeof(T) == 4) {
                add_block<T, D>(dv, gt, nb * 32, s, lane);
                add_block<T, D>(dk, qt, nb * 32, dp, lane);
            } else {
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const frag pf = pack8<T>(s, s2), df = pack8<T>(dp, s2);
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        dv[d] = mma<T>(TL::col_frag(gt, nb * 32 + 16 * s2, d, lane), pf, dv[d]);
                        dk[d] = mma<T>(TL::col_frag(qt, nb * 32 + 16 * s2, d, lane), df, dk[d]);
                    }
                }
            }
            if constexpr (sizeof(T) == 2) products_done();
        }
        g = gn;
        t = tn;
    }

    const int64_t prow = (int64_t)w.g * b.k_rows;
    if (bad) {                                               // (wave-uniform; causal_core.h, "not-a-number and infinities")
        for (int n = 0; n < 32 && kw + n < Tk; ++n) {
            const int kn = kw + n;
            const int64_t row = kf + kn;
            const T* kp = static_cast<const T*>(a.k.p) + row * a.k.row + (int64_t)w.kvh * a.k.head;
            const T* vp = static_cast<const T*>(a.v.p) + row * a.v.row + (int64_t)w.kvh * a.v.head;
            float xk[(D + 63) / 64] = {}, xv[(D + 63) / 64] = {};
            for (int gg = it0 / nt; gg <= (it1 - 1) / nt; ++gg) {
                const int r0 = max(max(max(it0, gg * nt) - gg * nt + t0, 0) * QT, kn - shift), r1 = min((min(it1, (gg + 1) * nt) - gg * nt + t0) * QT, Tq);
                const T* qp = reinterpret_cast<const T*>(qbase) + (int64_t)gg * a.q.head;
                const T* gp = reinterpret_cast<const T*>(gbase) + (int64_t)gg * b.dout.head;
                const float* lp = lbase + (int64_t)gg * a.q_rows;
                const float* dp = dbase + (int64_t)gg * a.q_rows;
                const auto prob = [&](int i) { return exp2_(fmaf(dot_rows<T, D>(qp + (int64_t)i * a.q.row, kp), c2, -lp[i])); };
                solo_column<T, D>(xv, r0, r1, gp, b.dout.row, prob);
                solo_column<T, D>(xk, r0, r1, qp, a.q.row, [&](int i) { return prob(i) * (dot_rows<T, D>(gp + (int64_t)i * b.dout.row, vp) + dp[i]); });
            }
#pragma unroll
            for (int e = 0; e < (D + 63) / 64; ++e) {
                const int d = lane + 64 * e;
                if (b.parts > 1) {
                    const int64_t i = ((prow + row) * a.kv_heads + w.kvh) * D + d;
                    b.part_k[i] = xk[e] * a.scale;
                    b.part_v[i] = xv[e];
                } else {
                    static_cast<T*>(b.dk.p)[row * b.dk.row + (int64_t)w.kvh * b.dk.head + d] = (T)(xk[e] * a.scale);
                    static_cast<T*>(b.dv.p)[row * b.dv.row + (int64_t)w.kvh * b.dv.head + d] = (T)xv[e];
                }
            }
        }
        return;
    }
    if (key < Tk) {
        const float pf = F16 ? exp2_(-log2p) : 1.f;
        const float fk = a.scale / F;
        const int64_t i = ((prow + kf + key) * a.kv_heads + w.kvh) * D + 4 * hi;
        T* dkd = static_cast<T*>(b.dk.p) + (int64_t)(kf + key) * b.dk.row + (int64_t)w.kvh * b.dk.head + 4 * hi;
        T* dvd = static_cast<T*>(b.dv.p) + (int64_t)(kf + key) * b.dv.row + (int64_t)w.kvh * b.dv.head + 4 * hi;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const f32x4 x = {dk[d][4 * r4] * fk, dk[d][4 * r4 + 1] * fk, dk[d][4 * r4 + 2] * fk, dk[d][4 * r4 + 3] * fk};
                const f32x4 y = {dv[d][4 * r4] * pf, dv[d][4 * r4 + 1] * pf, dv[d][4 * r4 + 2] * pf, dv[d][4 * r4 + 3] * pf};
                if (b.parts > 1) {
                    *reinterpret_cast<f32x4*>(b.part_k + i + 32 * d + 8 * r4) = x;
                    *reinterpret_cast<f32x4*>(b.part_v + i + 32 * d + 8 * r4) = y;
                } else {
                    store4<T>(dkd + 32 * d + 8 * r4, x[0], x[1], x[2], x[3]);
                    store4<T>(dvd + 32 * d + 8 * r4, y[0], y[1], y[2], y[3]);
                }
            }
    }
}

// dQ, or dK and dV (blockIdx.y): the parts summed in order, four channels a thread.
struct SumArgs { const float* src[2]; Rows3 out[2]; const int32_t* offsets; int64_t rows; int B, heads, parts; };
template <typename T, int D> __global__ __launch_bounds__(256) void causal_sum_kernel(SumArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, plane = a.rows * a.heads * D;
    const int64_t row = i / (a.heads * (D / 4));
    if (row < a.offsets[0] || row >= a.offsets[a.B]) return;
    const int h = (int)(i % (a.heads * (D / 4))) / (D / 4), d = (int)(i % (D / 4)) * 4;
    const float* src = a.src[blockIdx.y] + i * 4;
    f32x4 x = *reinterpret_cast<const f32x4*>(src);
    for (int p = 1; p < a.parts; ++p) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(src + p * plane);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] += y[k];
    }
    const Rows3& out = a.out[blockIdx.y];
    store4<T>(static_cast<T*>(out.p) + row * out.row + (int64_t)h * out.head + d, x[0], x[1], x[2], x[3]);
}
template <typename T, int D> void sum_parts(const SumArgs& a, unsigned planes, hipStream_t s) {
    hipLaunchKernelGGL((causal_sum_kernel<T, D>), dim3((unsigned)((a.rows * a.heads * (D / 4) + 255) / 256), planes), dim3(256), 0, s, a);
}

template <typename T, int D> hipError_t run(const CausalBwdArgs& b, hipStream_t s) {
    const CausalArgs& a = b.f;
    static DeviceOnce once;
    if (once.need()) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&causal_dq_kernel<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, DqShape<T, D>::LDS_B);
        if (e != hipSuccess) return e;
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(&causal_dkv_kernel<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, DkvShape<T, D>::LDS_B);
        if (e != hipSuccess) return e;
        once.mark();
    }
    const int nsub = work_subs(a.kv_heads);
    if (a.q_rows > 0) {
        const int positions = (int)(a.q_rows * a.group / QB) + a.B;
        hipLaunchKernelGGL((causal_dq_kernel<T, D>), dim3((unsigned)work_blocks(a.kv_heads, a.parts, positions)), dim3(256), (DqShape<T, D>::LDS_B), s, b, nsub, positions);
        if (a.parts > 1) sum_parts<T, D>({{b.part_q}, {b.dq}, a.q_offsets, a.q_rows, a.B, a.kv_heads * a.group, a.parts}, 1, s);
    }
    if (b.k_rows > 0) {
        const int positions = (int)(b.k_rows / KB) + a.B;
        hipLaunchKernelGGL((causal_dkv_kernel<T, D>), dim3((unsigned)work_blocks(a.kv_heads, b.parts, positions)), dim3(256), (DkvShape<T, D>::LDS_B), s, b, nsub,
                           positions);
        if (b.parts > 1) sum_parts<T, D>({{b.part_k, b.part_v}, {b.dk, b.dv}, a.k_offsets, b.k_rows, a.B, a.kv_heads, b.parts}, 2, s);
    }
    return hipGetLastError();
}

}  // namespace

// Parts the queries (and heads of a group) that a key tile meets are cut into: as many as bring the launch to 1200 workgroups - some rounds of the 512 to 768
// that run at once, so that causal tiles of unequal work end together; every part costs a plane of partial sums -, at least 4 tiles of 64 queries each.
// us of the kernel + the sum, bf16: 8 x 2584 frames, 8/2 heads of 64: 1 part 327, 2: 192 + 9, 3: 144 + 12, 4: 142 + 15, 5: 146 + 17; 3 clips up to 8191,
// 16/4 heads of 128: 1 part 1796, 2: 1016 + 16, 3: 772 + 22, 4: 726 + 27, 6: 732 + 38.  Lengths are on the device, so the averages over the batch decide.
int causal_bwd_parts(int64_t q_rows, int64_t k_rows, int B, int heads, int kv_heads) {
    if (B <= 0 || q_rows <= 0 || k_rows <= 0) return 1;
    const int64_t tiles = (k_rows + KB - 1) / KB > B ? (k_rows + KB - 1) / KB : B;
    const int64_t want = (1200 + tiles * kv_heads - 1) / (tiles * kv_heads), room = (q_rows / B + 63) / 64 * (heads / kv_heads) / 4;
    const int64_t p = want < room ? want : room;
    return p < 1 ? 1 : p > 16 ? 16 : (int)p;
}
int64_t causal_bwd_blocks(const CausalBwdArgs& b) { return causal::work_blocks(b.f.kv_heads, b.parts, (int)(b.k_rows / KB) + b.f.B); }

hipError_t launch_causal_bwd(int dtype, int head_dim, const CausalBwdArgs& b, hipStream_t s) {
    if (b.f.B <= 0) return hipSuccess;
    if (head_dim == 64) return dtype == 0 ? run<float, 64>(b, s) : dtype == 1 ? run<f16_t, 64>(b, s) : run<bf16_t, 64>(b, s);
    return dtype == 0 ? run<float, 128>(b, s) : dtype == 1 ? run<f16_t, 128>(b, s) : run<bf16_t, 128>(b, s);
}
