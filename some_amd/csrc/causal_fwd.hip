// Causal attention over packed clips, forward: out[i] = sum_j softmax_j(scale q_i . k_j) v_j over the keys j <= i + Tk - Tq of the clip (rows aligned at
// the end: the queries are the clip's last Tq frames), heads in groups that share keys and values.  A row that sees no key is 0 (log-sum -inf).
//
// One pass over the keys with a running maximum and sum (base 2, the scale folded into the exponent's multiplier).  A workgroup is 128 queries of one
// head, a wave 32 of them; S^T = K Q^T puts a query in every lane's column, so its maximum and sum are the lane's own registers plus one exchange
// with the other half, and P^T is already the B operand of O^T += V^T P^T (causal_core.h): no probability touches LDS.  K and V tiles go global ->
// LDS by DMA into a ring; V is read transposed by ds_read_b64_tr_b16.
#include "causal_core.h"

namespace {
using namespace causal;

constexpr int QB = 128;                          // queries per workgroup

template <typename T, int D> struct Shape {
    static constexpr int KT = (sizeof(T) == 4 && D == 128) ? 32 : 64;      // keys per tile
    static constexpr int TILE_B = KT * D * (int)sizeof(T);
    static constexpr int STAGES = 2;
    static constexpr int LDS_B = STAGES * 2 * TILE_B;
};

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void causal_fwd_kernel(CausalArgs a, int nsub, int slots) {
    constexpr int KT = Shape<T, D>::KT, NB = KT / 32, KS = D / 16, DB = D / 32;
    constexpr int TILE_B = Shape<T, D>::TILE_B, STAGES = Shape<T, D>::STAGES;
    typedef Tile<T, D> TL;
    typedef typename Frag<T>::type frag;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const Work w = find_work(a.kv_heads, nsub, a.group, slots);
    if (w.slot < 0) return;
    const Place pl = find_clip<QB>(a.q_offsets, a.B, w.slot);
    const int qf = a.q_offsets[pl.b], Tq = a.q_offsets[pl.b + 1] - qf;
    const int kf = a.k_offsets[pl.b], Tk = a.k_offsets[pl.b + 1] - kf;
    const int q0 = pl.tile * QB;
    if (q0 >= Tq) return;
    const int shift = a.causal ? Tk - Tq : 0x3fffffff;       // query i sees keys j <= i + shift

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const int head = w.kvh * a.group + w.g;
    const int qw = q0 + wave * 32, q = qw + l31;
    const T* qrow = static_cast<const T*>(a.q.p) + (int64_t)(qf + min(q, Tq - 1)) * a.q.row + (int64_t)head * a.q.head + 8 * hi;
    frag qfr[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qfr[ks] = load8<T>(qrow + 16 * ks);

    const int last_q = min(q0 + QB, Tq) - 1;
    const int nkeys = min(Tk, max(0, last_q + shift + 1));   // keys anybody here sees
    const int ntiles = (nkeys + KT - 1) / KT;
    const int seen_w = min(Tk, max(0, min(qw + 31, Tq - 1) + shift + 1));        // ... this wave sees (0 or less: none)
    const int limit = min(q + shift, Tk - 1);                // last key this lane's query sees
    const int full_w = min(Tk, max(0, qw + shift + 1));      // keys every query of the wave sees

    const char* kbase = reinterpret_cast<const char*>(static_cast<const T*>(a.k.p) + (int64_t)kf * a.k.row + (int64_t)w.kvh * a.k.head);
    const char* vbase = reinterpret_cast<const char*>(static_cast<const T*>(a.v.p) + (int64_t)kf * a.v.row + (int64_t)w.kvh * a.v.head);
    const int64_t kbytes = a.k.row * (int64_t)sizeof(T), vbytes = a.v.row * (int64_t)sizeof(T);
    Copier<T, D, KT, 256> ck, cv;
    ck.init(kbytes, tid);
    cv.init(vbytes, tid);
    auto fetch = [&](int t) {
        char* st = lds + (t % STAGES) * 2 * TILE_B;
        const int left = Tk - t * KT;
        ck.run(st, kbase + (int64_t)(t * KT) * kbytes, left, tid);
        cv.run(st + TILE_B, vbase + (int64_t)(t * KT) * vbytes, left, tid);
    };

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.f;                            // running maximum (of the raw products) and this half's share of the sum
    const float c2 = a.scale * 1.4426950408889634f;

    if (ntiles > 0) fetch(0);
    for (int t = 0; t < ntiles; ++t) {
        wait_vm<0>();
        __syncthreads();
        if (t + 1 < ntiles) fetch(t + 1);
        const char* kt = lds + (t % STAGES) * 2 * TILE_B;
        const char* vt = kt + TILE_B;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int key0 = t * KT + nb * 32;
            if (key0 >= seen_w) break;
            f32x16 s = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = mma<T>(TL::row_frag(kt, nb * 32 + l31, ks, hi), qfr[ks], s);
            const bool edge = key0 + 32 > full_w;
            if (edge) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = key0 + crow(r, hi) <= limit ? s[r] : -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
            mx = fmaxf(mx, other_half(mx));
            if (__any(mx > m)) {
                const float mn = fmaxf(m, mx);
                const float f = m == -INFINITY ? 0.f : exp2_((m - mn) * c2);
                m = mn;
                l *= f;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] *= f;
            }
            const float mc = m == -INFINITY ? 0.f : m * c2;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = exp2_(fmaf(s[r], c2, -mc));
#pragma unroll
            for (int r = 0; r < 16; ++r) l += s[r];
            if (edge && block_not_finite<T, D>(vt, nb * 32)) {
                add_by_hand<T, D>(o, s, vt, nb * 32, [&](int j) { return key0 + j <= limit; });
                continue;
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                const frag p = pack8<T>(s, s2);
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = mma<T>(TL::col_frag(vt, nb * 32 + 16 * s2, d, lane), p, o[d]);
            }
        }
    }

    if (q < Tq) {
        l += other_half(l);
        const float inv = limit >= 0 ? 1.f / l : 0.f;         // no visible key: zero
        T* orow = static_cast<T*>(a.out.p) + (int64_t)(qf + q) * a.out.row + (int64_t)head * a.out.head;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                T* p = orow + 32 * d + 8 * r4 + 4 * hi;
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<f32x4*>(p) = (f32x4){o[d][4 * r4] * inv, o[d][4 * r4 + 1] * inv, o[d][4 * r4 + 2] * inv, o[d][4 * r4 + 3] * inv};
                } else {
                    s16x4 x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = __builtin_bit_cast(short, (T)(o[d][4 * r4 + i] * inv));
                    *reinterpret_cast<s16x4*>(p) = x;
                }
            }
        if (a.lse && hi == 0) a.lse[(int64_t)head * a.q_rows + qf + q] = limit >= 0 ? m * c2 + log2_(l) : -INFINITY;
    }
}

template <typename T, int D> hipError_t run(const CausalArgs& a, hipStream_t s) {
    constexpr int lds = Shape<T, D>::LDS_B;
    static DeviceOnce once;
    if (once.need()) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&causal_fwd_kernel<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        once.mark();
    }
    const int slots = (int)(a.q_rows / QB) + a.B;
    hipLaunchKernelGGL((causal_fwd_kernel<T, D>), dim3((unsigned)work_blocks(a.kv_heads, a.group, slots)), dim3(256), lds, s, a, work_subs(a.kv_heads), slots);
    return hipGetLastError();
}

}  // namespace

int64_t causal_fwd_blocks(const CausalArgs& a) { return causal::work_blocks(a.kv_heads, a.group, (int)(a.q_rows / QB) + a.B); }

hipError_t launch_causal_fwd(int dtype, int head_dim, const CausalArgs& a, hipStream_t s) {
    if (a.B <= 0 || a.q_rows <= 0) return hipSuccess;
    if (head_dim == 64) return dtype == 0 ? run<float, 64>(a, s) : dtype == 1 ? run<f16_t, 64>(a, s) : run<bf16_t, 64>(a, s);
    return dtype == 0 ? run<float, 128>(a, s) : dtype == 1 ? run<f16_t, 128>(a, s) : run<bf16_t, 128>(a, s);
}
