// Causal attention over packed clips, forward: out[i] = sum_j softmax_j(scale q_i . k_j) v_j over the keys j <= i + Tk - Tq of the clip (rows aligned at
// the end: the queries are the clip's last Tq frames), heads in groups that share keys and values.  A row that sees no key is 0 (log-sum -inf).
//
// One pass over the keys with a running maximum and sum (base 2, the scale folded into the exponent's multiplier).  A workgroup is 128 queries - 128 /
// group frames with all heads of a group, which read every key tile together -, a wave 32 of them; S^T = K Q^T puts a query in every lane's column, so its
// maximum and sum are the lane's own registers plus one exchange with the other half, and P^T is already the B operand of O^T += V^T P^T (causal_core.h):
// no probability touches LDS.  K and V tiles go global -> LDS by DMA into a ring; V is read transposed by ds_read_b64_tr_b16.
// Bound by the products at heads of 128 - 2 clips up to 16384, 32/8 heads, bf16: 2.32 ms, 1090 TF/s, where a large matrix product reaches 1120 under the power
// limit - and at heads of 64 by the exponentials and what stands around them (8 x 2584, 8/2 heads, bf16: 83 us, 660 TF/s, VALU 60 % and products 29 % busy).
#include "causal_core.h"

namespace {
using namespace causal;

constexpr int QB = 128;                          // queries per workgroup

template <typename T, int D> struct Shape {
    static constexpr int KT = sizeof(T) == 4 ? 32 : 64;      // keys per tile (f32: one block, whose products are summed by themselves)
    static constexpr int TILE_B = KT * D * (int)sizeof(T);
    static constexpr int STAGES = 2;
    static constexpr int LDS_B = STAGES * 2 * TILE_B;
};

// one query, all its visible keys in [j0, j1) (causal_core.h, "not-a-number and infinities"): unnormalised sums, maximum and sum
template <typename T, int D>
__device__ __forceinline__ void solo_query(const CausalArgs& a, const T* q, const T* k, const T* v, int j0, int j1, float c2, float* m, float* l,
                                        float* o0, float* o1) {
    const int lane = threadIdx.x & 63;
    float mx = -INFINITY;
    for (int j = j0 + lane; j < j1; j += 64) mx = fmaxf(mx, dot_rows<T, D>(q, k + (int64_t)j * a.k.row));
#pragma unroll
    for (int x = 1; x < 64; x *= 2) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
    const float mc = mx == -INFINITY ? 0.f : mx * c2;
    float sum = 0.f, acc[(D + 63) / 64] = {};
    solo_column<T, D>(acc, j0, j1, v, a.v.row, [&](int j) {
        const float p = exp2_(fmaf(dot_rows<T, D>(q, k + (int64_t)j * a.k.row), c2, -mc));
        sum += p;
        return p;
    });
#pragma unroll
    for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x, 64);
    *m = mx;
    *l = sum;
    *o0 = acc[0];
    *o1 = D > 64 ? acc[(D + 63) / 64 - 1] : 0.f;
}

template <typename T, int D>
__global__ __launch_bounds__(256, (sizeof(T) == 2 ? (D == 64 ? 4 : 2) : (D == 64 ? 2 : 1))) void causal_fwd_kernel(CausalArgs a, int nsub, int positions) {
    typedef Shape<T, D> SH;
    constexpr int KT = SH::KT, NB = KT / 32, KS = D / 16, DB = D / 32, TILE_B = SH::TILE_B, STAGES = SH::STAGES;
    typedef Tile<T, D> TL;
    typedef typename Frag<T>::type frag;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const Work w = find_work(a.kv_heads, nsub, a.parts);
    if (w.pos >= positions) return;
    const Clip clip = find_clip<false, QB>(a.q_offsets, a.k_offsets, a.B, a.causal, a.group, w.pos);
    if (clip.b < 0) return;
    const int qf = clip.qf, Tq = clip.Tq, kf = clip.kf, Tk = clip.Tk, q0 = clip.tile * QB;
    const int shift = a.causal ? Tk - Tq : 0x3fffffff;       // query i sees keys j <= i + shift
    const int G = a.group, N = Tq * G, head0 = w.kvh * G, part = w.g;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const int qw = q0 + wave * 32;                           // the wave's first query
    const unsigned n_lane = (unsigned)min(qw + l31, N - 1);  // this lane's frame and head:
    const int q = (int)(n_lane / (unsigned)G), head = head0 + (int)(n_lane % (unsigned)G);
    const T* qrow = static_cast<const T*>(a.q.p) + (int64_t)(qf + q) * a.q.row + (int64_t)head * a.q.head + 8 * hi;
    frag qfr[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qfr[ks] = load8<T>(qrow + 16 * ks);

    const int last_q = (int)((unsigned)(min(q0 + QB, N) - 1) / (unsigned)G);
    const int nkeys = min(Tk, max(0, last_q + shift + 1));   // keys anybody here sees
    const int ntiles = (nkeys + KT - 1) / KT;
    // this part's tiles
    const int t_begin = (int)((int64_t)ntiles * part / a.parts), t_end = (int)((int64_t)ntiles * (part + 1) / a.parts);
    // keys this wave sees (a wave behind the clip's last query: none)
    const int seen_w = qw < N ? min(Tk, max(0, (int)((unsigned)min(qw + 31, N - 1) / (unsigned)G) + shift + 1)) : 0;
    const int full_w = min(Tk, max(0, (int)((unsigned)qw / (unsigned)G) + shift + 1));      // keys every query of the wave sees

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
    float m = -INFINITY, l = 0.f, lost = 0.f;                // running maximum (of the raw products), this half's share of the sum, what rounding added to it last (f32)
    const float c2 = a.scale * 1.4426950408889634f, slack = score_units(kSlack, c2), drop = score_units(kDrop, c2);
    bool bad = false;

    if (t_begin < t_end) fetch(t_begin);
    for (int t = t_begin; t < t_end; ++t) {
        wait_vm<0>();
        __syncthreads();
        if (t + 1 < t_end) fetch(t + 1);
        const char* kt = lds + (t % STAGES) * 2 * TILE_B;
        const char* vt = kt + TILE_B;
        const int key0 = t * KT;
        if (key0 >= seen_w) continue;
        f32x16 s[NB];
        if constexpr (sizeof(T) == 4 || D == 128) products_first();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            s[nb] = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[nb] = mma<T>(TL::row_frag(kt, nb * 32 + l31, ks, hi), qfr[ks], s[nb]);
        }
        if constexpr (sizeof(T) == 2) order_products<NB * KS, 1, 4>();
        if constexpr (sizeof(T) == 4 || D == 128) products_done();
        if (key0 + KT > full_w) {                            // some masked place in here
            const int limit = min(q + shift, Tk - 1);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                bad |= block_not_finite<T, D>(vt, nb * 32);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[nb][r] = key0 + nb * 32 + crow(r, hi) <= limit ? s[nb][r] : -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[nb][r]);
        mx = halves_max(mx);
        if (__any(max_moves<T>(mx, m, slack, drop))) {
            const float mn = max_moved<T>(mx, m, l, c2, slack, drop);
            const float f = m == -INFINITY ? 0.f : exp2_(row_base<T>(m, c2) - row_base<T>(mn, c2));
            m = mn;
            l *= f;
            lost *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= f;
        }
        const float mc = m == -INFINITY ? 0.f : row_base<T>(m, c2);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[nb][r] = exp2_(fmaf(s[nb][r], c2, -mc));
        // 32 keys' weights are summed by themselves: one by one, the equal weights of a long level row all round the same way (65 536 keys: off by 7e-4), and those of a
        // row with one dominating key are too small to move its sum at all.  f32 carries what the addition to the row's sum rounds as well (65 536 keys: 4e-5)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float w = s[nb][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) w += s[nb][r];
            if constexpr (sizeof(T) == 4) w -= lost;
            const float sum = l + w;
            if constexpr (sizeof(T) == 4) lost = (sum - l) - w;
            l = sum;
        }
        if constexpr (sizeof(T) == 4 || D == 128) products_first();
        if constexpr (sizeof(T) == 4) {
            // (16-bit products add eight keys at a time, and far below their own rounding).  The block's sum is too much for two waves a SIMD at heads of 128: 59
            // registers spilled, 4 x 4096 frames, 8/2 heads, 1810 us, one wave 1375
            static_assert(NB == 1, "a tile of 32 keys");
            add_block<T, D>(o, vt, 0, s[0], lane);
        } else {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const frag p = pack8<T>(s[nb], s2);
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[d] = mma<T>(TL::col_frag(vt, nb * 32 + 16 * s2, d, lane), p, o[d]);
                }
        }
        if constexpr (sizeof(T) == 2) order_products<NB * 2 * DB, 2, 3>();
        if constexpr (sizeof(T) == 4 || D == 128) products_done();
    }

    // A wave that sees one tile in all: where a row sees few keys, nothing averages the rounding of P out of O (nor of the gradients' D), so what it took goes
    // in too.  The tile still lies in the first stage, nobody writes there any more, and the maximum is the loop's.
    if constexpr (sizeof(T) == 2) {
        const bool few = t_begin == 0 && t_end > 0 && t_end <= STAGES && seen_w > 0 && seen_w <= KT && !bad;
        if (few) {                                           // (the rest of a weight may be nought or negative: an infinity of V that is seen must not meet it)
            bool inf = false;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) inf |= o[d][r] - o[d][r] != 0.f;
            bad = __any(inf);
        }
        if (few && !bad) {
            const float mc = m == -INFINITY ? 0.f : row_base<T>(m, c2);
            const int limit = min(q + shift, Tk - 1);
            for (int nb = 0; nb * 32 < seen_w; ++nb) {
                f32x16 s = zero16();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s = mma<T>(TL::row_frag(lds, nb * 32 + l31, ks, hi), qfr[ks], s);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = nb * 32 + crow(r, hi) <= limit ? exp2_(fmaf(s[r], c2, -mc)) : 0.f;
                    s[r] = p - (float)(T)p;
                }
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const frag p = pack8<T>(s, s2);
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[d] = mma<T>(TL::col_frag(lds + TILE_B, nb * 32 + 16 * s2, d, lane), p, o[d]);
                }
            }
        }
    }

    const int64_t prow = (int64_t)part * a.q_rows * a.kv_heads * a.group;
    if (bad) {                                               // (wave-uniform)
        for (int n = 0; n < 32 && qw + n < N; ++n) {
            const int qn = (qw + n) / G, hd = head0 + (qw + n) % G, limit = min(qn + shift, Tk - 1);
            float mm, ll, o0, o1;
            solo_query<T, D>(a, static_cast<const T*>(a.q.p) + (int64_t)(qf + qn) * a.q.row + (int64_t)hd * a.q.head, reinterpret_cast<const T*>(kbase),
                             reinterpret_cast<const T*>(vbase), t_begin * KT, min(t_end * KT, limit + 1), c2, &mm, &ll, &o0, &o1);
            if (a.parts > 1) {
                const int64_t i = prow + (int64_t)(qf + qn) * a.kv_heads * G + hd;
                a.part_o[i * D + lane] = o0;
                if (D > 64) a.part_o[i * D + 64 + lane] = o1;
                if (lane == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * i) = (f32x2){mm * c2, part == 0 && limit < 0 ? -1.f : ll};
            } else {
                const float inv = limit >= 0 ? 1.f / ll : 0.f;
                T* orow = static_cast<T*>(a.out.p) + (int64_t)(qf + qn) * a.out.row + (int64_t)hd * a.out.head;
                orow[lane] = (T)(o0 * inv);
                if (D > 64) orow[64 + lane] = (T)(o1 * inv);
                if constexpr (sizeof(T) == 2) {
                    if (a.rest) {
                        T* rrow = static_cast<T*>(a.rest) + ((int64_t)(qf + qn) * a.kv_heads * G + hd) * D;
                        rrow[lane] = (T)rest_of<T>(o0 * inv);
                        if (D > 64) rrow[64 + lane] = (T)rest_of<T>(o1 * inv);
                    }
                }
                if (a.lse && lane == 0) a.lse[(int64_t)hd * a.q_rows + qf + qn] = limit >= 0 ? mm * c2 + log2_(ll) : -INFINITY;
            }
        }
        return;
    }
    if (qw + l31 >= N) return;
    const float sum = halves_sum(l);
    const bool any = q + shift >= 0 && Tk > 0;
    if (a.parts > 1) {
        const int64_t i = prow + (int64_t)(qf + q) * a.kv_heads * G + head;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                store4<float>(a.part_o + i * D + 32 * d + 8 * r4 + 4 * hi, o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]);
        if (hi == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * i) = (f32x2){row_base<T>(m, c2), part == 0 && !any ? -1.f : sum};
    } else {
        const float inv = any ? 1.f / sum : 0.f;             // no visible key: zero
        T* orow = static_cast<T*>(a.out.p) + (int64_t)(qf + q) * a.out.row + (int64_t)head * a.out.head;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                store4<T>(orow + 32 * d + 8 * r4 + 4 * hi, o[d][4 * r4] * inv, o[d][4 * r4 + 1] * inv, o[d][4 * r4 + 2] * inv, o[d][4 * r4 + 3] * inv);
        if constexpr (sizeof(T) == 2) {
            if (a.rest) {
                T* rrow = static_cast<T*>(a.rest) + ((int64_t)(qf + q) * a.kv_heads * G + head) * D;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4)
                        store4_rest<T>(rrow + 32 * d + 8 * r4 + 4 * hi, o[d][4 * r4] * inv, o[d][4 * r4 + 1] * inv, o[d][4 * r4 + 2] * inv, o[d][4 * r4 + 3] * inv);
            }
        }
        if (a.lse && hi == 0) a.lse[(int64_t)head * a.q_rows + qf + q] = any ? row_base<T>(m, c2) + log2_(sum) : -INFINITY;
    }
}

// Joins the parts of the keys, in order, four channels a thread and four parts in flight (a clip's rows see keys in the first part or in none: it says so by
// a sum of -1).  Bound by latency where parts are few: 4160 rows of 8 heads of 64 in two parts take 6 us in f32.
template <typename T, int D> __global__ __launch_bounds__(256) void causal_join_kernel(CausalArgs a) {
    const int heads = a.kv_heads * a.group;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, i0 = id / (D / 4), row = i0 / heads;
    const int h = (int)(i0 - row * heads), d = (int)(id % (D / 4)) * 4;
    if (row < a.q_offsets[0] || row >= a.q_offsets[a.B]) return;
    const int64_t step = a.q_rows * heads;
    float m = -INFINITY, sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    bool any = true;
    for (int p0 = 0; p0 < a.parts; p0 += 4) {
        f32x2 ml[4];
        f32x4 x[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int64_t i = i0 + min(p0 + p, a.parts - 1) * step;
            ml[p] = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * i);
            x[p] = *reinterpret_cast<const f32x4*>(a.part_o + i * D + d);
        }
        if (p0 == 0) any = !(ml[0][1] < 0.f);
        float mm = m;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            if (p0 + p >= a.parts || ml[p][1] <= 0.f) ml[p][0] = -INFINITY, ml[p][1] = 0.f, x[p] = (f32x4){0.f, 0.f, 0.f, 0.f};      // adds nothing
            mm = fmaxf(mm, ml[p][0]);
        }
        const float f0 = m == -INFINITY ? 1.f : exp2_(m - mm);
        m = mm;
        sum *= f0;
        acc *= f0;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const float f = ml[p][0] == -INFINITY ? 1.f : exp2_(ml[p][0] - mm);
            sum = fmaf(ml[p][1], f, sum);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] = fmaf(x[p][k], f, acc[k]);
        }
    }
    const float inv = any ? 1.f / sum : 0.f;
    store4<T>(static_cast<T*>(a.out.p) + row * a.out.row + (int64_t)h * a.out.head + d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    if constexpr (sizeof(T) == 2) {
        if (a.rest) store4_rest<T>(static_cast<T*>(a.rest) + i0 * D + d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    }
    if (a.lse && d == 0) a.lse[(int64_t)h * a.q_rows + row] = any ? m + log2_(sum) : -INFINITY;
}

template <typename T, int D> hipError_t run(const CausalArgs& a, hipStream_t s) {
    constexpr int lds = Shape<T, D>::LDS_B;
    static DeviceOnce once;
    if (once.need()) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&causal_fwd_kernel<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        once.mark();
    }
    const int positions = (int)(a.q_rows * a.group / QB) + a.B;
    hipLaunchKernelGGL((causal_fwd_kernel<T, D>), dim3((unsigned)work_blocks(a.kv_heads, a.parts, positions)), dim3(256), lds, s, a, work_subs(a.kv_heads),
                       positions);
    if (a.parts > 1) hipLaunchKernelGGL((causal_join_kernel<T, D>), dim3((unsigned)((a.q_rows * a.kv_heads * a.group * (D / 4) + 255) / 256)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

int64_t causal_fwd_blocks(const CausalArgs& a) { return causal::work_blocks(a.kv_heads, a.parts, (int)(a.q_rows * a.group / 128) + a.B); }

// Parts the keys are cut into: 1 unless the queries alone give too few workgroups AND the keys are long (256 of them per part at least in f32, 512 in the
// 16-bit types).  Every part costs a plane of partial sums, so the launch is only brought to about 576 workgroups (2 per CU and a few more for balance): an f16
// chunk of 766 frames, 16/4 heads of 128, over 20 000 cached ones takes 4 parts 146 + 6 us, 5: 132 + 7, 6: 128 + 8, 8: 147 + 10, 12: 132 + 13.  8 x 520
// frames, 8 heads of 64, f32: 1 part 59 us, 2: 47 + 6.  2 x 1000, 8/1 heads of 128, f32: 1 part 167, 2: 92 + 6, 3: 69 + 7.  2 x 1500, 8/2 heads of 64, bf16:
// 1 part 32, 2: 22 + 5; 2 x 2000, 8/1 heads of 128: 1 part 53, 2: 38 + 9.  The gradient of the queries takes the same parts (and a sum): 2 x 1000, 8/1 heads of
// 128, f32: 1 part 229, 3: 95 + 6; 2 x 2000, bf16: 72, 2: 52 + 8.  Lengths are on the device, so the averages over the batch decide.
int causal_fwd_parts(int dtype, int64_t q_rows, int64_t k_rows, int B, int heads, int kv_heads) {
    if (B <= 0 || q_rows <= 0) return 1;
    const int64_t queries = q_rows * (heads / kv_heads), tiles = (queries + 127) / 128 > B ? (queries + 127) / 128 : B;
    const int64_t want = 576 / (tiles * kv_heads), room = k_rows / B / (dtype == 0 ? 256 : 512);
    const int64_t p = want < room ? want : room;
    return p < 1 ? 1 : p > 32 ? 32 : (int)p;
}

hipError_t launch_causal_fwd(int dtype, int head_dim, const CausalArgs& a, hipStream_t s) {
    if (a.B <= 0 || a.q_rows <= 0) return hipSuccess;
    if (head_dim == 64) return dtype == 0 ? run<float, 64>(a, s) : dtype == 1 ? run<f16_t, 64>(a, s) : run<bf16_t, 64>(a, s);
    return dtype == 0 ? run<float, 128>(a, s) : dtype == 1 ? run<f16_t, 128>(a, s) : run<bf16_t, 128>(a, s);
}
