// Attention of ONE new frame per stream over its cache: out[b, h] = sum_j softmax_j(scale q_bh . k_j) v_j over the first lengths[b] rows of the cache of kv
// head h / group.  Bound by reading the live rows of K and V once, so the keys are cut into chunks that fill the machine whatever the batch is:
//   step_kernel     block = (stream, kv head, chunk).  A wave takes every 4th 32 keys of the chunk, K straight into registers (a key is a row of the A
//                   operand), V through its own double-buffered LDS tile (DMA, no barrier in the loop), the next tile always in flight.  The heads of a
//                   group are the columns of its products, so a key is read once for all of them.  Running maximum and sum per wave, the waves of a
//                   block joined through LDS; one chunk in all: the output, otherwise a partial (O, m, l).
//   join_kernel     joins a stream's chunks in chunk order (the result does not depend on which block finished first).
// 32 streams of 8 x 128 (32 heads) in bf16, lengths up to 8192, take 69 + 5 us (4.6 TB/s); one of 517 frames, 8 x 64: 5.2 + 2.6 us, which is latency.  In f32 the
// products bound short caches: of their 32 columns a group of 4 heads fills 4.
#include "causal_core.h"

namespace {
using namespace causal;

constexpr int NW = 4;                            // waves of a block
template <typename T, int D> struct StepShape {
    static constexpr int TILE_B = 32 * D * (int)sizeof(T);
    static constexpr int WAVE_B = 2 * TILE_B;                              // two V tiles
    static constexpr int JOIN_B = NW * 32 * (D + 2) * 4;                   // what the join inside a block needs
    static constexpr int LDS_B = NW * WAVE_B > JOIN_B ? NW * WAVE_B : JOIN_B;
};

template <typename T, int D>
__global__ __launch_bounds__(NW * 64, (sizeof(T) == 4 && D == 128 ? 1 : 2)) void step_kernel(StepArgs a) {
    constexpr int TILE_B = StepShape<T, D>::TILE_B, KS = D / 16, DB = D / 32;
    typedef Tile<T, D> TL;
    typedef typename Frag<T>::type frag;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int hgs = (a.group + 31) / 32;                                   // blocks of 32 heads of a group
    // chunk outermost: workgroups go round the 8 XCDs in order, and whether a stream still has its n-th chunk depends on n
    const int per = a.kv_heads * hgs, unit = blockIdx.x % per, rest = blockIdx.x / per;
    const int kvh = unit / hgs, hg = unit % hgs, b = rest % a.B, chunk = rest / a.B;
    const int len = min(max(a.lengths[b], 0), a.capacity);
    const int lo = chunk * a.chunk, hi_key = min(len, lo + a.chunk);
    if (chunk > 0 && lo >= len) return;                                    // (chunk 0 of an empty stream writes its zeros)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const int heads = min(32, a.group - 32 * hg), head0 = kvh * a.group + 32 * hg;
    const T* qrow = static_cast<const T*>(a.q.p) + (int64_t)b * a.q.row + (int64_t)(head0 + min(l31, heads - 1)) * a.q.head + 8 * hi;
    frag qfr[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qfr[ks] = load8<T>(qrow + 16 * ks);

    const int64_t kbytes = a.k.row * (int64_t)sizeof(T), vbytes = a.v.row * (int64_t)sizeof(T);
    const char* kbase = reinterpret_cast<const char*>(static_cast<const T*>(a.k.p) + (int64_t)b * a.k_batch + (int64_t)kvh * a.k.head);
    const char* vbase = reinterpret_cast<const char*>(static_cast<const T*>(a.v.p) + (int64_t)b * a.v_batch + (int64_t)kvh * a.v.head);
    Copier<T, D, 32, 64> cv;
    cv.init(vbytes, lane);
    char* own = lds + wave * StepShape<T, D>::WAVE_B;
    const int ntiles = (max(0, hi_key - lo) + 31) / 32;
    frag kfr[KS], knext[KS];
    auto fetch = [&](int t, int stage) {                                   // (rows past the chunk: copies of its last one, V's to be zeroed)
        const int key0 = lo + t * 32;
        const T* krow = reinterpret_cast<const T*>(kbase + (int64_t)min(key0 + l31, hi_key - 1) * kbytes) + 8 * hi;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) knext[ks] = load8<T>(krow + 16 * ks);
        cv.run(own + stage * TILE_B, vbase + (int64_t)key0 * vbytes, hi_key - key0, lane);
    };

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.f;
    const float c2 = a.scale * 1.4426950408889634f, slack = score_units(kSlack, c2), drop = score_units(kDrop, c2);

    if (wave < ntiles) fetch(wave, 0);
    int stage = 0;
    for (int t = wave; t < ntiles; t += NW, stage ^= 1) {
        // tile t has landed; the other V tile was read an iteration ago, by this wave alone, and those reads have returned
        wait_vm<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kfr[ks] = knext[ks];
        if (t + NW < ntiles) fetch(t + NW, stage ^ 1);
        char* vt = own + stage * TILE_B;
        if (lo + t * 32 + 32 > hi_key) {                                   // values of places past the end: copies of the last one, which may be infinite
#pragma unroll 1
            for (int i = lane; i < 32 * TL::CHUNKS; i += 64)
                if (lo + t * 32 + i / TL::CHUNKS >= hi_key) *reinterpret_cast<uint4*>(vt + i * 16) = uint4{0, 0, 0, 0};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        f32x16 s = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = mma<T>(kfr[ks], qfr[ks], s);
        const int key0 = lo + t * 32;
        if (key0 + 32 > hi_key) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = key0 + crow(r, hi) < hi_key ? s[r] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = halves_max(mx);
        if (__any(max_moves<T>(mx, m, slack, drop))) {
            const float mn = max_moved<T>(mx, m, l, c2, slack, drop);
            const float f = m == -INFINITY ? 0.f : exp2_(row_base<T>(m, c2) - row_base<T>(mn, c2));
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= f;
        }
        const float mc = m == -INFINITY ? 0.f : row_base<T>(m, c2);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = exp2_(fmaf(s[r], c2, -mc));
#pragma unroll
        for (int r = 0; r < 16; ++r) l += s[r];
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            const frag p = pack8<T>(s, s2);
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = mma<T>(TL::col_frag(vt, 16 * s2, d, lane), p, o[d]);
        }
    }
    l = halves_sum(l);

    // join the waves: O [wave][head][D], then what it is relative to and l [wave][head]
    __syncthreads();
    float* ow = reinterpret_cast<float*>(lds);
    float* ml = ow + NW * 32 * D;
    if (l31 < heads) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                *reinterpret_cast<f32x4*>(ow + (wave * 32 + l31) * D + 32 * d + 8 * r4 + 4 * hi) = (f32x4){o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
        if (hi == 0) {
            ml[wave * 32 + l31] = row_base<T>(m, c2);
            ml[(NW + wave) * 32 + l31] = l;
        }
    }
    __syncthreads();
    for (int i = tid; i < heads * D; i += NW * 64) {
        const int h = i / D, d = i % D;
        float mm = -INFINITY;
#pragma unroll
        for (int x = 0; x < NW; ++x) mm = fmaxf(mm, ml[x * 32 + h]);
        float acc = 0.f, ll = 0.f;
#pragma unroll
        for (int x = 0; x < NW; ++x) {
            const float mx = ml[x * 32 + h];
            const float f = mx == -INFINITY ? (ml[(NW + x) * 32 + h] == 0.f ? 0.f : 1.f) : exp2_(mx - mm);
            acc = fmaf(ow[(x * 32 + h) * D + d], f, acc);
            ll = fmaf(ml[(NW + x) * 32 + h], f, ll);
        }
        if (a.chunks == 1) {
            const float v = len > 0 ? acc / ll : 0.f;
            static_cast<T*>(a.out.p)[(int64_t)b * a.out.row + (int64_t)(head0 + h) * a.out.head + d] = (T)v;
        } else {
            const int64_t slot = ((int64_t)b * a.kv_heads * a.group + head0 + h) * a.chunks + chunk;
            a.part_o[slot * D + d] = acc;
            if (d == 0) {
                a.part_ml[2 * slot] = mm;
                a.part_ml[2 * slot + 1] = ll;
            }
        }
    }
}

template <typename T, int D> __global__ __launch_bounds__(D) void join_kernel(StepArgs a) {
    const int heads = a.kv_heads * a.group, h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
    const int len = min(max(a.lengths[b], 0), a.capacity), n = (len + a.chunk - 1) / a.chunk;
    const int64_t slot = ((int64_t)b * heads + h) * a.chunks;
    float m = -INFINITY, acc = 0.f, ll = 0.f;
    for (int i0 = 0; i0 < n; i0 += 8) {                      // eight chunks in flight
        float mx[8], lx[8], x[8], mm = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t at = slot + min(i0 + i, n - 1);
            mx[i] = a.part_ml[2 * at];
            lx[i] = a.part_ml[2 * at + 1];
            x[i] = a.part_o[at * D + d];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i0 + i >= n) mx[i] = -INFINITY, lx[i] = 0.f;
            mm = fmaxf(mm, mx[i]);
        }
        const float f0 = m == -INFINITY ? 1.f : exp2_(m - mm);
        m = mm;
        acc *= f0;
        ll *= f0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = mx[i] == -INFINITY ? (lx[i] == 0.f ? 0.f : 1.f) : exp2_(mx[i] - mm);
            acc = i0 + i < n ? fmaf(x[i], f, acc) : acc;
            ll = fmaf(lx[i], f, ll);
        }
    }
    static_cast<T*>(a.out.p)[(int64_t)b * a.out.row + (int64_t)h * a.out.head + d] = (T)(len > 0 ? acc / ll : 0.f);
}

template <typename T, int D> hipError_t run(const StepArgs& a, hipStream_t s) {
    constexpr int lds = StepShape<T, D>::LDS_B;
    static DeviceOnce once;
    if (once.need()) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&step_kernel<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        once.mark();
    }
    const unsigned hgs = (unsigned)((a.group + 31) / 32);
    hipLaunchKernelGGL((step_kernel<T, D>), dim3((unsigned)a.chunks * (unsigned)a.kv_heads * hgs * (unsigned)a.B), dim3(NW * 64), lds, s, a);
    if (a.chunks > 1) hipLaunchKernelGGL((join_kernel<T, D>), dim3((unsigned)(a.kv_heads * a.group), (unsigned)a.B), dim3(D), 0, s, a);
    return hipGetLastError();
}

}  // namespace

// Keys of a chunk (us of the launches alone).  Up to 64 KiB of keys a stream and kv head there are no chunks and no join, for the second launch also costs the
// host 3.5 us: one stream of 8 x 64 in bf16, 512 frames whole 6.3, in chunks of 128 4.4 + 2.4; 1024 whole 8.5, in chunks of 256 5.2 + 2.4.  Beyond, a chunk has 128
// frames (256 where a row is 128 bytes: one stream of 8 x 64, 2584 frames 5.3 + 3.3, in chunks of 128 4.7 + 3.8; two of 5000, 8/2 heads, 5.6 + 4.1 and 4.9 + 5.5),
// and more as long as 256 blocks, one for each CU, remain (32 streams of 1024 frames, 32/8 heads of 128: 256 blocks 25, 512: 24 + 4), but not above 1024, for the
// sake of unequal streams (the 32 up to 8192 frames above: chunks of 512 72 + 4, of 1024 71 + 5, of 2048 73 + 5).
StepPlan step_plan(int dtype, int head_dim, int B, int kv_heads, int group, int max_len) {
    const int64_t units = (int64_t)B * kv_heads * ((group + 31) / 32);
    const int row = head_dim * (dtype == 0 ? 4 : 2);
    if (max_len <= 65536 / row) return {max_len > 0 ? max_len : 1, 1};
    int c = row == 128 ? 256 : 128;
    while (c < 1024 && units * ((max_len + 2 * c - 1) / (2 * c)) >= 256) c *= 2;
    return {c, (max_len + c - 1) / c};
}

hipError_t launch_attention_step(int dtype, int head_dim, const StepArgs& a, hipStream_t s) {
    if (a.B <= 0) return hipSuccess;
    if (head_dim == 64) return dtype == 0 ? run<float, 64>(a, s) : dtype == 1 ? run<f16_t, 64>(a, s) : run<bf16_t, 64>(a, s);
    return dtype == 0 ? run<float, 128>(a, s) : dtype == 1 ? run<f16_t, 128>(a, s) : run<bf16_t, 128>(a, s);
}
