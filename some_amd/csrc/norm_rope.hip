// Norm of queries and keys for each head with the position rotation in the same pass, and its gradients.  Per row and head, with n = x rsqrt(mean(x^2) + eps):
//     z = n gamma,   y_i = z_i cos a_i - z_{i + D/2} sin a_i,   y_{i + D/2} = z_{i + D/2} cos a_i + z_i sin a_i,   a_i = position theta^(-2 i / D)
//     dz = the rotation by -a of dy,   dgamma = sum dz n,   dx = rstd (dz gamma - n mean(dz gamma n))
// Bound by reading x (and dy) and writing y (dx) once: 25 300 rows of 32 + 8 heads of 128 in f16 take 97 us (5.3 TB/s), 82 688 rows of 16 + 4 heads of 64 in
// bf16 80 us forward (4.2 TB/s) and 128 + 4 us backward (4.0 TB/s; no less without sines and cosines); a large copy runs at 5.0 TB/s.
// A thread holds 8 channels of the lower half of a head and their partners in the upper half, so the rotation needs no exchange and D / 16 neighbouring lanes
// hold a head; it keeps its 8 sines and cosines for every head of its row that it works on.  The queries' heads and the keys' go to different blocks: in one,
// a thread would need both gains and two sets of gain gradients (backward, bf16: 152 us).
// The angle is reduced in 64 bits (position x turns-per-position, minus the whole turns): at position 10^6 a 32-bit product is off by 0.06 rad.
#include "causal_core.h"

namespace {
using namespace causal;

template <typename T> __device__ __forceinline__ void store8f(T* p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(p) = (f32x4){x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(p + 4) = (f32x4){x[4], x[5], x[6], x[7]};
    } else {
        s16x8 f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __builtin_bit_cast(short, (T)x[j]);
        *reinterpret_cast<s16x8*>(p) = f;
    }
}
template <int D> __device__ __forceinline__ float head_sum(float x) {
#pragma unroll
    for (int o = 1; o < D / 16; o *= 2) x += __shfl_xor(x, o, 64);
    return x;
}
__device__ __forceinline__ void angles(const NormRopeArgs& a, int64_t row, int i0, float (&c)[8], float (&s)[8]) {
    const double p = a.positions64 ? (double)static_cast<const int64_t*>(a.positions)[row] : (double)static_cast<const int32_t*>(a.positions)[row];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double t = p * a.turns[i0 + j];
        sincospif(2.f * (float)(t - __builtin_rint(t)), &s[j], &c[j]);
    }
}
template <typename T> struct Pair { typename Frag<T>::type lo, hi; };
template <typename T, int D> __device__ __forceinline__ Pair<T> load_pair(const T* p) { return {load8<T>(p), load8<T>(p + D / 2)}; }
template <typename T> __device__ __forceinline__ void widen(const Pair<T>& p, float (&u)[8], float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (sizeof(T) == 4) u[j] = p.lo[j], v[j] = p.hi[j];
        else u[j] = (float)__builtin_bit_cast(T, (short)p.lo[j]), v[j] = (float)__builtin_bit_cast(T, (short)p.hi[j]);
    }
}

// a row's heads h, h + step, ... < heads
template <typename T, int D>
__device__ __forceinline__ void rotate_heads(const Rows3& in, const Rows3& out, const float* gamma, float eps, int64_t row, int j, int h, int step, int heads,
                                             const float (&c)[8], const float (&s)[8]) {
    const T* x = static_cast<const T*>(in.p) + row * in.row + 8 * j;
    T* y = static_cast<T*>(out.p) + row * out.row + 8 * j;
    float gu[8], gv[8];
    widen<float>(load_pair<float, D>(gamma + 8 * j), gu, gv);
#pragma unroll 1
    for (; h < heads; h += step) {
        float u[8], v[8];
        widen<T>(load_pair<T, D>(x + (int64_t)h * in.head), u, v);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
        const float rstd = 1.f / sqrtf(head_sum<D>(ss) * (1.f / D) + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = u[i] * rstd * gu[i], q = v[i] * rstd * gv[i];
            u[i] = p * c[i] - q * s[i];
            v[i] = q * c[i] + p * s[i];
        }
        store8f<T>(y + (int64_t)h * out.head, u);
        store8f<T>(y + (int64_t)h * out.head + D / 2, v);
    }
}

// Blocks [0, q_blocks) work on the heads of q, the others on those of k: a thread has one gain and, backward, one set of its sums.
struct Side { const Rows3 &in, &grad, &out; const float* gamma; int heads, parts; int64_t block; };
__device__ __forceinline__ Side side_of(const NormRopeArgs& a) {
    if ((int)blockIdx.x < a.q_blocks) return {a.q, a.dq_in, a.q_out, a.gamma_q, a.heads, a.parts, (int64_t)blockIdx.x};
    return {a.k, a.dk_in, a.k_out, a.gamma_k, a.kv_heads, a.kv_parts, (int64_t)blockIdx.x - a.q_blocks};
}

template <typename T, int D> __global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a) {
    constexpr int L = D / 16;
    const Side side = side_of(a);
    const int j = threadIdx.x % L;
    const int64_t rest = side.block * (256 / L) + threadIdx.x / L, row = rest / side.parts;
    if (row >= a.rows) return;                               // (whole heads: the lanes of a head leave together)
    float c[8], s[8];
    angles(a, row, 8 * j, c, s);
    rotate_heads<T, D>(side.in, side.out, side.gamma, a.eps, row, j, (int)(rest - row * side.parts), side.parts, side.heads, c, s);
}

// Gradients: dx per row; dgamma of q and k summed over a thread's rows, then over the block's threads in a fixed order, then (gamma_grad_kernel) over the blocks.
template <typename T, int D>
__device__ __forceinline__ void rotate_heads_bwd(const Rows3& in, const Rows3& grad, const Rows3& out, const float* gamma, float eps, int64_t row, int j, int h, int step,
                                                 int heads, const float (&c)[8], const float (&s)[8], float (&acc)[16]) {
    const T* x = static_cast<const T*>(in.p) + row * in.row + 8 * j;
    const T* dy = static_cast<const T*>(grad.p) + row * grad.row + 8 * j;
    T* dx = static_cast<T*>(out.p) + row * out.row + 8 * j;
    float gu[8], gv[8];
    widen<float>(load_pair<float, D>(gamma + 8 * j), gu, gv);
#pragma unroll 1
    for (; h < heads; h += step) {
        float u[8], v[8], du[8], dv[8];
        widen<T>(load_pair<T, D>(x + (int64_t)h * in.head), u, v);
        widen<T>(load_pair<T, D>(dy + (int64_t)h * grad.head), du, dv);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
        const float rstd = 1.f / sqrtf(head_sum<D>(ss) * (1.f / D) + eps);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = du[i] * c[i] + dv[i] * s[i], q = dv[i] * c[i] - du[i] * s[i];
            u[i] *= rstd;
            v[i] *= rstd;
            acc[i] = fmaf(p, u[i], acc[i]);
            acc[8 + i] = fmaf(q, v[i], acc[8 + i]);
            du[i] = p * gu[i];
            dv[i] = q * gv[i];
            dot = fmaf(du[i], u[i], fmaf(dv[i], v[i], dot));
        }
        dot = head_sum<D>(dot) * (1.f / D);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            du[i] = rstd * fmaf(-u[i], dot, du[i]);
            dv[i] = rstd * fmaf(-v[i], dot, dv[i]);
        }
        store8f<T>(dx + (int64_t)h * out.head, du);
        store8f<T>(dx + (int64_t)h * out.head + D / 2, dv);
    }
}

template <typename T, int D> __global__ __launch_bounds__(256, 3) void norm_rope_bwd_kernel(NormRopeArgs a) {
    constexpr int L = D / 16;
    __shared__ float red[256][17];
    const Side side = side_of(a);
    const int tid = threadIdx.x, j = tid % L;
    const int64_t total = a.rows * side.parts, stride = (int64_t)((int)blockIdx.x < a.q_blocks ? a.q_blocks : (int)gridDim.x - a.q_blocks) * (256 / L);
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    for (int64_t rest = side.block * (256 / L) + tid / L; rest < total; rest += stride) {
        const int64_t row = rest / side.parts;
        float c[8], s[8];
        angles(a, row, 8 * j, c, s);
        rotate_heads_bwd<T, D>(side.in, side.grad, side.out, side.gamma, a.eps, row, j, (int)(rest - row * side.parts), side.parts, side.heads, c, s, acc);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) red[tid][i] = acc[i];
    __syncthreads();
    if (tid < D) {                                           // channel tid: lanes of class (tid % (D / 2)) / 8, value tid % 8 (+ 8 in the upper half)
        const int half = tid / (D / 2), cc = tid % (D / 2);
        float sum = 0.f;
#pragma unroll 8
        for (int t = cc / 8; t < 256; t += L) sum += red[t][half * 8 + cc % 8];
        a.partial[(int64_t)blockIdx.x * D + tid] = sum;
    }
}

// dgamma: a block sums four channels over the blocks of q or of k, each thread over every 256th of them, then the threads in a tree
__global__ __launch_bounds__(256) void gamma_grad_kernel(const float* __restrict__ partial, int q_blocks, int blocks, int D, float* dgq, float* dgk, int accumulate) {
    __shared__ double red[4][4];
    const bool isq = (int)blockIdx.x < D / 4;
    const int ch = 4 * (blockIdx.x % (D / 4)), t = threadIdx.x, end = isq ? q_blocks : blocks;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (int b = (isq ? 0 : q_blocks) + t; b < end; b += 256) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(partial + (int64_t)b * D + ch);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += (double)x[i];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += __shfl_xor(s[i], o, 64);
    if (t % 64 == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[t / 64][i] = s[i];
    __syncthreads();
    if (t < 4) {
        const double sum = red[0][t] + red[1][t] + red[2][t] + red[3][t];
        float* out = (isq ? dgq : dgk) + ch + t;
        *out = accumulate ? *out + (float)sum : (float)sum;
    }
}

template <typename T, int D> hipError_t run(const NormRopeArgs& a, int blocks, bool bwd, hipStream_t s) {
    if (bwd) hipLaunchKernelGGL((norm_rope_bwd_kernel<T, D>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((norm_rope_kernel<T, D>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}
template <typename T> hipError_t run(int head_dim, const NormRopeArgs& a, int blocks, bool bwd, hipStream_t s) {
    return head_dim == 64 ? run<T, 64>(a, blocks, bwd, s) : run<T, 128>(a, blocks, bwd, s);
}

// Heads a thread walks: one while rows are few (latency), more - one set of sines for all of them - while twice the threads that run at once remain: 2 forward
// (25 300 rows of 32 + 8 heads of 128, f16: 1 head 113 us, 2: 97, 4: 101, 8: 106), 4 backward, whose blocks stay for many rows (82 688 rows of 16 + 4 heads
// of 64, bf16: 1: 138 us, 2: 130, 4: 128, 8: 130).
int heads_of_a_thread(int64_t rows, int heads, int head_dim, int most) {
    int per = 1;
    while (per < most && per < heads && rows * ((heads + 2 * per - 1) / (2 * per)) * (head_dim / 16) >= (int64_t)256 * 2048) per *= 2;
    return per;
}
// sets parts and q_blocks; the launch's blocks, at most `limit` (> 1)
int64_t share(NormRopeArgs& a, int head_dim, int most, int64_t limit) {
    const int per = heads_of_a_thread(a.rows, a.heads + a.kv_heads, head_dim, most), rows = 256 / (head_dim / 16);
    a.parts = (a.heads + per - 1) / per;
    a.kv_parts = (a.kv_heads + per - 1) / per;
    int64_t nq = (a.rows * a.parts + rows - 1) / rows, nk = (a.rows * a.kv_parts + rows - 1) / rows;
    if (nq + nk > limit) {
        nk = nk * limit / (nq + nk);
        nk = nk < 1 ? 1 : nk < limit ? nk : limit - 1;
        nq = limit - nk;
    }
    a.q_blocks = (int)nq;
    return nq + nk;
}
constexpr int64_t kBwdBlocks = 1536;                         // two rounds of what runs at once (the bf16 case above: 768 blocks 134 us, 1536: 129, 2304: 130)

}  // namespace

int64_t norm_rope_blocks(int64_t rows, int heads, int kv_heads, int head_dim) {
    NormRopeArgs a;
    a.rows = rows;
    a.heads = heads;
    a.kv_heads = kv_heads;
    return share(a, head_dim, 2, (int64_t)1 << 40);
}

int norm_rope_bwd_blocks(int64_t rows, int heads, int kv_heads, int head_dim) {
    NormRopeArgs a;
    a.rows = rows;
    a.heads = heads;
    a.kv_heads = kv_heads;
    return (int)share(a, head_dim, 4, kBwdBlocks);
}

hipError_t launch_norm_rope(int dtype, int head_dim, NormRopeArgs a, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    const int blocks = (int)share(a, head_dim, 2, 0x7fffffff);
    return dtype == 0 ? run<float>(head_dim, a, blocks, false, s) : dtype == 1 ? run<f16_t>(head_dim, a, blocks, false, s) : run<bf16_t>(head_dim, a, blocks, false, s);
}

hipError_t launch_norm_rope_bwd(int dtype, int head_dim, NormRopeArgs a, float* dgq, float* dgk, int accumulate, hipStream_t s) {
    const int blocks = (int)share(a, head_dim, 4, kBwdBlocks);
    if (blocks > 0) {
        const hipError_t e = dtype == 0 ? run<float>(head_dim, a, blocks, true, s) : dtype == 1 ? run<f16_t>(head_dim, a, blocks, true, s) : run<bf16_t>(head_dim, a, blocks, true, s);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(gamma_grad_kernel, dim3((unsigned)(2 * head_dim / 4)), dim3(256), 0, s, a.partial, a.q_blocks, blocks, head_dim, dgq, dgk, accumulate);
    return hipGetLastError();
}
