// Norm of queries and keys for each head with the position rotation in the same pass, and its gradients.  Per row and head, with n = x rsqrt(mean(x^2) + eps):
//     z = n gamma,   y_i = z_i cos a_i - z_{i + D/2} sin a_i,   y_{i + D/2} = z_{i + D/2} cos a_i + z_i sin a_i,   a_i = position theta^(-2 i / D)
//     dz = the rotation by -a of dy,   dgamma = sum dz n,   dx = rstd (dz gamma - n mean(dz gamma n))
// Bound by reading x (and dy) and writing y (dx) once.  A thread holds 8 channels of the lower half of a head and their partners in the upper half, so the
// rotation needs no exchange and D / 16 neighbouring lanes hold a head; it keeps its 8 sines and cosines for every head of its row that it works on.
// The angle is reduced in 64 bits (position x turns-per-position, minus the whole turns): at position 10^6 a 32-bit product is off by 0.06 rad.
#include "causal_core.h"

namespace {
using namespace causal;

template <typename T> __device__ __forceinline__ void load8f(const T* p, float (&x)[8]) {
    const typename Frag<T>::type f = load8<T>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (sizeof(T) == 4) x[j] = f[j];
        else x[j] = (float)__builtin_bit_cast(T, (short)f[j]);
    }
}
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
template <typename T> struct Head { const T* x; const T* dy; T* y; };

// thread -> (row, slice of the row's heads, 8 channel pairs)
struct Spot { int64_t row; int part, j; };

template <typename T, int D> __global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a) {
    constexpr int L = D / 16;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int j = (int)(id % L);
    const int64_t rest = id / L, row = rest / a.parts;
    const int part = (int)(rest - row * a.parts);
    if (row >= a.rows) return;                               // (whole heads: the lanes of a head leave together)
    float c[8], s[8];
    angles(a, row, 8 * j, c, s);
    const int heads = a.heads + a.kv_heads;
    for (int h = part; h < heads; h += a.parts) {
        const bool isq = h < a.heads;
        const Rows3 &in = isq ? a.q : a.k, &out = isq ? a.q_out : a.k_out;
        const int hh = isq ? h : h - a.heads;
        const float* g = (isq ? a.gamma_q : a.gamma_k) + 8 * j;
        const T* x = static_cast<const T*>(in.p) + row * in.row + (int64_t)hh * in.head + 8 * j;
        T* y = static_cast<T*>(out.p) + row * out.row + (int64_t)hh * out.head + 8 * j;
        float u[8], v[8], gu[8], gv[8];
        load8f<T>(x, u);
        load8f<T>(x + D / 2, v);
        load8f<float>(g, gu);
        load8f<float>(g + D / 2, gv);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
        const float rstd = 1.f / sqrtf(head_sum<D>(ss) * (1.f / D) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = u[i] * rstd * gu[i], q = v[i] * rstd * gv[i];
            u[i] = p * c[i] - q * s[i];
            v[i] = q * c[i] + p * s[i];
        }
        store8f<T>(y, u);
        store8f<T>(y + D / 2, v);
    }
}

// Gradients: dx per row; dgamma of q and k summed over a thread's rows, then over the block's threads in a fixed order, then (gamma_grad_kernel) over the blocks.
template <typename T, int D> __global__ __launch_bounds__(256) void norm_rope_bwd_kernel(NormRopeArgs a) {
    constexpr int L = D / 16;
    __shared__ float red[256][17];
    const int tid = threadIdx.x, j = tid % L;
    const int heads = a.heads + a.kv_heads;
    float acc[2][16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[0][i] = acc[1][i] = 0.f;
    const int64_t total = a.rows * a.parts;
    for (int64_t rest = (int64_t)blockIdx.x * (256 / L) + tid / L; rest < total; rest += (int64_t)gridDim.x * (256 / L)) {
        const int64_t row = rest / a.parts;
        const int part = (int)(rest - row * a.parts);
        float c[8], s[8];
        angles(a, row, 8 * j, c, s);
        for (int h = part; h < heads; h += a.parts) {
            const bool isq = h < a.heads;
            const Rows3 &in = isq ? a.q : a.k, &grad = isq ? a.dq_in : a.dk_in, &out = isq ? a.q_out : a.k_out;
            const int hh = isq ? h : h - a.heads;
            const float* g = (isq ? a.gamma_q : a.gamma_k) + 8 * j;
            const T* x = static_cast<const T*>(in.p) + row * in.row + (int64_t)hh * in.head + 8 * j;
            const T* dy = static_cast<const T*>(grad.p) + row * grad.row + (int64_t)hh * grad.head + 8 * j;
            T* dx = static_cast<T*>(out.p) + row * out.row + (int64_t)hh * out.head + 8 * j;
            float u[8], v[8], du[8], dv[8], gu[8], gv[8];
            load8f<T>(x, u);
            load8f<T>(x + D / 2, v);
            load8f<T>(dy, du);
            load8f<T>(dy + D / 2, dv);
            load8f<float>(g, gu);
            load8f<float>(g + D / 2, gv);
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
            const float rstd = 1.f / sqrtf(head_sum<D>(ss) * (1.f / D) + a.eps);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = du[i] * c[i] + dv[i] * s[i], q = dv[i] * c[i] - du[i] * s[i];
                u[i] *= rstd;
                v[i] *= rstd;
                if (isq) {
                    acc[0][i] = fmaf(p, u[i], acc[0][i]);
                    acc[0][8 + i] = fmaf(q, v[i], acc[0][8 + i]);
                } else {
                    acc[1][i] = fmaf(p, u[i], acc[1][i]);
                    acc[1][8 + i] = fmaf(q, v[i], acc[1][8 + i]);
                }
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
            store8f<T>(dx, du);
            store8f<T>(dx + D / 2, dv);
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) red[tid][i] = acc[k][i];
        __syncthreads();
        if (tid < D) {                                       // channel tid: lanes of class (tid % (D / 2)) / 8, value tid % 8 (+ 8 in the upper half)
            const int half = tid / (D / 2), cc = tid % (D / 2);
            float sum = 0.f;
            for (int t = cc / 8; t < 256; t += L) sum += red[t][half * 8 + cc % 8];
            a.partial[((int64_t)blockIdx.x * 2 + k) * D + tid] = sum;
        }
    }
}

__global__ __launch_bounds__(256) void gamma_grad_kernel(const float* __restrict__ partial, int blocks, int D, float* dgq, float* dgk, int accumulate) {
    // one block per 8 channels of the 2 D; 32 threads each walk a channel's partials
    __shared__ double red[256];
    const int ch = blockIdx.x * 8 + (threadIdx.x & 7), t = threadIdx.x >> 3;
    double s = 0.0;
    for (int b = t; b < blocks; b += 32) s += (double)partial[(int64_t)b * 2 * D + ch];
    red[threadIdx.x] = s;
    __syncthreads();
    if (t == 0) {
        for (int i = 1; i < 32; ++i) s += red[i * 8 + threadIdx.x];
        float* out = ch < D ? dgq + ch : dgk + (ch - D);
        *out = accumulate ? *out + (float)s : (float)s;
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

// Threads per row: one head each while rows are few (latency), more heads per thread - one set of sines for all of them - once the machine is full.
int parts_of(int64_t rows, int heads, int head_dim) {
    int per = 1;
    while (per < 8 && per < heads && rows * ((heads + 2 * per - 1) / (2 * per)) * (head_dim / 16) >= (int64_t)256 * 2048) per *= 2;
    return (heads + per - 1) / per;
}

}  // namespace

int norm_rope_bwd_blocks(int64_t rows, int heads, int head_dim) {
    const int64_t items = rows * parts_of(rows, heads, head_dim), per = 256 / (head_dim / 16);
    const int64_t n = (items + per - 1) / per;
    return (int)(n < 1 ? 1 : n > 2048 ? 2048 : n);
}

hipError_t launch_norm_rope(int dtype, int head_dim, NormRopeArgs a, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    a.parts = parts_of(a.rows, a.heads + a.kv_heads, head_dim);
    const int64_t blocks = (a.rows * a.parts * (head_dim / 16) + 255) / 256;
    return dtype == 0 ? run<float>(head_dim, a, (int)blocks, false, s) : dtype == 1 ? run<f16_t>(head_dim, a, (int)blocks, false, s) : run<bf16_t>(head_dim, a, (int)blocks, false, s);
}

hipError_t launch_norm_rope_bwd(int dtype, int head_dim, NormRopeArgs a, float* dgq, float* dgk, int accumulate, hipStream_t s) {
    const int blocks = norm_rope_bwd_blocks(a.rows, a.heads + a.kv_heads, head_dim);
    a.parts = parts_of(a.rows, a.heads + a.kv_heads, head_dim);
    const hipError_t e = dtype == 0 ? run<float>(head_dim, a, blocks, true, s) : dtype == 1 ? run<f16_t>(head_dim, a, blocks, true, s) : run<bf16_t>(head_dim, a, blocks, true, s);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(gamma_grad_kernel, dim3((unsigned)(2 * head_dim / 8)), dim3(256), 0, s, a.partial, blocks, head_dim, dgq, dgk, accumulate);
    return hipGetLastError();
}
