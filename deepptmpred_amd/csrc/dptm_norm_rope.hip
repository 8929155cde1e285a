// Norm of every query and key head and the position rotation, in one pass over the rows.
//
//   r = (mean x^2 + eps)^-1/2;  y = x r g;  (a, b) -> (a cos - b sin, b cos + a sin) for the pairs (i, i + D/2) or (2i, 2i+1)
//   backward: dy back by the opposite rotation;  dg = sum dy x r;  dx = r (g dy - x r^2 mean(g dy x))
//
// Bound by memory: 2 (forward) or 3 (backward) times the data.  D / 16 lanes share a head; a lane holds eight elements of either
// half, so both kinds of pairs are its own, the loads are 16 bytes wide, and the sum over the head is at most three
// exchanges.  A thread keeps the angles and gains of its elements in registers over the heads of a row that it takes.
// All arithmetic is fp32; results are rounded once to the tensors' type.
#include "dptm_layers.h"

namespace dptm {
namespace {

template <typename T> struct Vec { typedef T v8 __attribute__((ext_vector_type(8))); };

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const typename Vec<T>::v8 v = *reinterpret_cast<const typename Vec<T>::v8*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    typename Vec<T>::v8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)x[e];
    *reinterpret_cast<typename Vec<T>::v8*>(p) = v;
}

struct Angles { float c0[8], s0[8], c1[8], s1[8]; };   // of the first and the second eight elements, per element

template <int D>
__device__ __forceinline__ void load_angles(const NormRopeArgs& a, int64_t row, int chunk, bool neighbours, Angles& g) {
    const int64_t pos = a.positions ? (int64_t)a.positions[row] : row;
    if (pos < 0 || pos >= a.n_pos) {      // no such angle: the row says so
#pragma unroll
        for (int e = 0; e < 8; ++e) g.c0[e] = g.s0[e] = g.c1[e] = g.s1[e] = __builtin_nanf("");
        return;
    }
    const float* c = a.cosv + pos * (D / 2);
    const float* s = a.sinv + pos * (D / 2);
    if (neighbours) {
        typedef float f4 __attribute__((ext_vector_type(4)));
        const f4 cl = *reinterpret_cast<const f4*>(c + 4 * chunk), ch = *reinterpret_cast<const f4*>(c + D / 4 + 4 * chunk);
        const f4 sl = *reinterpret_cast<const f4*>(s + 4 * chunk), sh = *reinterpret_cast<const f4*>(s + D / 4 + 4 * chunk);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            g.c0[e] = cl[e / 2], g.s0[e] = sl[e / 2];
            g.c1[e] = ch[e / 2], g.s1[e] = sh[e / 2];
        }
    } else {
        load8<float>(c + 8 * chunk, g.c0);
        load8<float>(s + 8 * chunk, g.s0);
#pragma unroll
        for (int e = 0; e < 8; ++e) g.c1[e] = g.c0[e], g.s1[e] = g.s0[e];
    }
}

// rotates (x0, x1) in place; dir 1 or -1
template <bool NEIGHBOURS>
__device__ __forceinline__ void rotate(float (&x0)[8], float (&x1)[8], const Angles& g, float dir) {
    if constexpr (NEIGHBOURS) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float a = x0[e], b = x0[e + 1], p = x1[e], q = x1[e + 1];
            x0[e] = fmaf(a, g.c0[e], -dir * b * g.s0[e]);
            x0[e + 1] = fmaf(b, g.c0[e], dir * a * g.s0[e]);
            x1[e] = fmaf(p, g.c1[e], -dir * q * g.s1[e]);
            x1[e + 1] = fmaf(q, g.c1[e], dir * p * g.s1[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = x0[e], b = x1[e];
            x0[e] = fmaf(a, g.c0[e], -dir * b * g.s0[e]);
            x1[e] = fmaf(b, g.c0[e], dir * a * g.s0[e]);
        }
    }
}

template <int LANES>
__device__ __forceinline__ float sum_of(float v) {
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

constexpr int kThreads = 256;

// One block takes kThreads / (D / 16) units of (row, first head); a thread goes on with the heads head + hstep, ...
// GRAD: the backward pass, with the sums for the gain gradients kept over all units of the block.
template <typename T, int D, bool NEIGHBOURS, bool GRAD>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs a, int hstep, int64_t units) {
    constexpr int L = D / 16;
    const int chunk = threadIdx.x % L, all = a.heads[0] + a.heads[1];
    float g0[2][8], g1[2][8], d0[2][8], d1[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            g0[t][e] = a.gain[t] ? a.gain[t][8 * chunk + e] : 1.f;
            g1[t][e] = a.gain[t] ? a.gain[t][D / 2 + 8 * chunk + e] : 1.f;
            d0[t][e] = d1[t][e] = 0.f;
        }
    // a whole group of lanes runs out of units together: units are counted per group
    for (int64_t u = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L; u < units; u += (int64_t)gridDim.x * (kThreads / L)) {
        const int64_t row = u / hstep;
        Angles ang;
        load_angles<D>(a, row, chunk, NEIGHBOURS, ang);
        for (int head = (int)(u - row * hstep); head < all; head += hstep) {
            const bool isk = head >= a.heads[0];
            const int t = isk ? 1 : 0, hh = isk ? head - a.heads[0] : head;
            const bool norm = a.gain[t] != nullptr;
            const T* px = static_cast<const T*>(a.x[t].p) + row * a.x[t].row + hh * a.x[t].head + 8 * chunk;
            float x0[8], x1[8];
            load8<T>(px, x0);
            load8<T>(px + D / 2, x1);
            float r = 1.f;
            if (norm) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], ss));
                // sqrt and divide, not the approximate reciprocal root: the norm is part of every output
                r = 1.f / sqrtf(sum_of<L>(ss) * (1.f / D) + a.eps);
            }
            if constexpr (!GRAD) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x0[e] *= r * (isk ? g0[1][e] : g0[0][e]);
                    x1[e] *= r * (isk ? g1[1][e] : g1[0][e]);
                }
                rotate<NEIGHBOURS>(x0, x1, ang, 1.f);
                T* py = static_cast<T*>(a.y[t].p) + row * a.y[t].row + hh * a.y[t].head + 8 * chunk;
                store8<T>(py, x0);
                store8<T>(py + D / 2, x1);
            } else {
                const T* pd = static_cast<const T*>(a.dy[t].p) + row * a.dy[t].row + hh * a.dy[t].head + 8 * chunk;
                float y0[8], y1[8];
                load8<T>(pd, y0);
                load8<T>(pd + D / 2, y1);
                rotate<NEIGHBOURS>(y0, y1, ang, -1.f);
                if (norm) {
                    float dot = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float z0 = y0[e] * x0[e] * r, z1 = y1[e] * x1[e] * r;
                        d0[0][e] += isk ? 0.f : z0, d1[0][e] += isk ? 0.f : z1;
                        d0[1][e] += isk ? z0 : 0.f, d1[1][e] += isk ? z1 : 0.f;
                        y0[e] *= isk ? g0[1][e] : g0[0][e];
                        y1[e] *= isk ? g1[1][e] : g1[0][e];
                        dot = fmaf(y0[e], x0[e], fmaf(y1[e], x1[e], dot));
                    }
                    const float f = sum_of<L>(dot) * (1.f / D) * r * r;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        y0[e] = r * fmaf(-f, x0[e], y0[e]);
                        y1[e] = r * fmaf(-f, x1[e], y1[e]);
                    }
                }
                T* po = static_cast<T*>(a.dx[t].p) + row * a.dx[t].row + hh * a.dx[t].head + 8 * chunk;
                store8<T>(po, y0);
                store8<T>(po + D / 2, y1);
            }
        }
    }
    if constexpr (GRAD) {
        // the block's threads with one chunk, in order of their index
        __shared__ float sums[kThreads * 17];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (!a.gain[t]) continue;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sums[threadIdx.x * 17 + e] = d0[t][e];
                sums[threadIdx.x * 17 + 8 + e] = d1[t][e];
            }
            __syncthreads();
            if (threadIdx.x < D) {
                const int e = threadIdx.x % (D / 2), c = e / 8, at = e % 8 + (threadIdx.x < D / 2 ? 0 : 8);
                float x = 0.f;
                for (int i = c; i < kThreads; i += L) x += sums[i * 17 + at];
                a.part[t][(int64_t)blockIdx.x * D + threadIdx.x] = x;
            }
        }
    }
}

// gain gradients from the blocks' sums, in 64 bits and in a fixed order: one wavefront a column
__global__ __launch_bounds__(64) void gain_sum_kernel(const float* p0, const float* p1, float* o0, float* o1, int blocks, int dim) {
    const float* p = blockIdx.y ? p1 : p0;
    float* o = blockIdx.y ? o1 : o0;
    if (!o) return;
    double x = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 64) x += (double)p[(int64_t)i * dim + blockIdx.x];
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
    if (threadIdx.x == 0) o[blockIdx.x] = (float)x;
}

// heads a thread takes in a row: one while the call does not fill the card, four beyond
int head_step(int64_t rows, int all, int dim) {
    const int64_t threads = rows * all * (dim / 16);
    return threads > 4 * 256 * 2048 ? (all + 3) / 4 : all;
}

template <typename T, int D>
hipError_t forward(const NormRopeArgs& a, hipStream_t s) {
    const int all = a.heads[0] + a.heads[1], step = head_step(a.rows, all, D);
    const int64_t units = a.rows * step, blocks = (units + kThreads / (D / 16) - 1) / (kThreads / (D / 16));
    if (a.interleaved)
        hipLaunchKernelGGL((norm_rope_kernel<T, D, true, false>), dim3((unsigned)blocks), dim3(kThreads), 0, s, a, step, units);
    else
        hipLaunchKernelGGL((norm_rope_kernel<T, D, false, false>), dim3((unsigned)blocks), dim3(kThreads), 0, s, a, step, units);
    return hipGetLastError();
}

template <typename T, int D>
hipError_t backward(const NormRopeArgs& a, hipStream_t s) {
    const int all = a.heads[0] + a.heads[1], step = head_step(a.rows, all, D);
    const int64_t units = a.rows * step;
    const int blocks = norm_rope_blocks(a.rows, all, D);
    if (a.interleaved)
        hipLaunchKernelGGL((norm_rope_kernel<T, D, true, true>), dim3(blocks), dim3(kThreads), 0, s, a, step, units);
    else
        hipLaunchKernelGGL((norm_rope_kernel<T, D, false, true>), dim3(blocks), dim3(kThreads), 0, s, a, step, units);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || (!a.gain[0] && !a.gain[1])) return e;
    hipLaunchKernelGGL(gain_sum_kernel, dim3(D, 2), dim3(64), 0, s, a.part[0], a.part[1], a.gain[0] ? a.dgain[0] : nullptr,
                       a.gain[1] ? a.dgain[1] : nullptr, blocks, D);
    return hipGetLastError();
}

template <typename T>
hipError_t by_dim(const NormRopeArgs& a, bool grad, hipStream_t s) {
    switch (a.dim) {
        case 16: return grad ? backward<T, 16>(a, s) : forward<T, 16>(a, s);
        case 32: return grad ? backward<T, 32>(a, s) : forward<T, 32>(a, s);
        case 64: return grad ? backward<T, 64>(a, s) : forward<T, 64>(a, s);
        default: return grad ? backward<T, 128>(a, s) : forward<T, 128>(a, s);
    }
}

hipError_t by_type(const NormRopeArgs& a, int dtype, bool grad, hipStream_t s) {
    return dtype == 1 ? by_dim<__bf16>(a, grad, s) : dtype == 2 ? by_dim<_Float16>(a, grad, s) : by_dim<float>(a, grad, s);
}

}  // namespace

// blocks of the backward pass: they walk over the units, so that there are few partial sums
int norm_rope_blocks(int64_t rows, int heads, int dim) {
    const int64_t per = kThreads / (dim / 16), units = rows * head_step(rows, heads, dim);
    const int64_t want = (units + per - 1) / per;
    return (int)(want < 1024 ? (want < 1 ? 1 : want) : 1024);
}

hipError_t norm_rope_forward(const NormRopeArgs& a, int dtype, hipStream_t s) { return by_type(a, dtype, false, s); }
hipError_t norm_rope_backward(const NormRopeArgs& a, int dtype, hipStream_t s) { return by_type(a, dtype, true, s); }

}  // namespace dptm
