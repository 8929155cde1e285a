// Norm of every query and key head and the position rotation, in one pass over the rows.
//
//   r = (mean x^2 + eps)^-1/2;  y = x r g;  (a, b) -> (a cos - b sin, b cos + a sin) for the pairs (i, i + D/2) or (2i, 2i+1)
//   backward: dy back by the opposite rotation;  dg = sum dy x r;  dx = r (g dy - x r^2 mean(g dy x))
//
// Bound by memory: 2 (forward) or 3 (backward) times the data.  D / 16 lanes share a head; a lane holds eight elements of either
// half, so both kinds of pairs are its own, the loads are 16 bytes wide, and the sum over the head is at most three
// exchanges.  A thread keeps the angles and gains of its elements in registers over the heads of a row that it takes.
// All arithmetic is fp32; results are rounded once to the tensors' type.  65,539 rows of 40 heads of 64, bf16: forward 125 us for
// 671 MB (5.4 TB/s), backward 228 + 5 us for 1,007 MB (4.4 TB/s; a large copy reaches 5.05); 482 rows 4.4 us, the launch.
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

template <int D, bool NEIGHBOURS>
__device__ __forceinline__ void load_angles(const float* cosv, const float* sinv, const int* positions, int n_pos, int64_t row, int chunk, Angles& g) {
    const int64_t want = positions ? (int64_t)positions[row] : row;
    const bool there = want >= 0 && want < n_pos;
    const int64_t pos = there ? want : 0;
    const float* c = cosv + pos * (D / 2);
    const float* s = sinv + pos * (D / 2);
    // no such angle: the row says so
    const float none = __builtin_nanf("");
    if constexpr (NEIGHBOURS) {
        typedef float f4 __attribute__((ext_vector_type(4)));
        f4 cl{none, none, none, none}, ch = cl, sl = cl, sh = cl;
        if (there) {
            cl = *reinterpret_cast<const f4*>(c + 4 * chunk), ch = *reinterpret_cast<const f4*>(c + D / 4 + 4 * chunk);
            sl = *reinterpret_cast<const f4*>(s + 4 * chunk), sh = *reinterpret_cast<const f4*>(s + D / 4 + 4 * chunk);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            g.c0[e] = cl[e / 2], g.s0[e] = sl[e / 2];
            g.c1[e] = ch[e / 2], g.s1[e] = sh[e / 2];
        }
    } else {
        typedef float f8 __attribute__((ext_vector_type(8)));
        f8 cl{none, none, none, none, none, none, none, none}, sl = cl;
        if (there) cl = *reinterpret_cast<const f8*>(c + 8 * chunk), sl = *reinterpret_cast<const f8*>(s + 8 * chunk);
#pragma unroll
        for (int e = 0; e < 8; ++e) g.c0[e] = g.c1[e] = cl[e], g.s0[e] = g.s1[e] = sl[e];
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

// a head's place: the tensors of q and k lie apart; both addresses are formed and one chosen, because a choice between the
// arguments themselves would move those to private memory
template <typename T>
__device__ __forceinline__ T* head_ptr(Strided q, Strided k, bool isk, int64_t row, int head, int chunk) {
    T* pq = static_cast<T*>(q.p) + row * q.row + head * q.head + 8 * chunk;
    T* pk = static_cast<T*>(k.p) + row * k.row + head * k.head + 8 * chunk;
    return isk ? pk : pq;
}

// One block takes kThreads / (D / 16) units of (row, first head) at a time; a thread has the heads head, head + hstep, ...
// (HEADS of them), all asked for before the first is used.  GRAD: the backward pass, with the sums for the gain
// gradients kept over all units of the block.
template <typename T, int D, bool NEIGHBOURS, bool GRAD, int HEADS>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs a, int hstep, int64_t units) {
    constexpr int L = D / 16;
    const int chunk = threadIdx.x % L, all = a.heads[0] + a.heads[1];
    const bool norm_q = a.gain[0] != nullptr, norm_k = a.gain[1] != nullptr;
    const int heads_q = a.heads[0];
    float gq0[8], gq1[8], gk0[8], gk1[8], d0[2][8], d1[2][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        gq0[e] = gq1[e] = gk0[e] = gk1[e] = 1.f;
        d0[0][e] = d0[1][e] = d1[0][e] = d1[1][e] = 0.f;
    }
    if (norm_q) load8<float>(a.gain[0] + 8 * chunk, gq0), load8<float>(a.gain[0] + D / 2 + 8 * chunk, gq1);
    if (norm_k) load8<float>(a.gain[1] + 8 * chunk, gk0), load8<float>(a.gain[1] + D / 2 + 8 * chunk, gk1);
    // a whole group of lanes runs out of units together: units are counted per group
    for (int64_t u = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L; u < units; u += (int64_t)gridDim.x * (kThreads / L)) {
        const int64_t row = u / hstep;
        const int first = (int)(u - row * hstep);
        float x0[HEADS][8], x1[HEADS][8], y0[HEADS][8], y1[HEADS][8];
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            const int head = first + i * hstep;
            if (head >= all) break;
            const bool isk = head >= heads_q;
            const int hh = isk ? head - heads_q : head;
            const T* px = head_ptr<T>(a.x[0], a.x[1], isk, row, hh, chunk);
            load8<T>(px, x0[i]);
            load8<T>(px + D / 2, x1[i]);
            if constexpr (GRAD) {
                const T* pd = head_ptr<T>(a.dy[0], a.dy[1], isk, row, hh, chunk);
                load8<T>(pd, y0[i]);
                load8<T>(pd + D / 2, y1[i]);
            }
        }
        Angles ang;
        load_angles<D, NEIGHBOURS>(a.cosv, a.sinv, a.positions, a.n_pos, row, chunk, ang);
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            const int head = first + i * hstep;
            if (head >= all) break;
            const bool isk = head >= heads_q, norm = isk ? norm_k : norm_q;
            const int hh = isk ? head - heads_q : head;
            float r = 1.f;
            if (norm) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(x0[i][e], x0[i][e], fmaf(x1[i][e], x1[i][e], ss));
                // sqrt and divide, not the approximate reciprocal root: the norm is part of every output
                r = 1.f / sqrtf(sum_of<L>(ss) * (1.f / D) + a.eps);
            }
            if constexpr (!GRAD) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x0[i][e] *= r * (isk ? gk0[e] : gq0[e]);
                    x1[i][e] *= r * (isk ? gk1[e] : gq1[e]);
                }
                rotate<NEIGHBOURS>(x0[i], x1[i], ang, 1.f);
                T* py = head_ptr<T>(a.y[0], a.y[1], isk, row, hh, chunk);
                store8<T>(py, x0[i]);
                store8<T>(py + D / 2, x1[i]);
            } else {
                rotate<NEIGHBOURS>(y0[i], y1[i], ang, -1.f);
                if (norm) {
                    float dot = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float z0 = y0[i][e] * x0[i][e] * r, z1 = y1[i][e] * x1[i][e] * r;
                        d0[0][e] += isk ? 0.f : z0, d1[0][e] += isk ? 0.f : z1;
                        d0[1][e] += isk ? z0 : 0.f, d1[1][e] += isk ? z1 : 0.f;
                        y0[i][e] *= isk ? gk0[e] : gq0[e];
                        y1[i][e] *= isk ? gk1[e] : gq1[e];
                        dot = fmaf(y0[i][e], x0[i][e], fmaf(y1[i][e], x1[i][e], dot));
                    }
                    const float f = sum_of<L>(dot) * (1.f / D) * r * r;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        y0[i][e] = r * fmaf(-f, x0[i][e], y0[i][e]);
                        y1[i][e] = r * fmaf(-f, x1[i][e], y1[i][e]);
                    }
                }
                T* po = head_ptr<T>(a.dx[0], a.dx[1], isk, row, hh, chunk);
                store8<T>(po, y0[i]);
                store8<T>(po + D / 2, y1[i]);
            }
        }
    }
    if constexpr (GRAD) {
        // the block's threads with one chunk: kThreads / D threads a column for every so many of them, in order of their index
        // (one thread a column walks over 4096 / D of them: at heads of 32 two thirds of a short call's last 3 us).  In 64 bits: in 32
        // the gains' gradients were 1.7 times as far off as those of elementary operations (now 1.3: a thread's own sums)
        __shared__ float sums[kThreads * 17];
        __shared__ double some[kThreads];
        constexpr int kSplit = kThreads / D;
        const int col = threadIdx.x % D, c = col % (D / 2) / 8, at = col % 8 + (col < D / 2 ? 0 : 8);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (!(t ? norm_k : norm_q)) continue;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sums[threadIdx.x * 17 + e] = d0[t][e];
                sums[threadIdx.x * 17 + 8 + e] = d1[t][e];
            }
            __syncthreads();
            double x = 0.0;
#pragma unroll 8
            for (int i = c + L * (threadIdx.x / D); i < kThreads; i += L * kSplit) x += (double)sums[i * 17 + at];
            some[threadIdx.x] = x;
            __syncthreads();
            if (threadIdx.x < D) {
#pragma unroll
                for (int k = 1; k < kSplit; ++k) x += some[k * D + col];
                (t ? a.part[1] : a.part[0])[(int64_t)blockIdx.x * D + col] = (float)x;
            }
        }
    }
}

// gain gradients from the blocks' sums, in 64 bits and in a fixed order: 64 columns a block where there are as many, the
// threads in rows below each other
__global__ __launch_bounds__(1024) void gain_sum_kernel(const float* p0, const float* p1, float* o0, float* o1, int blocks, int dim) {
    __shared__ double sums[1024];
    const float* p = blockIdx.y ? p1 : p0;
    float* o = blockIdx.y ? o1 : o0;
    if (!o) return;
    const int cols = dim < 16 ? dim : 16, rows = 1024 / cols;
    const int col = blockIdx.x * cols + threadIdx.x % cols, row = threadIdx.x / cols;
    double x = 0.0;
#pragma unroll 8
    for (int i = row; i < blocks; i += rows) x += (double)p[(int64_t)i * dim + col];
    sums[threadIdx.x] = x;
    for (int k = rows / 2; k; k >>= 1) {
        __syncthreads();
        if (row < k) sums[threadIdx.x] += sums[threadIdx.x + k * cols];
    }
    if (row == 0) o[col] = (float)sums[threadIdx.x];
}

// heads a thread takes in a row: one while the call does not fill the card (8,000 rows of 40 heads of 64, bf16: forward 17.3 us and
// backward 31.6, with more heads 18.2 and 34.7), HEADS beyond (65,539 rows: 145 and 218 with one, 122 and 212)
constexpr int kForwardHeads = 4, kBackwardHeads = 2;
bool large(int64_t rows, int all, int dim) { return rows * all * (dim / 16) > 4 * 256 * 2048; }

template <typename T, int D, bool GRAD, int HEADS>
hipError_t run(const NormRopeArgs& a, int blocks, hipStream_t s) {
    const int all = a.heads[0] + a.heads[1], step = (all + HEADS - 1) / HEADS;
    const int64_t units = a.rows * step;
    if (!GRAD) blocks = (int)((units + kThreads / (D / 16) - 1) / (kThreads / (D / 16)));
    return launch(a.interleaved ? norm_rope_kernel<T, D, true, GRAD, HEADS> : norm_rope_kernel<T, D, false, GRAD, HEADS>, dim3(blocks), dim3(kThreads), 0, s,
                  a, step, units);
}

template <typename T, int D>
hipError_t forward(const NormRopeArgs& a, hipStream_t s) {
    return large(a.rows, a.heads[0] + a.heads[1], D) ? run<T, D, false, kForwardHeads>(a, 0, s) : run<T, D, false, 1>(a, 0, s);
}

template <typename T, int D>
hipError_t backward(const NormRopeArgs& a, hipStream_t s) {
    const int all = a.heads[0] + a.heads[1], blocks = norm_rope_blocks(a.rows, all, D);
    const hipError_t e = large(a.rows, all, D) ? run<T, D, true, kBackwardHeads>(a, blocks, s) : run<T, D, true, 1>(a, blocks, s);
    if (e != hipSuccess || (!a.gain[0] && !a.gain[1])) return e;
    return launch(gain_sum_kernel, dim3(D / 16, 2), dim3(1024), 0, s, a.part[0], a.part[1], a.gain[0] ? a.dgain[0] : nullptr,
                  a.gain[1] ? a.dgain[1] : nullptr, blocks, D);
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
    const int64_t per = kThreads / (dim / 16), step = large(rows, heads, dim) ? (heads + kBackwardHeads - 1) / kBackwardHeads : heads;
    const int64_t want = (rows * step + per - 1) / per;
    return (int)(want < 1536 ? (want < 1 ? 1 : want) : 1536);
}

hipError_t norm_rope_forward(const NormRopeArgs& a, int dtype, hipStream_t s) { return by_type(a, dtype, false, s); }
hipError_t norm_rope_backward(const NormRopeArgs& a, int dtype, hipStream_t s) { return by_type(a, dtype, true, s); }

}  // namespace dptm
