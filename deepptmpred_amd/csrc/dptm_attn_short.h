// Attention over packed sequences, backward pass of batches whose sequences have up to 64 rows and 64 keys: windows.
//
// One workgroup per sequence and head forms dq, dk, dv and the bias gradient together, because nothing of it is needed
// elsewhere: scores and weights once (five products for the seven of the two kernels in dptm_attn_grad.h), every tensor read once,
// one launch for two.  A wavefront owns 32 keys and goes over the rows as the dk, dv kernel does; dS then crosses over through LDS, in
// fp32, into the layout that dq needs and along whose diagonals the bias gradient lies.
//
// Backward pass of 1,000 windows, 8 heads, with a bias, this kernel against those two, in us: 51 rows, bf16 heads of 64 157 : 280,
// of 32 79 : 154, f16 heads of 16 58 : 137, fp32 heads of 64 389 : 695; 33 rows, fp32 heads of 32 156 : 251; 21 rows, fp32 heads of 16
// 68 : 120; one window 25 : 27.  It is bound by its 128 threads' way from memory through five barriers back: the bytes of 8,192
// windows' heads of 16 in fp32 take 29 us, their matrix instructions 41, the kernel 125.  Heads of 128 would leave one
// wavefront a SIMD, and heads that share keys would need a sum over workgroups: both take the two kernels.
#pragma once
#include "dptm_attn_grad.h"

namespace dptm {
namespace {

constexpr int kShort = 64;       // rows, and keys
constexpr int kDsRow = 72;       // floats between rows of dS: the two halves of a wavefront write 32 banks apart

template <typename T, int D> constexpr int kShortFirst = 2 * kShort * D * (int)sizeof(T) > 4 * kShort * kDsRow ? 2 * kShort * D * (int)sizeof(T)
                                                                                                          : 4 * kShort * kDsRow;
template <typename T, int D> inline size_t short_lds(const AttnArgs& a) {
    return kShortFirst<T, D> + kShort * D * sizeof(T) + (2 * kShort + 4 * kShort + bias_floats(a)) * 4;
}

template <typename T, int D, bool BIAS>
__global__ __launch_bounds__(128, (D * sizeof(T) <= 64 ? 3 : 2)) void attn_short_grad_kernel(AttnArgs a, int k_items_at) {
    constexpr int DT = D >= 32 ? D / 32 : 1, ST = D / 16, kBytes = kShort * D * (int)sizeof(T);
    extern __shared__ char smem[];
    char* qt = smem;                                        // rows of q and dout, later dS
    char* gt = smem + kBytes;
    float* ds = reinterpret_cast<float*>(smem);
    char* kt = smem + kShortFirst<T, D>;
    float* rowref = reinterpret_cast<float*>(kt + kBytes);
    float* rowdelta = rowref + kShort;
    float* sums = rowdelta + kShort;                        // [2][128]: by key - row + 64, per half of the rows
    float* bias = sums + 4 * kShort;
    const int reach = a.bias.reach;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // heads of a sequence next to each other: a head's row may be part of a cache line
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int item = id / a.heads, head = id - item * a.heads;
    const QItem qi = reinterpret_cast<const QItem*>(a.plan + a.items_at)[item];
    const KItem ki = reinterpret_cast<const KItem*>(a.plan + k_items_at)[item];
    const int nq = qi.nq, nk = ki.nk, pos0 = ki.pos0;
    const int words = 2 * reach + 1 + 2 * kFarPad;
    float* part = a.part_bias + ((int64_t)head * a.n_items + item) * words;
    if (nq == 0 || nk == 0) {
        constexpr int kChunks = D * (int)sizeof(T) / 16;
        for (int i = tid; i < (nq + nk) * kChunks; i += 128) {
            const int row = i / kChunks;
            char* q = reinterpret_cast<char*>(const_cast<T*>(row < nq ? row_ptr<T>(a.dq, (int64_t)qi.q0 + row, head) : row_ptr<T>(a.dk, (int64_t)ki.k0 + row - nq, head)));
            *reinterpret_cast<u32x4_a*>(q + i % kChunks * 16) = u32x4_a{0, 0, 0, 0};
            if (row >= nq)
                *reinterpret_cast<u32x4_a*>(reinterpret_cast<char*>(const_cast<T*>(row_ptr<T>(a.dv, (int64_t)ki.k0 + row - nq, head))) + i % kChunks * 16) = u32x4_a{0, 0, 0, 0};
        }
        if constexpr (BIAS)
            for (int i = tid; i < words; i += 128) part[i] = 0.f;
        return;
    }
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;
    const int mine = 32 * w + (lane & 31);                  // this lane's key, and its row
    const int keyc = min(mine, nk - 1), rowc = min(mine, nq - 1);
    const int64_t qr = (int64_t)qi.q0 + rowc;

    Stage<T, D, kShort, 128> sq(a.q.row * (int)sizeof(T), tid), sg(a.dout.row * (int)sizeof(T), tid), sk(a.k.row * (int)sizeof(T), tid);
    sq.load(reinterpret_cast<const char*>(row_ptr<T>(a.q, qi.q0, head)), nq, tid);
    sg.load(reinterpret_cast<const char*>(row_ptr<T>(a.dout, qi.q0, head)), nq, tid);
    sk.load(reinterpret_cast<const char*>(row_ptr<T>(a.k, ki.k0, head)), nk, tid);
    const char* vrow = reinterpret_cast<const char*>(row_ptr<T>(a.v, (int64_t)ki.k0 + keyc, head));
    const char* grow = reinterpret_cast<const char*>(row_ptr<T>(a.dout, qr, head));
    const char* orow = reinterpret_cast<const char*>(row_ptr<T>(a.out, qr, head));
    const float lse = a.lse[(int64_t)head * a.q_rows + qr];
    V8<T> kf[ST], vf[ST];
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        const V8<T> g = global_frag<T>(grow, s, h), o = global_frag<T>(orow, s, h);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)g[e], (float)o[e], delta);
        vf[s] = global_frag<T>(vrow, s, h);
    }
    delta = half_sum(delta);
    if constexpr (BIAS) load_bias<T>(bias, a.bias, 1.f / a.scale, a.heads, head, tid, 128);
    sq.store(qt, tid);
    sg.store(gt, tid);
    sk.store(kt, tid);
    unsigned odd = 0;
    if (!Sight(win, pos0, pos0 + nq - 1).all(0, nk)) odd = sq.not_finite() | sg.not_finite() | sk.not_finite();
    if (h == 0) {
        // rows behind the last weigh nothing: their scores start from -inf
        rowref[mine] = mine < nq ? lse_log2(lse) * (-1.f / c) : kMinusInf;
        rowdelta[mine] = mine < nq ? -delta : 0.f;
    }
    const bool redo = __syncthreads_or((int)odd);
    if (redo) {
        if (h == 0 && mine < nq) a.delta[(int64_t)head * a.q_rows + qr] = delta;
        __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < ST; ++s) kf[s] = Tile<T, D>::row_frag(kt, mine, s, h);

    f32x16_a dk[DT], dv[DT], d_s[2];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) d_s[u][r] = 0.f;
        const int r0 = 32 * u;
        const Sight sight(win, pos0 + r0, pos0 + min(r0 + 31, nq - 1));
        if ((32 * w < nk) & (r0 < nq) & !sight.none(32 * w, 32)) {
            const bool full = (32 * w + 32 <= nk) & (r0 + 32 <= nq) & sight.all(32 * w, 32);
            const int far = mine - (pos0 + r0 + 4 * h);     // to the row of register 0
            f32x16_a s, p;
            const V4<float>* less = reinterpret_cast<const V4<float>*>(rowref + r0 + 4 * h);
            const V4<float>* del = reinterpret_cast<const V4<float>*>(rowdelta + r0 + 4 * h);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const V4<float> y = less[2 * x], z = del[2 * x];
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * x + e] = y[e], p[4 * x + e] = z[e];
            }
            if constexpr (BIAS) {
                const float* b = bias + bias_at(far - kBiasPad, reach) + kBiasPad;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] += b[-reg_row(r)];
            }
            row_products<T, D, 4>(s, p, qt, gt, r0, kf, vf, lane);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = __builtin_amdgcn_exp2f(s[r] * c);
                p[r] *= s[r];
            }
            if (!full) {
                // row c is seen if far - c <= right and far - c >= -left, or the key is one of the first
                const int lo = far - win.right, hi = min(mine < win.sinks ? kFar : far + win.left, nq - 1 - r0 - 4 * h);
                const int m = mine < nk ? max(hi - lo + 1, 0) : 0;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool see = (unsigned)(reg_row(r) - lo) < (unsigned)m;
                    s[r] = see ? s[r] : 0.f;
                    p[r] = see ? p[r] : 0.f;
                }
            }
            Cols<T, D> cols;
            cols.read(gt, r0, lane);
            cols.product(dv, s);
            cols.read(qt, r0, lane);
            cols.product(dk, p);
            d_s[u] = p;
        }
    }
    if (redo) {
        float x[16 * DT], y[16 * DT];
        dkv_by_pairs<T, D, DT, BIAS>(kernel_args(), x, y, k_items_at, item, head, keyc, h);
        take<DT>(dk, x);
        take<DT>(dv, y);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[(32 * u + reg_row(r) + 4 * h) * kDsRow + mine] = d_s[u][r];
    __syncthreads();
    if (mine < nk) {
        T* ok = const_cast<T*>(row_ptr<T>(a.dk, (int64_t)ki.k0 + mine, head));
        T* ov = const_cast<T*>(row_ptr<T>(a.dv, (int64_t)ki.k0 + mine, head));
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < (D >= 32 ? 4 : 2); ++x) {
                V4<T> y, z;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (T)(dk[d][4 * x + e] * a.scale), z[e] = (T)dv[d][4 * x + e];
                *reinterpret_cast<V4<T>*>(ok + 32 * d + 8 * x + 4 * h) = y;
                *reinterpret_cast<V4<T>*>(ov + 32 * d + 8 * x + 4 * h) = z;
            }
    }
    f32x16_a dq[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if ((32 * w < nq) & (32 * u < nk)) {
            Cols<T, D> cols;
            cols.read(kt, 32 * u, lane);
            f32x16_a s;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const V4<float> y = *reinterpret_cast<const V4<float>*>(ds + mine * kDsRow + 32 * u + 8 * x + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * x + e] = y[e];
            }
            cols.product(dq, s);
        }
    if constexpr (BIAS) {
        // lane l adds up keys l, l + 1, ... of rows 0, 1, ..., which wrap to the diagonal 64 below
        float up[2] = {0.f, 0.f}, down[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int row = 32 * w + i;
            const float x = ds[row * kDsRow + ((row + lane) & 63)];
            const bool wraps = row + lane >= 64;
            up[i & 1] += wraps ? 0.f : x;
            down[i & 1] += wraps ? x : 0.f;
        }
        sums[128 * w + lane] = down[0] + down[1];
        sums[128 * w + 64 + lane] = up[0] + up[1];
    }
    if (redo) {
        float t[16 * DT];
        dq_by_pairs<T, D, DT, BIAS>(kernel_args(), t, item, head, rowc, pos0 + rowc, bias, h);
        take<DT>(dq, t);
    }
    if (mine < nq) {
        T* o = const_cast<T*>(row_ptr<T>(a.dq, (int64_t)qi.q0 + mine, head));
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < (D >= 32 ? 4 : 2); ++x) {
                V4<T> y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (T)(dq[d][4 * x + e] * a.scale);
                *reinterpret_cast<V4<T>*>(o + 32 * d + 8 * x + 4 * h) = y;
            }
    }
    if constexpr (BIAS) {
        __syncthreads();
        for (int i = tid; i < words; i += 128) {
            // the word's distance from a row's position to a key, as an index of `sums`; the outer words take what lies beyond
            const int t = i - reach - kFarPad + pos0 + 64;
            const int from = i == 0 ? 0 : max(t, 0), to = i == words - 1 ? 127 : min(t, 127);
            float x = 0.f;
            for (int k = from; k <= to; ++k) x += sums[k] + sums[128 + k];
            part[i] = x;
        }
    }
}

template <typename T, int D>
hipError_t short_grad_dim(const AttnArgs& a, int k_items_at, hipStream_t s) {
    if constexpr (D <= kShortDim) {
        const int64_t blocks = (int64_t)a.n_items * a.heads;
        return a.bias.table ? start(attn_short_grad_kernel<T, D, true>, blocks, 128, short_lds<T, D>(a), s, a, k_items_at)
                            : start(attn_short_grad_kernel<T, D, false>, blocks, 128, short_lds<T, D>(a), s, a, k_items_at);
    } else {
        return hipErrorInvalidValue;
    }
}

}  // namespace
}  // namespace dptm
