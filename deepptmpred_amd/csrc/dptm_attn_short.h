// Attention over packed sequences, backward pass of batches whose sequences have up to 64 rows and 64 keys: windows.
//
// One workgroup per sequence and head forms dq, dk, dv and the bias gradient together, because nothing of it is needed
// elsewhere: scores and weights once (five products for the seven of the two kernels in dptm_attn_grad.h), every tensor read once,
// one launch for two.  A wavefront owns 32 keys and goes over the rows as the dk, dv kernel does; dS then crosses over through LDS, in
// fp32, into the layout that dq needs and along whose diagonals the bias gradient lies.
//
// dS_ij = P_ij (dP_ij - delta_i): delta_i = sum_j P_ij dP_ij is summed from the pairs themselves, in fp32, and `out` is not read.  From
// out as it was rounded (dout_i . out_i, as the other kernels have it) the error of dq and dk of a bf16 window of some 50 keys
// is 1.7 times that of rounding the results, so 1.4 times.  Where a delta is not finite, dS of hidden pairs is set to zero once more.
//
// Backward pass of 1,000 windows, 8 heads, with a bias, this kernel against those two, in us: 51 rows, bf16 heads of 64 144 : 280,
// of 32 75 : 154, f16 heads of 16 61 : 137, fp32 heads of 64 323 : 695; 33 rows, fp32 heads of 32 149 : 251; 21 rows, bf16 heads of 64
// 51 : 161, fp32 heads of 16 47 : 120; one window 25 : 27.  Of 2,048 windows of 51 rows with 4 fp32 heads of 16 the bytes take
// 29 us, the matrix instructions 65 (products that end in the head's 16 columns fill half of each), the kernel 125: the rest is a
// workgroup's way from memory through five barriers back.  Heads of 128 would leave one wavefront a SIMD, and heads that
// share keys would need a sum over workgroups: both take the two kernels.
#pragma once
#include "dptm_attn_grad.h"

namespace dptm {
namespace {

// N = 1 or 2 wavefronts, for up to 32 N rows and keys
template <typename T, int D, int N> struct Short {
    static constexpr int kRows = 32 * N, kBytes = kRows * D * (int)sizeof(T);
    static constexpr int kDsRow = kRows + 8;       // floats between rows of dS: the two halves of a wavefront write 32 banks apart
    static constexpr int kFirst = 2 * kBytes > 4 * kRows * kDsRow ? 2 * kBytes : 4 * kRows * kDsRow;
    static constexpr int kFloats = (1 + N + 4) * kRows;
    static size_t lds(const AttnArgs& a) { return kFirst + kBytes + (kFloats + bias_floats(a)) * 4; }
};

// x or y of this lane, and the same of the one that CTRL names, added
template <int CTRL> __device__ __forceinline__ float with_lane(float x, float y, bool take_y) {
    const float p = x + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, true));
    const float q = y + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(y), CTRL, 0xf, 0xf, true));
    return take_y ? q : p;
}
// Sums of the 16 registers over the 32 lanes of each half of a wavefront: lane l gets that of register l % 16.  Every step halves
// the values a lane still carries.
__device__ __forceinline__ float lane_sums(const f32x16_a& x, int lane) {
    float a[8], b[4], c[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = with_lane<0xb1>(x[2 * i], x[2 * i + 1], lane & 1);       // lane ^ 1
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = with_lane<0x4e>(a[2 * i], a[2 * i + 1], lane & 2);       // lane ^ 2
#pragma unroll
    for (int i = 0; i < 2; ++i) c[i] = (lane & 4 ? b[2 * i + 1] : b[2 * i]) + __shfl_xor(lane & 4 ? b[2 * i] : b[2 * i + 1], 4);
    const float d = with_lane<0x128>(c[0], c[1], lane & 8);                                     // lane ^ 8
    return d + __shfl_xor(d, 16);
}

template <typename T, int D, int N, bool BIAS>
__global__ __launch_bounds__(64 * N, 2) void attn_short_grad_kernel(AttnArgs a, int k_items_at) {
    using S = Short<T, D, N>;
    constexpr int DT = D >= 32 ? D / 32 : 1, ST = D / 16, NT = 64 * N, kRows = S::kRows, kBytes = S::kBytes, kDsRow = S::kDsRow;
    extern __shared__ char smem[];
    char* qt = smem;                                        // rows of q and dout, later dS
    char* gt = smem + kBytes;
    float* ds = reinterpret_cast<float*>(smem);
    char* kt = smem + S::kFirst;
    float* rowref = reinterpret_cast<float*>(kt + kBytes);
    float* rowdelta = rowref + kRows;                       // [N][kRows]: of a wavefront's keys
    float* sums = rowdelta + N * kRows;                     // [2][2 kRows]: by key - row + kRows, per half of the rows
    float* bias = sums + 4 * kRows;
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
        for (int i = tid; i < (nq + nk) * kChunks; i += NT) {
            const int row = i / kChunks;
            char* q = reinterpret_cast<char*>(const_cast<T*>(row < nq ? row_ptr<T>(a.dq, (int64_t)qi.q0 + row, head) : row_ptr<T>(a.dk, (int64_t)ki.k0 + row - nq, head)));
            *reinterpret_cast<u32x4_a*>(q + i % kChunks * 16) = u32x4_a{0, 0, 0, 0};
            if (row >= nq)
                *reinterpret_cast<u32x4_a*>(reinterpret_cast<char*>(const_cast<T*>(row_ptr<T>(a.dv, (int64_t)ki.k0 + row - nq, head))) + i % kChunks * 16) = u32x4_a{0, 0, 0, 0};
        }
        if constexpr (BIAS)
            for (int i = tid; i < words; i += NT) part[i] = 0.f;
        return;
    }
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;
    const int mine = 32 * w + (lane & 31);                  // this lane's key, and its row
    const int keyc = min(mine, nk - 1), rowc = min(mine, nq - 1);
    const int64_t qr = (int64_t)qi.q0 + rowc;

    Stage<T, D, kRows, NT> sq(a.q.row * (int)sizeof(T), tid), sg(a.dout.row * (int)sizeof(T), tid), sk(a.k.row * (int)sizeof(T), tid);
    sq.load(reinterpret_cast<const char*>(row_ptr<T>(a.q, qi.q0, head)), nq, tid);
    sg.load(reinterpret_cast<const char*>(row_ptr<T>(a.dout, qi.q0, head)), nq, tid);
    sk.load(reinterpret_cast<const char*>(row_ptr<T>(a.k, ki.k0, head)), nk, tid);
    const char* vrow = reinterpret_cast<const char*>(row_ptr<T>(a.v, (int64_t)ki.k0 + keyc, head));
    const float lse = a.lse[(int64_t)head * a.q_rows + qr];
    V8<T> kf[ST], vf[ST];
#pragma unroll
    for (int s = 0; s < ST; ++s) vf[s] = global_frag<T>(vrow, s, h);
    bool hides = false;                                     // the table hides a bucket of this head
    if constexpr (BIAS) {
        hides = table_hides<T>(a.bias, a.heads, head, 1);
        load_bias<T>(bias, a.bias, 1.f / a.scale, a.heads, head, tid, NT);
    }
    sq.store(qt, tid);
    sg.store(gt, tid);
    sk.store(kt, tid);
    unsigned odd = 0;
    const bool whole = Sight(win, pos0, pos0 + nq - 1).all(0, nk);
    if (hides | !whole) odd = sq.not_finite() | sg.not_finite() | sk.not_finite();
    if (h == 0) rowref[mine] = mine < nq ? lse_log2(lse) * (kLseLast<T> ? -1.f : -1.f / c) : kMinusInf;      // rows behind the last weigh nothing
    bool redo = __syncthreads_or((int)odd);
    auto delta_of_out = [&] { return dot_rows<T, D>(row_ptr<T>(a.dout, qr, head), row_ptr<T>(a.out, qr, head)); };
    if (redo) {
        if (h == 0 && mine < nq) a.delta[(int64_t)head * a.q_rows + qr] = delta_of_out();
        __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < ST; ++s) kf[s] = Tile<T, D>::row_frag(kt, mine, s, h);

    // pairs of this lane's key and the 32 rows from 32 u on that do not count become zero: row c is seen if far - c <= right and
    // far - c >= -left, or the key is one of the first
    auto hide_rows = [&](f32x16_a& x, int u) {
        const int r0 = 32 * u + 4 * h, far = mine - (pos0 + r0);      // to the row of register 0
        const int lo = far - win.right, hi = min(mine < win.sinks ? kFar : far + win.left, nq - 1 - r0);
        const int m = mine < nk ? max(hi - lo + 1, 0) : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = (unsigned)(reg_row(r) - lo) < (unsigned)m ? x[r] : 0.f;
    };
    auto bias_of = [&](int u) { return bias + bias_at(mine - (pos0 + 32 * u + 4 * h) - kBiasPad, reach) + kBiasPad; };     // minus the row
    // the same for the pairs that the table hides
    auto hide_buckets = [&](f32x16_a& x, int u) {
        const float* b = bias_of(u);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = b[-reg_row(r)] == kMinusInf ? 0.f : x[r];
    };
    // sums of a row's pairs over this wavefront's keys, by row
    auto row_sums = [&](const f32x16_a& x, int u) {
        const float sum = Lift<T>::off_first(lane_sums(x, lane));
        if ((lane & 16) == 0) rowdelta[kRows * w + 32 * u + reg_row(lane & 15) + 4 * h] = sum;
    };
    f32x16_a dk[DT], dv[DT], weight[N], d_s[N];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        f32x16_a &s = weight[u], &p = d_s[u];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = p[r] = 0.f;
        const int r0 = 32 * u;
        const Sight sight(win, pos0 + r0, pos0 + min(r0 + 31, nq - 1));
        {
            const bool full = (32 * w + 32 <= nk) & (r0 + 32 <= nq) & sight.all(32 * w, 32);
            const V4<float>* less = reinterpret_cast<const V4<float>*>(rowref + r0 + 4 * h);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const V4<float> y = kLseLast<T> ? V4<float>{0.f, 0.f, 0.f, 0.f} : less[2 * x];
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * x + e] = y[e];
            }
            if constexpr (BIAS) {
                const float* b = bias_of(u);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] += b[-reg_row(r)];
            }
            row_products<T, D, 4>(s, p, qt, gt, r0, kf, vf, lane);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                V4<float> y{0.f, 0.f, 0.f, 0.f};
                if constexpr (kLseLast<T>) y = less[2 * x];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * x + e;
                    s[r] = __builtin_amdgcn_exp2f(kLseLast<T> ? fmaf(s[r], c, y[e]) : Lift<T>::kOn ? fmaf(s[r], c, Lift<T>().log2()) : s[r] * c);
                    p[r] *= s[r];
                }
            }
            if (!full) {
                hide_rows(s, u);
                hide_rows(p, u);
            }
            Cols<T, D> cols;
            cols.read(gt, r0, lane);
            cols.product(dv, s);
        }
        row_sums(p, u);
    }
    __syncthreads();
    // A row's delta is not finite (a value row of NaN, say): what it is multiplied with is zero where pairs are hidden, but the product
    // is not.  All wavefronts read the same sums, so they agree
    const int of_row = min(lane, kRows - 1);
    const bool lost = __ballot(!finite(rowdelta[of_row] + (N == 2 ? rowdelta[kRows + of_row] : 0.f)));
    if constexpr (BIAS) {
        if (lost & hides) {
            __syncthreads();
#pragma unroll
            for (int u = 0; u < N; ++u) {
                hide_buckets(weight[u], u);
                hide_buckets(d_s[u], u);
                row_sums(d_s[u], u);
            }
            if (!redo && h == 0 && mine < nq) a.delta[(int64_t)head * a.q_rows + qr] = delta_of_out();
            redo = true;
            __syncthreads();
        }
    }
    Lift<T> lift_k, lift_q;      // of dk and dq; weight and d_s hold what is lifted by the first power, and so do dv's sums
#pragma unroll
    for (int u = 0; u < N; ++u)
        if ((32 * w < nk) & (32 * u < nq)) {
            const V4<float>* del = reinterpret_cast<const V4<float>*>(rowdelta + 32 * u + 4 * h);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                V4<float> y = del[2 * x];
                if constexpr (N == 2) y += del[2 * x + kRows / 4];
#pragma unroll
                for (int e = 0; e < 4; ++e) d_s[u][4 * x + e] = fmaf(-y[e], weight[u][4 * x + e], d_s[u][4 * x + e]);
            }
            if (lost) hide_rows(d_s[u], u);
            if (lost & hides) hide_buckets(d_s[u], u);
            Cols<T, D> cols;
            cols.read(qt, 32 * u, lane);
            f32x16_a x = d_s[u];
            if (Lift<T>::kOn && lift_k.moved) Lift<T>::down(x, Lift<T>::kFirst - lift_k.e);
            lift_k.settle(x, dk);
            cols.product(dk, x);
        }
    float dk_by = lift_k.off(a.scale), dv_by = Lift<T>::off_first(1.f);
    if (redo) {
        float x[16 * DT], y[16 * DT];
        dkv_by_pairs<T, D, DT, BIAS>(kernel_args(), x, y, k_items_at, item, head, keyc, h);
        take<DT>(dk, x);
        take<DT>(dv, y);
        dk_by = a.scale, dv_by = 1.f;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < N; ++u)
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
                for (int e = 0; e < 4; ++e) y[e] = (T)(dk[d][4 * x + e] * dk_by), z[e] = (T)(dv[d][4 * x + e] * dv_by);
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
    for (int u = 0; u < N; ++u)
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
            if (Lift<T>::kOn && lift_q.moved) Lift<T>::down(s, Lift<T>::kFirst - lift_q.e);
            lift_q.settle(s, dq);
            cols.product(dq, s);
        }
    if constexpr (BIAS) {
        // Half of the threads for half of the rows each; thread l adds up keys l, l + 1, ... of rows 0, 1, ..., which wrap
        // to the diagonal kRows below
        const int l = tid & (kRows - 1), half = tid / kRows;
        float up[2] = {0.f, 0.f}, down[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kRows / 2; ++i) {
            const int row = kRows / 2 * half + i;
            const float x = ds[row * kDsRow + ((row + l) & (kRows - 1))];
            const bool wraps = row + l >= kRows;
            up[i & 1] += wraps ? 0.f : x;
            down[i & 1] += wraps ? x : 0.f;
        }
        sums[2 * kRows * half + l] = down[0] + down[1];
        sums[2 * kRows * half + kRows + l] = up[0] + up[1];
    }
    float dq_by = lift_q.off(a.scale);
    if (redo) {
        float t[16 * DT];
        dq_by_pairs<T, D, DT, BIAS>(kernel_args(), t, false, item, head, rowc, pos0 + rowc, bias, h);
        take<DT>(dq, t);
        dq_by = a.scale;
    }
    if (mine < nq) {
        T* o = const_cast<T*>(row_ptr<T>(a.dq, (int64_t)qi.q0 + mine, head));
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < (D >= 32 ? 4 : 2); ++x) {
                V4<T> y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (T)(dq[d][4 * x + e] * dq_by);
                *reinterpret_cast<V4<T>*>(o + 32 * d + 8 * x + 4 * h) = y;
            }
    }
    if constexpr (BIAS) {
        __syncthreads();
        for (int i = tid; i < words; i += NT) {
            // the word's distance from a row's position to a key, as an index of `sums`; the outer words take what lies beyond
            const int t = i - reach - kFarPad + pos0 + kRows, last = 2 * kRows - 1;
            const int from = i == 0 ? 0 : max(t, 0), to = i == words - 1 ? last : min(t, last);
            float x = 0.f;
            for (int k = from; k <= to; ++k) x += sums[k] + sums[2 * kRows + k];
            part[i] = Lift<T>::off_first(x);
        }
    }
}

template <typename T, int D, int N>
hipError_t short_grad_waves(const AttnArgs& a, int k_items_at, hipStream_t s) {
    const int64_t blocks = (int64_t)a.n_items * a.heads;
    return a.bias.table ? start(attn_short_grad_kernel<T, D, N, true>, blocks, 64 * N, Short<T, D, N>::lds(a), s, a, k_items_at)
                        : start(attn_short_grad_kernel<T, D, N, false>, blocks, 64 * N, Short<T, D, N>::lds(a), s, a, k_items_at);
}
template <typename T, int D>
hipError_t short_grad_dim(const AttnArgs& a, int waves, int k_items_at, hipStream_t s) {
    if constexpr (D <= kShortDim) return waves == 1 ? short_grad_waves<T, D, 1>(a, k_items_at, s) : short_grad_waves<T, D, 2>(a, k_items_at, s);
    else return hipErrorInvalidValue;
}

}  // namespace
}  // namespace dptm
