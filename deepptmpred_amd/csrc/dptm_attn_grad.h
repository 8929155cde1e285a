// Attention over packed sequences: backward kernels.
//
//   P_ij = exp(s_ij - lse_i);  delta_i = dout_i . out_i;  dP_ij = dout_i . v_j;  dS = P (dP - delta)
//   dq_i = scale sum_j dS_ij k_j;  dk_j = scale sum_i dS_ij q_i;  dv_j = sum_i P_ij dout_i;  dtable[b] = sum dS over bucket b
//
// Two kernels, one that owns queries (dq, delta, bias) and one that owns keys (dk, dv, over the query heads that share
// the key head).  Scores are computed twice, 7 products for the 5 a single kernel would need, and in turn nothing is added
// through atomics: results do not depend on the order in which workgroups run.  P and dS are rounded to the tensors' type for
// the products that sum them; everything else stays in 32 bits.
#pragma once
#include "dptm_attn_kernels.h"

namespace dptm {
namespace {

// weight of an empty row (lse = -inf) is 0 everywhere: its reference is +inf
__device__ __forceinline__ float lse_log2(float lse) { return lse == kMinusInf ? __builtin_inff() : lse * kLog2e; }

template <typename T, int D, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64) void attn_dq_kernel(AttnArgs a) {
    constexpr int kBK = kKeysPerTile<T>, NK = kBK / 32, DT = D >= 32 ? D / 32 : 1, ST = D / 16;
    constexpr int kBytes = kBK * D * (int)sizeof(T);
    extern __shared__ char smem[];
    float* bias = reinterpret_cast<float*>(smem + 4 * kBytes);
    const int reach = a.bias.reach, nb = a.bias.n_buckets;
    float* bins = bias + (BIAS ? ((2 * reach + 1 + 3) & ~3) : 0);                        // [NW][nb][64]
    unsigned char* bucket = reinterpret_cast<unsigned char*>(bins + (BIAS ? NW * nb * 64 : 0));
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int head = id / a.n_items, item = id - head * a.n_items;
    const QItem it = reinterpret_cast<const QItem*>(a.plan + a.items_at)[item];
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;

    const int first = min(32 * w, it.nq - 1), last = min(32 * w + 31, it.nq - 1);
    const bool active = 32 * w < it.nq;
    const int row = 32 * w + (lane & 31), rowc = min(row, it.nq - 1);
    const Rows rw = rows_of(a, it.q0, it.pos0, first, last, rowc);
    const int64_t qr = (int64_t)it.q0 + rowc;
    const char* qrow = static_cast<const char*>(a.q.p) + (qr * a.q.row + (int64_t)head * a.q.head) * (int)sizeof(T);
    const char* grow = static_cast<const char*>(a.dout.p) + (qr * a.dout.row + (int64_t)head * a.dout.head) * (int)sizeof(T);
    const char* orow = static_cast<const char*>(a.out.p) + (qr * a.out.row + (int64_t)head * a.out.head) * (int)sizeof(T);
    V8<T> q[ST], g[ST];
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        q[s] = global_frag<T>(qrow, s, h);
        g[s] = global_frag<T>(grow, s, h);
        const V8<T> o = global_frag<T>(orow, s, h);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)g[s][e], (float)o[e], delta);
    }
    delta = half_sum(delta);
    const float lse = a.lse[(int64_t)head * a.q_rows + qr];
    const float ref = lse_log2(lse);
    if (h == 0 && row < it.nq) a.delta[(int64_t)head * a.q_rows + qr] = delta;

    const int hk = head / a.group;
    const char* kbase = static_cast<const char*>(a.k.p) + ((int64_t)it.k0 * a.k.row + (int64_t)hk * a.k.head) * (int)sizeof(T);
    const char* vbase = static_cast<const char*>(a.v.p) + ((int64_t)it.k0 * a.v.row + (int64_t)hk * a.v.head) * (int)sizeof(T);
    const int64_t kstep = a.k.row * (int)sizeof(T), vstep = a.v.row * (int)sizeof(T);
    const int ns = (it.sink_end + kBK - 1) / kBK, n = ns + (it.ke - it.kb + kBK - 1) / kBK;
    Stage<T, D, kBK, NW * 64> sk, sv;
    auto fetch = [&](int t) {
        const int j0 = t < ns ? t * kBK : it.kb + (t - ns) * kBK, j1 = t < ns ? it.sink_end : it.ke;
        sk.load(kbase + j0 * kstep, kstep, j1 - j0, tid);
        sv.load(vbase + j0 * vstep, vstep, j1 - j0, tid);
    };
    f32x16_a acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    if (n > 0) fetch(0);
    if constexpr (BIAS) {
        load_bias<T>(bias, a.bias, a.heads, head, tid, NW * 64);
        for (int i = tid; i < NW * nb * 64; i += NW * 64) bins[i] = 0.f;
        for (int i = tid; i < 2 * reach + 1; i += NW * 64) bucket[i] = (unsigned char)min(max(a.bias.buckets[i], 0), nb - 1);
    }
    if (n > 0) {
        sk.store(smem, tid);
        sv.store(smem + 2 * kBytes, tid);
    }
    __syncthreads();
    for (int t = 0; t < n; ++t) {
        if (t + 1 < n) fetch(t + 1);
        const char* kt = smem + (t & 1) * kBytes;
        const char* vt = smem + (2 + (t & 1)) * kBytes;
        const int j0 = t < ns ? t * kBK : it.kb + (t - ns) * kBK, j1 = min(j0 + kBK, t < ns ? it.sink_end : it.ke);
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int a0 = j0 + 32 * k, a1 = min(a0 + 32, j1);
            if (active && a0 < j1 && !none_visible(win, rw.pmin, rw.pmax, a0, a1)) {
                const bool full = a1 - a0 == 32 && all_visible(win, rw.pmin, rw.pmax, a0, a1);
                f32x16_a s, p;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = p[r] = 0.f;
#pragma unroll
                for (int st = 0; st < ST; ++st) {
                    mma(s, Tile<T, D>::row_frag(kt, 32 * k + (lane & 31), st, h), q[st]);
                    mma(p, Tile<T, D>::row_frag(vt, 32 * k + (lane & 31), st, h), g[st]);
                }
                const bool one = a0 - rw.pmax >= reach || a0 + 31 - rw.pmin <= -reach;   // one bucket for the whole tile
                const int far0 = a0 + 4 * h - rw.pos + reach;
                if constexpr (BIAS) {
                    if (one) {
                        const float b = bias[a0 - rw.pmax >= reach ? 2 * reach : 0];
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, b);
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, bias[min(max(far0 + reg_row(r), 0), 2 * reach)]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float x = BIAS ? s[r] - ref : fmaf(s[r], c, -ref);
                    s[r] = __builtin_amdgcn_exp2f(x) * (p[r] - delta);
                }
                if (!full) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = a0 + 4 * h + reg_row(r);
                        s[r] = ((j < j1) & visible(win, j - rw.pos, j)) ? s[r] : 0.f;
                    }
                }
                if constexpr (BIAS) {
                    // a lane adds into a column of its own: no two threads meet, and the order is the program's
                    float* mine = bins + w * nb * 64 + lane;
                    const bool counts = row < it.nq;
                    if (one) {
                        float sum = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) sum += s[r];
                        const int b = bucket[a0 - rw.pmax >= reach ? 2 * reach : 0];
                        if (counts) __hip_atomic_fetch_add(mine + b * 64, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    } else if (counts) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int b = bucket[min(max(far0 + reg_row(r), 0), 2 * reach)];
                            __hip_atomic_fetch_add(mine + b * 64, s[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const V8<T> b = pack8<T>(s, x);
                    if (full) {
#pragma unroll
                        for (int d = 0; d < DT; ++d) mma(acc[d], Tile<T, D>::col_frag(kt, 32 * k + 16 * x, d, lane), b);
                    } else {
#pragma unroll
                        for (int d = 0; d < DT; ++d) mma_guarded<T>(acc[d], Tile<T, D>::col_frag(kt, 32 * k + 16 * x, d, lane), b);
                    }
                }
            }
        }
        if (t + 1 < n) {
            sk.store(smem + ((t + 1) & 1) * kBytes, tid);
            sv.store(smem + (2 + ((t + 1) & 1)) * kBytes, tid);
        }
        __syncthreads();
    }
    if (row < it.nq) {
        T* o = static_cast<T*>(a.dq.p) + ((int64_t)it.q0 + row) * a.dq.row + (int64_t)head * a.dq.head;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < (D >= 32 ? 4 : 2); ++x) {
                V4<T> y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (T)(acc[d][4 * x + e] * a.scale);
                *reinterpret_cast<V4<T>*>(o + 32 * d + 8 * x + 4 * h) = y;
            }
    }
    if constexpr (BIAS) {
        for (int b = w; b < nb; b += NW) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) sum += bins[(i * nb + b) * 64 + lane];
#pragma unroll
            for (int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k);
            if (lane == 0) a.part_bias[((int64_t)head * a.n_items + item) * nb + b] = sum;
        }
    }
}

// dtable[b][head] from the tiles' sums, in 64 bits and in a fixed order
template <typename T>
__global__ __launch_bounds__(256) void attn_dtable_kernel(const float* part, int n_items, int nb, int heads, T* dtable) {
    __shared__ double sums[256];
    const int b = blockIdx.x % nb, head = blockIdx.x / nb;
    double x = 0.0;
    for (int i = threadIdx.x; i < n_items; i += 256) x += (double)part[((int64_t)head * n_items + i) * nb + b];
    sums[threadIdx.x] = x;
    __syncthreads();
    for (int k = 128; k; k >>= 1) {
        if ((int)threadIdx.x < k) sums[threadIdx.x] += sums[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) dtable[(int64_t)b * heads + head] = (T)(float)sums[0];
}

template <typename T, int D, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64) void attn_dkv_kernel(AttnArgs a) {
    constexpr int kBQ = kKeysPerTile<T>, NQ = kBQ / 32, DT = D >= 32 ? D / 32 : 1, ST = D / 16;
    constexpr int kBytes = kBQ * D * (int)sizeof(T);
    extern __shared__ char smem[];
    float* rowref = reinterpret_cast<float*>(smem + 4 * kBytes);   // [2][kBQ] each
    float* rowdelta = rowref + 2 * kBQ;
    int* rowpos = reinterpret_cast<int*>(rowdelta + 2 * kBQ);
    float* bias = reinterpret_cast<float*>(rowpos + 2 * kBQ);
    const int reach = a.bias.reach;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = a.heads / a.group;
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int hk = id / a.n_items;
    const KItem it = reinterpret_cast<const KItem*>(a.plan + a.items_at)[id - hk * a.n_items];
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;
    const bool active = 32 * w < it.nk;
    const int key = 32 * w + (lane & 31), keyc = min(key, it.nk - 1);
    const int j = it.j0 + key;                                      // index in the sequence
    const int j0 = it.j0 + 32 * w, j1 = it.j0 + min(32 * w + 32, it.nk);
    const int64_t kr = (int64_t)it.k0 + keyc;
    const char* krow = static_cast<const char*>(a.k.p) + (kr * a.k.row + (int64_t)hk * a.k.head) * (int)sizeof(T);
    const char* vrow = static_cast<const char*>(a.v.p) + (kr * a.v.row + (int64_t)hk * a.v.head) * (int)sizeof(T);
    V8<T> kf[ST], vf[ST];
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        kf[s] = global_frag<T>(krow, s, h);
        vf[s] = global_frag<T>(vrow, s, h);
    }
    f32x16_a dk[DT], dv[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;

    const int nt = (it.qe - it.qb + kBQ - 1) / kBQ, n = nt * a.group;
    const int64_t qstep = a.q.row * (int)sizeof(T), gstep = a.dout.row * (int)sizeof(T);
    Stage<T, D, kBQ, NW * 64> sq, sg;
    float nref = 0.f, ndelta = 0.f;
    int npos = 0;
    auto fetch = [&](int step) {
        const int g = step / nt, head = hk * a.group + g, i0 = it.qb + (step - g * nt) * kBQ;
        const int64_t r0 = (int64_t)it.q0 + i0;
        const int valid = it.qe - i0;
        sq.load(static_cast<const char*>(a.q.p) + (r0 * a.q.row + (int64_t)head * a.q.head) * (int)sizeof(T), qstep, valid, tid);
        sg.load(static_cast<const char*>(a.dout.p) + (r0 * a.dout.row + (int64_t)head * a.dout.head) * (int)sizeof(T), gstep, valid, tid);
        if (tid < kBQ) {
            nref = __builtin_inff();
            ndelta = 0.f;
            npos = 0;
            if (tid < valid) {
                const int64_t at = (int64_t)head * a.q_rows + r0 + tid;
                nref = lse_log2(a.lse[at]);
                ndelta = a.delta[at];
                npos = row_position(a.plan, a.has_pos, a.pos_at, it.pos0 + i0, it.q0 + i0, tid);
            }
        }
    };
    auto put = [&](int buf) {
        sq.store(smem + buf * kBytes, tid);
        sg.store(smem + (2 + buf) * kBytes, tid);
        if (tid < kBQ) {
            rowref[buf * kBQ + tid] = nref;
            rowdelta[buf * kBQ + tid] = ndelta;
            rowpos[buf * kBQ + tid] = npos;
        }
    };
    if (n > 0) {
        fetch(0);
        if constexpr (BIAS) load_bias<T>(bias, a.bias, a.heads, hk * a.group, tid, NW * 64);
        put(0);
    }
    __syncthreads();
    for (int t = 0; t < n; ++t) {
        if (t + 1 < n) fetch(t + 1);
        const int buf = t & 1, g = t / nt, i0 = it.qb + (t - g * nt) * kBQ;
        const char* qt = smem + buf * kBytes;
        const char* gt = smem + (2 + buf) * kBytes;
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            const int r0 = i0 + 32 * u;
            if (!active || r0 >= it.qe) continue;
            int pmin, pmax;
            if (a.has_pos) {
                pmin = a.plan[a.tiles_at + 2 * (it.tile0 + (r0 >> 5))];
                pmax = a.plan[a.tiles_at + 2 * (it.tile0 + (r0 >> 5)) + 1];
            } else {
                pmin = it.pos0 + r0;
                pmax = it.pos0 + min(r0 + 31, it.nseq - 1);
            }
            if (none_visible(win, pmin, pmax, j0, j1)) continue;
            // rows behind the last weigh nothing by their reference of +inf
            const bool full = all_visible(win, pmin, pmax, j0, j0 + 32);
            f32x16_a s, p;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = p[r] = 0.f;
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                mma(s, Tile<T, D>::row_frag(qt, 32 * u + (lane & 31), st, h), kf[st]);
                mma(p, Tile<T, D>::row_frag(gt, 32 * u + (lane & 31), st, h), vf[st]);
            }
            const float* ref = rowref + buf * kBQ + 32 * u + 4 * h;
            const float* del = rowdelta + buf * kBQ + 32 * u + 4 * h;
            const int* pos = rowpos + buf * kBQ + 32 * u + 4 * h;
            if constexpr (BIAS) {
                if (j0 - pmax >= reach || j0 + 31 - pmin <= -reach) {
                    const float b = bias[j0 - pmax >= reach ? 2 * reach : 0];
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, b);
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, bias[min(max(j - pos[reg_row(r)] + reach, 0), 2 * reach)]);
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = BIAS ? s[r] - ref[reg_row(r)] : fmaf(s[r], c, -ref[reg_row(r)]);
                s[r] = __builtin_amdgcn_exp2f(x);
            }
            if (!full) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = visible(win, j - pos[reg_row(r)], j) ? s[r] : 0.f;
            }
            // dS of a hidden pair is 0 whatever its operands hold
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = full ? s[r] * (p[r] - del[reg_row(r)]) : s[r] == 0.f ? 0.f : s[r] * (p[r] - del[reg_row(r)]);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const V8<T> pw = pack8<T>(s, x), ps = pack8<T>(p, x);
                if (full) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        mma(dv[d], Tile<T, D>::col_frag(gt, 32 * u + 16 * x, d, lane), pw);
                        mma(dk[d], Tile<T, D>::col_frag(qt, 32 * u + 16 * x, d, lane), ps);
                    }
                } else {
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        mma_guarded<T>(dv[d], Tile<T, D>::col_frag(gt, 32 * u + 16 * x, d, lane), pw);
                        mma_guarded<T>(dk[d], Tile<T, D>::col_frag(qt, 32 * u + 16 * x, d, lane), ps);
                    }
                }
            }
        }
        if (t + 1 < n) {
            put((t + 1) & 1);
            if constexpr (BIAS) {
                if ((t + 1) / nt != g) {     // the next query head's bias, once nobody reads this one's
                    __syncthreads();
                    load_bias<T>(bias, a.bias, a.heads, hk * a.group + g + 1, tid, NW * 64);
                }
            }
        }
        __syncthreads();
    }
    if (key < it.nk) {
        if (it.slot < 0) {
            T* ok = static_cast<T*>(a.dk.p) + ((int64_t)it.k0 + key) * a.dk.row + (int64_t)hk * a.dk.head;
            T* ov = static_cast<T*>(a.dv.p) + ((int64_t)it.k0 + key) * a.dv.row + (int64_t)hk * a.dv.head;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int x = 0; x < (D >= 32 ? 4 : 2); ++x) {
                    V4<T> y, z;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = (T)(dk[d][4 * x + e] * a.scale);
                        z[e] = (T)dv[d][4 * x + e];
                    }
                    *reinterpret_cast<V4<T>*>(ok + 32 * d + 8 * x + 4 * h) = y;
                    *reinterpret_cast<V4<T>*>(ov + 32 * d + 8 * x + 4 * h) = z;
                }
        } else {
            float* ok = a.part_o + (((int64_t)it.slot * kvh + hk) * 2 * (NW * 32) + key) * D;
            float* ov = ok + (int64_t)NW * 32 * D;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int x = 0; x < (D >= 32 ? 4 : 2); ++x) {
                    V4<float> y, z;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = dk[d][4 * x + e] * a.scale;
                        z[e] = dv[d][4 * x + e];
                    }
                    *reinterpret_cast<V4<float>*>(ok + 32 * d + 8 * x + 4 * h) = y;
                    *reinterpret_cast<V4<float>*>(ov + 32 * d + 8 * x + 4 * h) = z;
                }
        }
    }
}

// dk, dv of a tile of keys from the parts of several workgroups (grid.y: keys and values)
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(AttnArgs a, int n_join, int join_at, int tile_keys) {
    const int kvh = a.heads / a.group;
    const int hk = blockIdx.x / n_join;
    const Join jn = reinterpret_cast<const Join*>(a.plan + join_at)[blockIdx.x - hk * n_join];
    const Strided& to = blockIdx.y ? a.dv : a.dk;
    for (int i = threadIdx.x; i < jn.n * (D / 4); i += 256) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        V4<float> x{0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < jn.slots; ++k)
            x += *reinterpret_cast<const V4<float>*>(a.part_o + ((((int64_t)(jn.slot0 + k) * kvh + hk) * 2 + blockIdx.y) * tile_keys + r) * D + d);
        V4<T> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
        *reinterpret_cast<V4<T>*>(static_cast<T*>(to.p) + ((int64_t)jn.row0 + r) * to.row + (int64_t)hk * to.head + d) = y;
    }
}

template <typename T, int D>
hipError_t dq_dim(const AttnArgs& a, int waves, hipStream_t s) {
    const int64_t blocks = (int64_t)a.n_items * a.heads;
    size_t lds = 4 * kKeysPerTile<T> * D * sizeof(T);
    if (a.bias.table) lds += bias_floats(a) * 4 + (size_t)waves * a.bias.n_buckets * 64 * 4 + bias_floats(a);
    if (waves == 2)
        return a.bias.table ? start(attn_dq_kernel<T, D, 2, true>, blocks, 128, lds, s, a) : start(attn_dq_kernel<T, D, 2, false>, blocks, 128, lds, s, a);
    return a.bias.table ? start(attn_dq_kernel<T, D, 4, true>, blocks, 256, lds, s, a) : start(attn_dq_kernel<T, D, 4, false>, blocks, 256, lds, s, a);
}

template <typename T, int D>
hipError_t dkv_dim(const AttnArgs& a, int waves, hipStream_t s) {
    const int64_t blocks = (int64_t)a.n_items * (a.heads / a.group);
    const size_t lds = 4 * kKeysPerTile<T> * D * sizeof(T) + 6 * kKeysPerTile<T> * 4 + bias_floats(a) * 4;
    if (waves == 2)
        return a.bias.table ? start(attn_dkv_kernel<T, D, 2, true>, blocks, 128, lds, s, a) : start(attn_dkv_kernel<T, D, 2, false>, blocks, 128, lds, s, a);
    return a.bias.table ? start(attn_dkv_kernel<T, D, 4, true>, blocks, 256, lds, s, a) : start(attn_dkv_kernel<T, D, 4, false>, blocks, 256, lds, s, a);
}

template <typename T, int D>
hipError_t dkv_join_dim(const AttnArgs& a, int n_join, int join_at, int tile_keys, hipStream_t s) {
    if (n_join == 0) return hipSuccess;
    hipLaunchKernelGGL((attn_dkv_join_kernel<T, D>), dim3((unsigned)n_join * (a.heads / a.group), 2), dim3(256), 0, s, a, n_join, join_at, tile_keys);
    return hipGetLastError();
}

}  // namespace
}  // namespace dptm

#define DPTM_ATTN_BY_DIM(F, ...)                 \
    dim == 16 ? F<E, 16>(__VA_ARGS__)            \
    : dim == 32 ? F<E, 32>(__VA_ARGS__)          \
    : dim == 64 ? F<E, 64>(__VA_ARGS__)          \
                : F<E, 128>(__VA_ARGS__)

// the launchers of one element type
#define DPTM_ATTN_DEFINE(NAME, TYPE)                                                                                       \
    namespace dptm {                                                                                                       \
    using E = TYPE;                                                                                                        \
    hipError_t attn_forward_##NAME(const AttnArgs& a, int dim, int mode, hipStream_t s) { return DPTM_ATTN_BY_DIM(forward_dim, a, mode, s); } \
    hipError_t attn_dq_##NAME(const AttnArgs& a, int dim, int waves, hipStream_t s) { return DPTM_ATTN_BY_DIM(dq_dim, a, waves, s); }         \
    hipError_t attn_dkv_##NAME(const AttnArgs& a, int dim, int waves, hipStream_t s) { return DPTM_ATTN_BY_DIM(dkv_dim, a, waves, s); }       \
    hipError_t attn_join_##NAME(const AttnArgs& a, int dim, int n, int at, hipStream_t s) {                                \
        const int64_t blocks = (int64_t)n * a.heads;                                                                       \
        return dim == 16 ? start(attn_join_kernel<E, 16>, blocks, 256, 0, s, a, n, at)                                     \
             : dim == 32 ? start(attn_join_kernel<E, 32>, blocks, 256, 0, s, a, n, at)                                     \
             : dim == 64 ? start(attn_join_kernel<E, 64>, blocks, 256, 0, s, a, n, at)                                     \
                         : start(attn_join_kernel<E, 128>, blocks, 256, 0, s, a, n, at);                                   \
    }                                                                                                                      \
    hipError_t attn_dkv_join_##NAME(const AttnArgs& a, int dim, int n, int at, int keys, hipStream_t s) {                  \
        return DPTM_ATTN_BY_DIM(dkv_join_dim, a, n, at, keys, s);                                                          \
    }                                                                                                                      \
    hipError_t attn_dtable_##NAME(const AttnArgs& a, int n_items, hipStream_t s) {                                         \
        return start(attn_dtable_kernel<E>, (int64_t)a.bias.n_buckets * a.heads, 256, 0, s, (const float*)a.part_bias, n_items, \
                     a.bias.n_buckets, a.heads, static_cast<E*>(a.dtable));                                                \
    }                                                                                                                      \
    }
