// Attention over packed sequences: forward kernels (dptm_attn_device.h explains the layout the products use).
//
//   visible(i, j): 0 <= j < keys of i's sequence, j - p_i <= right, and (j - p_i >= -left or j < sinks)
//   s_ij = scale q_i . k_j + bias(j - p_i);  lse_i = log sum_j exp s_ij;  out_i = sum_j exp(s_ij - lse_i) v_j
//
// One pass over the keys with a running maximum m and sum l per query, in units of log2 and in 32 bits.  The weights are
// rounded to the tensors' type for the second product (fp32: not at all), l sums them unrounded.
//
// What bounds them.  Long sequences in 16 bits: vector and matrix instructions, which do not overlap here, and at heads of 128 the LDS
// reads between them.  Heads of 64 with a bias: the vector unit works on a tile's softmax for twice as long as its matrix instructions take
// (46 and 23 % of the busy cycles); heads of 128: 33 and 41 %, a quarter is waiting.  32,768 rows, 20 heads, bf16: 550 TFLOP/s in
// sequences of 1,024, 710 of 4,096; heads of 128 700 and 810; a large plain product reaches 1,228.  Few queries over long keys: memory (64 new tokens over caches of up to
// 4,099 keys, 8 key heads of 128: 839 MB in 164 us, 5.1 TB/s; a large copy reaches 5.05).  One short protein: the way of a tile
// from memory through two products and a join in LDS (482 rows, 20 heads: 12.8 us for 5 MB).
#pragma once
#include "dptm_attn_device.h"

namespace dptm {
namespace {

// float16 weights are kept 2^10 times larger than exp2(s - m): a weight of 2^-24 of the largest is then still a normal number.
// The maximum that the weights refer to is only moved when a score passes it by more than 2^kLazy, so the largest
// weight is 2^(kShift + kLazy): 2^14 in float16, whose largest number is 65504.
template <typename T> constexpr float kShift = sizeof(T) == 2 && Elem<T>::kExp == 0x7c00 ? 10.f : 0.f;
template <> constexpr float kShift<float> = 0.f;
template <typename T> constexpr float kUnshift = kShift<T> > 0.f ? 0x1p-10f : 1.f;    // before the logarithm: lse keeps its last bits
constexpr float kLazy = 4.f;
// A maximum leaves NaN out, the sum does not: a row that meets NaN has lse NaN, and -inf stays with rows that see nothing.
template <typename T>
__device__ __forceinline__ float lse_of(float m, float l) {
    return l == 0.f ? kMinusInf : (m + __log2f(l * kUnshift<T>)) * kLn2;
}

// keys of a tile in LDS: 64 where the registers that carry the next tile allow it
template <typename T, int D> constexpr int kKeysPerTile = sizeof(T) == 2 ? 64 : 32;

// Wavefronts a SIMD that the compiler is held to; more registers than that allows cost more than they give.  Three in the
// forward kernel with 16-bit heads up to 64 (168 registers; two, with up to 198, took 171 us of a 48-protein batch where three took
// 131, now 127); two otherwise; one for fp32 heads of 128, whose operands alone take 128 registers (two: 5.4 ms and a spill
// of 64 registers, one: 3.6 ms without, 32,768 rows in sequences of 1,024).
template <typename T, int D> constexpr int kForwardWaves = sizeof(T) * D >= 512 ? 1 : sizeof(T) == 2 && D <= 64 ? 3 : 2;

// what a wavefront knows of its 32 queries
struct Rows {
    int pos, pmin, pmax;
};

// scores of 32 NK keys -> weights (in place), running maximum and sum, accumulators moved to the new maximum.  Per element
// a multiply-add, an exp2, half a three-way maximum, an add and half a conversion: with head dimension 64 that is
// half as long again as the element's matrix instructions, which is why nothing else is done per element.
template <typename T, int NK, int DT>
__device__ __forceinline__ void softmax_step(f32x16_a (&s)[NK], const float (&more)[NK], f32x16_a (&acc)[DT], float& m, float& l, float c, const Rows& w,
                                             const Window& win, int j0, int j1, bool full, int h) {
    if (!full) {
#pragma unroll
        for (int k = 0; k < NK; ++k) hide(s[k], lane_mask(win, w.pos, j0 + 32 * k + 4 * h, j1), kMinusInf);
    }
    float mx = kMinusInf;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        float x = s[k][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) x = fmaxf(x, s[k][r]);
        mx = fmaxf(mx, fmaf(x, c, more[k]));
    }
    mx = half_max(mx);
    const bool grow = mx > m + kLazy || (m == kMinusInf && mx > m);
    if (__ballot(grow)) {
        const float alpha = grow ? __builtin_amdgcn_exp2f(m - mx) : 1.f;
        m = grow ? mx : m;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    }
    const float ref = (m == kMinusInf ? 0.f : m) - kShift<T>;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        const float less = more[k] - ref;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[k][r], c, less));
            s[k][r] = p;
            sum += p;
        }
    }
    l += sum;
}

template <typename T>
__device__ __forceinline__ const T* row_ptr(const Strided& t, int64_t row, int head) {
    return static_cast<const T*>(t.p) + row * t.row + (int64_t)head * t.head;
}
template <typename T, int D>
__device__ __forceinline__ float dot_rows(const T* a, const T* b) {
    float s = 0.f;
    for (int d = 0; d < D; d += 8) {
        const V8<T> x = *reinterpret_cast<const V8<T>*>(a + d), y = *reinterpret_cast<const V8<T>*>(b + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf((float)x[e], (float)y[e], s);
    }
    return s;
}
// column of the head that accumulator register r of tile d holds in half-wave h (head dimension 16: half a tile)
template <int D> __device__ __forceinline__ int reg_col(int d, int r, int h) { return (32 * d + reg_row(r) + 4 * h) & (D - 1); }

// The functions that do rows over are out of line and keep their sums in private memory: such rows are rare, and the kernels
// that call them shall not pay with registers.  They are handed the kernel's arguments where the launch put them, because a
// reference to the kernel's copy would move that into private memory too.
__device__ __forceinline__ const AttnArgs& kernel_args() {
    return *(const AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
}
#define DPTM_COLD __device__ __attribute__((noinline))

// The rows of a wavefront once more, pair by pair: hidden pairs do not enter.  For tiles `first`, `first + every`, ... of `keys` keys.
template <typename T, int D, int DT, bool BIAS>
DPTM_COLD void forward_by_pairs(const AttnArgs& a, float* acc, float* ml, int item, int head, int row, int pos, int first, int every, int keys,
                                const float* bias, int h) {
    const QItem& it = reinterpret_cast<const QItem*>(a.plan + a.items_at)[item];
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;
    const int hk = head / a.group;
    const T* q = row_ptr<T>(a.q, (int64_t)it.q0 + row, head);
    const int ns = (it.sink_end + keys - 1) / keys, n = ns + (it.ke - it.kb + keys - 1) / keys;
#pragma unroll 1
    for (int i = 0; i < 16 * DT; ++i) acc[i] = 0.f;
    float m = kMinusInf, l = 0.f;
    for (int t = first; t < n; t += every) {
        const int j0 = t < ns ? t * keys : it.kb + (t - ns) * keys, j1 = min(j0 + keys, t < ns ? it.sink_end : it.ke);
        for (int j = j0; j < j1; ++j) {
            float s = dot_rows<T, D>(q, row_ptr<T>(a.k, (int64_t)it.k0 + j, hk));
            const float b = BIAS ? bias[bias_at(j - pos, a.bias.reach)] : 0.f;
            s = (s + b) * c;
            s = visible(win, j - pos, j) & (b != kMinusInf) ? s : kMinusInf;
            const float top = fmaxf(m, s), f = m == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(m - top);
            const float p = s == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(s - top + kShift<T>);
            m = top;
            l = l * f + p;
            const T* v = row_ptr<T>(a.v, (int64_t)it.k0 + j, hk);
#pragma unroll 1
            for (int i = 0; i < 16 * DT; ++i)
                acc[i] = acc[i] * f + (s == kMinusInf ? 0.f : (float)(T)p * (float)v[reg_col<D>(i >> 4, i & 15, h)]);
        }
    }
    ml[0] = m;
    ml[1] = h ? 0.f : l;      // the caller adds the halves
}
// accumulators <-> what the functions above leave
template <int DT>
__device__ __forceinline__ void take(f32x16_a (&acc)[DT], const float* from) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = from[16 * d + r];
}

__device__ __forceinline__ Rows rows_of(const AttnArgs& a, int q0, int pos0, int first, int last, int mine) {
    Rows w;
    if (a.has_pos) {
        w.pos = a.plan[a.pos_at + q0 + mine];
        w.pmin = wave_min(w.pos);
        w.pmax = wave_max(w.pos);
    } else {
        w.pos = pos0 + mine;
        w.pmin = pos0 + first;
        w.pmax = pos0 + last;
    }
    return w;
}

// ---- many queries: NW wavefronts of 32 queries share tiles of keys and values in LDS (two buffers, one barrier a tile)
template <typename T, int D, int NW, bool BIAS>
__global__ __launch_bounds__(NW * 64, (kForwardWaves<T, D>)) void attn_fwd_wide_kernel(AttnArgs a) {
    constexpr int kBK = kKeysPerTile<T, D>, NK = kBK / 32, DT = D >= 32 ? D / 32 : 1, ST = D / 16;
    constexpr int kBytes = kBK * D * (int)sizeof(T);
    extern __shared__ char smem[];
    float* bias = reinterpret_cast<float*>(smem + 4 * kBytes);
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int head = a.by_sequence ? id % a.heads : id / a.n_items, item = a.by_sequence ? id / a.heads : id - head * a.n_items;
    const QItem it = reinterpret_cast<const QItem*>(a.plan + a.items_at)[item];
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;

    const int first = min(32 * w, it.nq - 1), last = min(32 * w + 31, it.nq - 1);
    const bool active = 32 * w < it.nq;
    const int row = 32 * w + (lane & 31), rowc = min(row, it.nq - 1);
    const Rows rw = rows_of(a, it.q0, it.pos0, first, last, rowc);
    const char* qrow = static_cast<const char*>(a.q.p) + (((int64_t)it.q0 + rowc) * a.q.row + (int64_t)head * a.q.head) * (int)sizeof(T);
    V8<T> q[ST];
#pragma unroll
    for (int s = 0; s < ST; ++s) q[s] = global_frag<T>(qrow, s, h);

    const int hk = head / a.group;
    const char* kbase = static_cast<const char*>(a.k.p) + ((int64_t)it.k0 * a.k.row + (int64_t)hk * a.k.head) * (int)sizeof(T);
    const char* vbase = static_cast<const char*>(a.v.p) + ((int64_t)it.k0 * a.v.row + (int64_t)hk * a.v.head) * (int)sizeof(T);
    const int64_t kstep = a.k.row * (int)sizeof(T), vstep = a.v.row * (int)sizeof(T);
    Stage<T, D, kBK, NW * 64> sk(kstep, tid), sv(vstep, tid);
    auto fetch = [&](const KeyWalk& at) {
        sk.load(kbase + at.j0 * kstep, at.end - at.j0, tid);
        sv.load(vbase + at.j0 * vstep, at.end - at.j0, tid);
    };
    const Sight sight(win, rw.pmin, rw.pmax), whole(win, it.pos0, it.pos0 + it.nq - 1);
    const int above_from = rw.pmax + a.bias.reach, below_to = rw.pmin - a.bias.reach - 31;     // 32 keys of one bias
    unsigned odd = 0;
    auto put = [&](const KeyWalk& at, int buf) {
        sk.store(smem + buf * kBytes, tid);
        sv.store(smem + (2 + buf) * kBytes, tid);
        if (a.has_pos | !whole.all(at.j0, kBK)) odd |= sv.not_finite();
    };
    f32x16_a acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    float m = kMinusInf, l = 0.f;

    KeyWalk at(it);
    if (at.more()) fetch(at);
    if constexpr (BIAS) load_bias<T>(bias, a.bias, 1.f / a.scale, a.heads, head, tid, NW * 64);
    if (at.more()) put(at, 0);
    __syncthreads();
    for (int buf = 0; at.more(); buf ^= 1) {
        const KeyWalk after = at.next(kBK);
        if (after.more()) fetch(after);
        const char* kt = smem + buf * kBytes;
        const char* vt = smem + (2 + buf) * kBytes;
        if (active & !sight.none(at.j0, kBK)) {
            const bool full = (at.j0 + kBK <= at.end) & sight.all(at.j0, kBK);
            f32x16_a s[NK];
            float more[NK];      // one bias for the 32 keys, where they are far
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const V8<T> first_k = Tile<T, D>::row_frag(kt, 32 * k + (lane & 31), 0, h);
                const int k0 = at.j0 + 32 * k;
                const bool above = k0 >= above_from;
                more[k] = 0.f;
                if (BIAS && !(above | (k0 <= below_to))) {
                    init_bias(s[k], bias, a.bias.reach, k0 + 4 * h - rw.pos);
                    mma(s[k], first_k, q[0]);
                } else {
                    if constexpr (BIAS) more[k] = c * bias[above ? 2 * a.bias.reach + kBiasPad : 0];
                    f32x16_a zero;
#pragma unroll
                    for (int r = 0; r < 16; ++r) zero[r] = 0.f;
                    s[k] = zero;
                    mma(s[k], first_k, q[0]);
                }
#pragma unroll
                for (int st = 1; st < ST; ++st) mma(s[k], Tile<T, D>::row_frag(kt, 32 * k + (lane & 31), st, h), q[st]);
            }
            softmax_step<T, NK, DT>(s, more, acc, m, l, c, rw, win, at.j0, at.end, full, h);
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                Cols<T, D> v;
                v.read(vt, 32 * k, lane);
                v.product(acc, s[k]);
            }
        }
        if (after.more()) put(after, buf ^ 1);
        __syncthreads();
        at = after;
    }
    bool redo = __syncthreads_or((int)odd);
    if constexpr (BIAS)
        if (!redo && __ballot(!finite(l + sum_of_all(acc)))) redo = table_hides<T>(a.bias, a.heads, head, 1);
    if (redo) {
        float t[16 * DT], ml[2];
        forward_by_pairs<T, D, DT, BIAS>(kernel_args(), t, ml, item, head, rowc, rw.pos, 0, 1, kBK, bias, h);
        take<DT>(acc, t);
        m = ml[0], l = ml[1];
    }
    if (row < it.nq) {
        l = half_sum(l);
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        T* o = static_cast<T*>(a.out.p) + ((int64_t)it.q0 + row) * a.out.row + (int64_t)head * a.out.head;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < (D >= 32 ? 4 : 2); ++g) {
                V4<T> x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (T)(acc[d][4 * g + e] * inv);
                *reinterpret_cast<V4<T>*>(o + 32 * d + 8 * g + 4 * h) = x;
            }
        if (h == 0) a.lse[(int64_t)head * a.q_rows + it.q0 + row] = lse_of<T>(m, l);
    }
}

// ---- few queries: the four wavefronts of a workgroup (eight: 17.1 us instead of 12.6 for the 482 rows of one protein, 20 heads)
// ---- hold the SAME 32 rows and take every fourth tile of 32 keys, and a long range of keys is cut over workgroups as well (53
// ---- rows over 34,003 keys, 20 heads: 42 us, and 6 to join); the parts meet in LDS, those of several workgroups in attn_join_kernel.
// ---- A row is a query of one of `pack` heads that share their keys, so that keys are read once for all of them
template <typename T, int D, bool BIAS>
__global__ __launch_bounds__(256, sizeof(T) * D >= 512 ? 1 : 2) void attn_fwd_split_kernel(AttnArgs a) {
    constexpr int NW = 4, DT = D >= 32 ? D / 32 : 1, ST = D / 16, kPad = D + 4;
    constexpr int kBytes = 32 * D * (int)sizeof(T);
    extern __shared__ char smem[];
    float* ml = reinterpret_cast<float*>(smem);                 // [NW][32][2]
    float* bias = ml + NW * 64;                                 // [pack][bias_room]
    const int room = BIAS ? bias_room(a.bias.reach) : 0;
    char* tiles = smem + (NW * 64 + a.pack * room) * 4;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int pack = a.pack, head0 = id / a.n_items * pack;
    const QItem it = reinterpret_cast<const QItem*>(a.plan + a.items_at)[id - id / a.n_items * a.n_items];
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;
    const int rows = it.nq * pack, row = min(lane & 31, rows - 1), query = row / pack, head = head0 + row - query * pack;
    const Rows rw = rows_of(a, it.q0, it.pos0, 0, it.nq - 1, query);
    const T* qrow = row_ptr<T>(a.q, (int64_t)it.q0 + query, head);
    V8<T> q[ST];
#pragma unroll
    for (int s = 0; s < ST; ++s) q[s] = global_frag<T>(reinterpret_cast<const char*>(qrow), s, h);
    const int hk = head0 / a.group;
    const char* kbase = reinterpret_cast<const char*>(row_ptr<T>(a.k, it.k0, hk));
    const char* vbase = reinterpret_cast<const char*>(row_ptr<T>(a.v, it.k0, hk));
    const int64_t kstep = a.k.row * (int)sizeof(T), vstep = a.v.row * (int)sizeof(T);
    const int ns = (it.sink_end + 31) / 32, n = ns + (it.ke - it.kb + 31) / 32;
    V8<T> kf[ST];
    Stage<T, D, 32, 64> sv(vstep, lane);
    char* vt = tiles + w * kBytes;
    auto fetch = [&](int t) {
        const int j0 = t < ns ? t * 32 : it.kb + (t - ns) * 32, j1 = t < ns ? it.sink_end : it.ke;
        const char* krow = kbase + min(j0 + (lane & 31), j1 - 1) * kstep;
#pragma unroll
        for (int s = 0; s < ST; ++s) kf[s] = global_frag<T>(krow, s, h);
        sv.load(vbase + j0 * vstep, j1 - j0, lane);
    };
    if (w < n) fetch(w);
    if constexpr (BIAS) {
        for (int p = 0; p < pack; ++p) load_bias<T>(bias + p * room, a.bias, 1.f / a.scale, a.heads, head0 + p, tid, NW * 64);
        __syncthreads();
        bias += (head - head0) * room;
    }
    f32x16_a acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    float m = kMinusInf, l = 0.f;
    const Sight sight(win, rw.pmin, rw.pmax);
    unsigned odd = 0;
    for (int t = w; t < n; t += NW) {
        const int j0 = t < ns ? t * 32 : it.kb + (t - ns) * 32, j1 = min(j0 + 32, t < ns ? it.sink_end : it.ke);
        f32x16_a s[1];
        float more[1] = {0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
        if constexpr (BIAS) {
            const bool above = j0 >= rw.pmax + a.bias.reach;
            if (above | (j0 + 31 <= rw.pmin - a.bias.reach)) more[0] = c * bias[above ? 2 * a.bias.reach + kBiasPad : 0];
            else init_bias(s[0], bias, a.bias.reach, j0 + 4 * h - rw.pos);
        }
#pragma unroll
        for (int st = 0; st < ST; ++st) mma(s[0], kf[st], q[st]);
        const bool full = (j1 - j0 == 32) & sight.all(j0, 32);
        __builtin_amdgcn_wave_barrier();
        sv.store(vt, lane);
        if (!full) odd |= sv.not_finite();
        if (t + NW < n) fetch(t + NW);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        softmax_step<T, 1, DT>(s, more, acc, m, l, c, rw, win, j0, j1, full, h);
        Cols<T, D> v;
        v.read(vt, 0, lane);
        v.product(acc, s[0]);
    }
    bool redo = __ballot(odd != 0);
    if constexpr (BIAS)
        if (!redo && __ballot(!finite(l + sum_of_all(acc)))) redo = table_hides<T>(a.bias, a.heads, head0, pack);
    if (redo) {
        float t[16 * DT], x[2];
        forward_by_pairs<T, D, DT, BIAS>(kernel_args(), t, x, id - id / a.n_items * a.n_items, head, query, rw.pos, w, NW, 32, bias, h);
        take<DT>(acc, t);
        m = x[0], l = x[1];
    }
    l = half_sum(l);
    if (h == 0) {
        ml[(w * 32 + lane) * 2] = m;
        ml[(w * 32 + lane) * 2 + 1] = l;
    }
    __syncthreads();
    float top = kMinusInf;
#pragma unroll
    for (int i = 0; i < NW; ++i) top = fmaxf(top, ml[(i * 32 + (lane & 31)) * 2]);
    const float f = m == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(m - top);
    float* o = reinterpret_cast<float*>(tiles);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < (D >= 32 ? 4 : 2); ++g) {
            V4<float> x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = acc[d][4 * g + e] * f;
            *reinterpret_cast<V4<float>*>(o + (w * 32 + (lane & 31)) * kPad + 32 * d + 8 * g + 4 * h) = x;
        }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += NW * 64) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4, qi = r / pack, hd = head0 + r - qi * pack;
        float t = kMinusInf, sum = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) t = fmaxf(t, ml[(k * 32 + r) * 2]);
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const float mk = ml[(k * 32 + r) * 2];
            sum += ml[(k * 32 + r) * 2 + 1] * (mk == kMinusInf ? 1.f : __builtin_amdgcn_exp2f(mk - t));     // without a score 0, or NaN
        }
        V4<float> x = *reinterpret_cast<V4<float>*>(o + r * kPad + d);
#pragma unroll
        for (int k = 1; k < NW; ++k) x += *reinterpret_cast<V4<float>*>(o + (k * 32 + r) * kPad + d);
        if (it.slot < 0) {
            const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
            V4<T> y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)(x[e] * inv);
            *reinterpret_cast<V4<T>*>(const_cast<T*>(row_ptr<T>(a.out, (int64_t)it.q0 + qi, hd)) + d) = y;
            if (d == 0) a.lse[(int64_t)hd * a.q_rows + it.q0 + qi] = lse_of<T>(t, sum);
        } else {
            const int64_t at = ((int64_t)it.slot * (a.heads / pack) + head0 / pack) * 32 + r;
            *reinterpret_cast<V4<float>*>(a.part_o + at * D + d) = x;
            if (d == 0) {
                a.part_ml[at * 2] = t;
                a.part_ml[at * 2 + 1] = sum;
            }
        }
    }
}

// the parts of one tile of rows from several workgroups: eight rows a block, one thread for four columns
constexpr int kJoinRows = 8;
template <typename T, int D>
__global__ __launch_bounds__(kJoinRows * (D / 4)) void attn_join_kernel(AttnArgs a, int n_join, int join_at) {
    const int hp = blockIdx.x / n_join, pack = a.pack, heads = a.heads / pack;
    const Join jn = reinterpret_cast<const Join*>(a.plan + join_at)[blockIdx.x - hp * n_join];
    const int r = blockIdx.y * kJoinRows + threadIdx.x / (D / 4), d = (threadIdx.x % (D / 4)) * 4;
    if (r >= jn.n * pack) return;
    const int64_t first = ((int64_t)jn.slot0 * heads + hp) * 32 + r, next = (int64_t)heads * 32;
    float m = kMinusInf, l = 0.f;
#pragma unroll 8
    for (int k = 0; k < jn.slots; ++k) m = fmaxf(m, a.part_ml[(first + k * next) * 2]);
    V4<float> x{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < jn.slots; ++k) {
        const int64_t at = first + k * next;
        const float mk = a.part_ml[at * 2], lk = a.part_ml[at * 2 + 1];
        const V4<float> xk = *reinterpret_cast<const V4<float>*>(a.part_o + at * D + d);
        const float f = mk == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(mk - m);
        l += mk == kMinusInf ? lk : lk * f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += xk[e] * f;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    V4<T> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(x[e] * inv);
    const int qi = r / pack, head = hp * pack + r - qi * pack;
    *reinterpret_cast<V4<T>*>(const_cast<T*>(row_ptr<T>(a.out, (int64_t)jn.row0 + qi, head)) + d) = y;
    if (d == 0) a.lse[(int64_t)head * a.q_rows + jn.row0 + qi] = lse_of<T>(m, l);
}

template <typename K>
hipError_t lds_room(K kernel, size_t bytes) {
    return bytes > 65536 ? hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)
                         : hipSuccess;
}
template <typename K, typename... A>
hipError_t start(K kernel, int64_t blocks, int threads, size_t lds, hipStream_t s, const A&... args) {
    if (blocks == 0) return hipSuccess;
    const hipError_t e = lds_room(kernel, lds);
    if (e != hipSuccess) return e;
    return launch(kernel, dim3((unsigned)blocks), dim3(threads), lds, s, args...);
}
inline size_t bias_floats(const AttnArgs& a) { return a.bias.table ? (size_t)bias_room(a.bias.reach) : 0; }

template <typename T, int D>
hipError_t forward_dim(const AttnArgs& a, int mode, hipStream_t s) {
    const int64_t blocks = (int64_t)a.n_items * a.heads;
    if (mode == kSplitKeys) {
        const size_t v = 4 * 32 * D * sizeof(T), o = 4 * 32 * (D + 4) * 4;
        const size_t lds = (4 * 64 + a.pack * bias_floats(a)) * 4 + (v > o ? v : o);
        return a.bias.table ? start(attn_fwd_split_kernel<T, D, true>, blocks / a.pack, 256, lds, s, a)
                            : start(attn_fwd_split_kernel<T, D, false>, blocks / a.pack, 256, lds, s, a);
    }
    const size_t lds = 4 * kKeysPerTile<T, D> * D * sizeof(T) + bias_floats(a) * 4;
    if (mode == kWide64)
        return a.bias.table ? start(attn_fwd_wide_kernel<T, D, 2, true>, blocks, 128, lds, s, a)
                            : start(attn_fwd_wide_kernel<T, D, 2, false>, blocks, 128, lds, s, a);
    return a.bias.table ? start(attn_fwd_wide_kernel<T, D, 4, true>, blocks, 256, lds, s, a)
                        : start(attn_fwd_wide_kernel<T, D, 4, false>, blocks, 256, lds, s, a);
}

template <typename T, int D>
hipError_t join_dim(const AttnArgs& a, int n_join, int join_at, hipStream_t s) {
    if (n_join == 0) return hipSuccess;
    return launch(attn_join_kernel<T, D>, dim3((unsigned)(n_join * (a.heads / a.pack)), 32 / kJoinRows), dim3(kJoinRows * (D / 4)), 0, s, a, n_join,
                  join_at);
}

}  // namespace
}  // namespace dptm
