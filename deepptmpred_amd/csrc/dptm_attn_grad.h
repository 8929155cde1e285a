// Attention over packed sequences: backward kernels.
//
//   P_ij = exp(s_ij - lse_i);  delta_i = dout_i . out_i;  dP_ij = dout_i . v_j;  dS = P (dP - delta)
//   dq_i = scale sum_j dS_ij k_j;  dk_j = scale sum_i dS_ij q_i;  dv_j = sum_i P_ij dout_i;  dtable[b] = sum dS over bucket b
//
// Two kernels, one that owns queries (dq, delta) and one that owns keys (dk, dv over the query heads that share the key head,
// and the bias gradient).  Scores are computed twice, 7 products for the 5 a single kernel would need, and in turn nothing is
// added through atomics: results do not depend on the order in which workgroups run.  P and dS are rounded to the tensors'
// type for the products that sum them; everything else stays in 32 bits.
//
// The kernel that owns queries is bound by instructions, vector and matrix together (51 and 29 % of the busy cycles; they do not run side
// by side on this hardware).  The one that owns keys is not: 33 and 19 %, the rest of its time its two wavefronts a SIMD wait, for the most
// part for fragments from LDS, of which it reads twice as many to a vector instruction.  48 proteins of up to 1,024 residues, 20 heads of 64,
// with a bias: 172 us for dq, 286 for dk, dv and the bias.  32,768 rows in sequences of 4,096 without one: 605 TFLOP/s by the five products
// that count, heads of 128 510.
#pragma once
#include "dptm_attn_kernels.h"

namespace dptm {
namespace {

// weight of an empty row (lse = -inf) is 0 everywhere: its reference is +inf
__device__ __forceinline__ float lse_log2(float lse) { return lse == kMinusInf ? __builtin_inff() : lse * kLog2e; }

// float16 holds 2^-24 to 65504, and the pairs' P and dS of a long row or a small gradient lie below that (8,192 keys, dout of size
// 1e-3: dq and dk 7 times as far off as rounding them makes them, of size 1e-4 10 % of their size; gradients of some 1e5 were infinite).
// For float16 alone both are therefore formed larger by a power of two, which is part of the exponent that exp2 takes.
//   dk, dv and short sequences: 2^13.  What rounding a pair then takes away is 2^-38 at least, and the results' own rounding 2^-25.  A
// lane -- a key -- that meets a |dS| above 2^14 so lifted goes on with a smaller power of two, and its sums move along: eight three-way
// maxima a tile (16,001 rows, window of 512, with the bias: 162 -> 172 us, or 192 from memory).
//   dq: a lane is a query, and its dout says how large dS is, so that no tile has to be looked at: the power takes the largest |dout| to
// 2^4.  P of 2^-20 still keeps all bits then; rows whose sums come out infinite (|dP - delta| of thousands of times |dout|, values in the
// hundreds or thousands) are done over pair by pair.
template <typename T> struct Lift {
    static constexpr bool kOn = sizeof(T) == 2 && Elem<T>::kExp == 0x7c00;
    static constexpr int kFirst = kOn ? 13 : 0;
    int e = kFirst;
    bool moved = false;       // some lane of the wavefront has another power than 2^kFirst
    __device__ __forceinline__ float log2() const { return kOn ? (float)e : 0.f; }
    __device__ __forceinline__ float off(float x) const { return kOn ? __builtin_amdgcn_ldexpf(x, -e) : x; }
    // of what was lifted by 2^kFirst
    __device__ __forceinline__ static float off_first(float x) { return kOn ? x * 0x1p-13f : x; }
    __device__ __forceinline__ static void down(f32x16_a& x, int by) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_ldexpf(x[r], -by);
    }
    // w is lifted by 2^e and about to be summed, sums are what earlier ones have been summed in
    template <int DT, typename... Sums>
    __device__ __forceinline__ void settle(f32x16_a& w, f32x16_a (&acc)[DT], Sums&... sums) {
        if constexpr (kOn) {
            float top = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r += 2) top = fmaxf(fmaxf(fabsf(w[r]), fabsf(w[r + 1])), top);
            top = half_max(top);
            if (__ballot(top > 0x1p14f)) {
                const int by = top > 0x1p14f ? min((int)(__float_as_uint(top) >> 23) - 127 - 12, e + 100) : 0;
                e -= by;
                moved = true;
                down(w, by);
                auto all = [&](f32x16_a (&x)[DT]) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) down(x[d], by);
                };
                all(acc);
                (all(sums), ...);
            }
        }
    }
};

// A wavefront's rows of dq once more, pair by pair (see Stage::not_finite); `mend`: the row's delta takes on the sum of its dS.
template <typename T, int D, int DT, bool BIAS>
DPTM_COLD void dq_by_pairs(const AttnArgs& a, float* acc, bool mend, int item, int head, int row, int pos, const float* bias, int h) {
    const QItem& it = reinterpret_cast<const QItem*>(a.plan + a.items_at)[item];
    const Window win{a.left, a.right, a.sinks};
    const int hk = head / a.group;
    const int64_t qr = (int64_t)it.q0 + row;
    const T* q = row_ptr<T>(a.q, qr, head);
    const T* g = row_ptr<T>(a.dout, qr, head);
    const float ref = lse_log2(a.lse[(int64_t)head * a.q_rows + qr]), delta = a.delta[(int64_t)head * a.q_rows + qr];
#pragma unroll 1
    for (int i = 0; i < 16 * DT; ++i) acc[i] = 0.f;
    float sum = 0.f;
    for (int j = 0; j < it.ke; ++j) {
        if (j >= it.sink_end && j < it.kb) continue;
        const T* k = row_ptr<T>(a.k, (int64_t)it.k0 + j, hk);
        float s = dot_rows<T, D>(q, k);
        const float b = BIAS ? bias[bias_at(j - pos, a.bias.reach)] : 0.f;
        s += b;
        const float ds = __builtin_amdgcn_exp2f(fmaf(s, a.scale * kLog2e, -ref)) * (dot_rows<T, D>(g, row_ptr<T>(a.v, (int64_t)it.k0 + j, hk)) - delta);
        const bool see = visible(win, j - pos, j) & (b != kMinusInf);
        sum += see ? ds : 0.f;
#pragma unroll 1
        for (int i = 0; i < 16 * DT; ++i) acc[i] += see ? ds * (float)k[reg_col<D>(i >> 4, i & 15, h)] : 0.f;
    }
    if (mend) a.delta[(int64_t)head * a.q_rows + qr] = delta + sum;
}

// rows of a tile in LDS: fewer than in the forward pass where a wavefront's own operands and sums take the registers
template <typename T, int D> constexpr int kRowsPerTile = sizeof(T) == 2 && D <= 64 ? 64 : 32;
// 16-bit heads of 64 in the kernel that owns queries: its registers fit three wavefronts a SIMD (tiles of 32 keys, fragments asked
// for one product ahead, columns read after the scores), 32 proteins of 1,024 residues, 20 heads, bf16: 485 -> 406 us, with a bias
// 524 -> 450.  With the bins of a list of positions (POS) they do not: two wavefronts, tiles of 64 keys, reads as early as they go.
template <typename T, int D, bool POS> constexpr bool kDqThree = sizeof(T) == 2 && D == 64 && !POS;
template <typename T, int D, bool POS> constexpr int kDqKeys = kDqThree<T, D, POS> ? 32 : kRowsPerTile<T, D>;
template <typename T, int D, bool POS> constexpr int kDqWaves = D * sizeof(T) <= 64 || kDqThree<T, D, POS> ? 3 : D * sizeof(T) >= 512 ? 1 : 2;

// Bias gradient, in the kernel that owns keys.  Far tiles (one bucket) are summed in a register.  In a near one the rows
// stand at consecutive positions, so that equal distances are the diagonals of its 32 x 32 dS: it goes to LDS with zeros between its
// rows, lane l adds diagonal l up (32 reads at a fixed stride) and keeps the sum by distance; what distances share a bucket is
// left to attn_dtable_kernel.  With every element added into its bucket by LDS atomics instead 48 proteins took 540 us more.  The kernel
// that owns queries would do it some 30 us faster, but before delta is known to its last bits (see below): the gradient
// of a bucket was off by up to 1.65 times what rounding it gives, and here is not by more.
// Rows at positions from a list (POS) have no diagonals.  There it is the kernel that owns queries; each lane adds into a column
// of its own per bucket, and no order but the program's enters either.  In the 16-bit types that kernel goes over the keys twice, the
// first time for what its delta lacks: without it the gradient of a bucket was off by up to 4.8 times what rounding it gives (1,500
// rows and keys), with it 1.0 times.  The backward pass of 8 x 1,022 listed rows, 20 heads of 64, bf16, takes 598 us for 522.
constexpr int kShearRow = 68;                   // 32 values and 36 zeros: 17 chunks of 16 bytes, so that rows start on different banks
constexpr int kShear = 32 * kShearRow + 32;   // floats, 32 zeros in front
__host__ __device__ inline int bin_floats(int waves, int n_buckets, int reach) { return waves * n_buckets * 64 + (bias_room(reach) + 3) / 4; }
__host__ __device__ inline int diagonal_room(int reach) { return (2 * reach + 1 + 2 * kFarPad + 3) & ~3; }
__host__ __device__ inline int diagonal_floats(int waves, int reach) { return waves * (kShear + diagonal_room(reach)); }

// Rounding in the 16-bit types.  delta is taken from `out`, which was rounded, and dS is rounded for the product with K: with rounding
// the result, three errors of the same size, and dq and dk of rows that see few keys were off by 1.5 to 1.7 times what
// rounding the results alone gives.  The first is mended for dk and the bias: a row's dS has to add up to nothing, so what they do
// add up to is what delta lacks, and the kernel leaves the sum of both behind.  For dq it comes too late; there half of what
// rounding dS takes away goes through the product a second time (Cols::product_more_bits), and both gradients stay within 1.43
// times.  Together they cost 4 to 10 % of this kernel (without a bias 406 -> 443 us); the whole of what the rounding takes
// away would cost another 6 to 10 %.
template <typename T, int D, int NW, bool BIAS, bool POS>
__global__ __launch_bounds__(NW * 64, (kDqWaves<T, D, POS>)) void attn_dq_kernel(AttnArgs a) {
    constexpr int kBK = kDqKeys<T, D, POS>, NK = kBK / 32, DT = D >= 32 ? D / 32 : 1, ST = D / 16;
    constexpr bool kEarly = D <= 64 && !kDqThree<T, D, POS>;
    constexpr bool kTwice = POS && sizeof(T) == 2;      // the first time for delta alone
    constexpr int kBytes = kBK * D * (int)sizeof(T);
    extern __shared__ char smem[];
    float* bias = reinterpret_cast<float*>(smem + 4 * kBytes);
    const int reach = a.bias.reach, nb = a.bias.n_buckets;
    float* more = bias + (BIAS ? bias_room(reach) : 0);                              // POS: bins of the wavefronts, [nb][64] each
    unsigned char* bucket = reinterpret_cast<unsigned char*>(more + NW * nb * 64);
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    float* bins = more + w * nb * 64;
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
    const T* qrow = row_ptr<T>(a.q, qr, head);
    const T* grow = row_ptr<T>(a.dout, qr, head);
    const T* orow = row_ptr<T>(a.out, qr, head);
    V8<T> q[ST], g[ST];
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        q[s] = global_frag<T>(reinterpret_cast<const char*>(qrow), s, h);
        g[s] = global_frag<T>(reinterpret_cast<const char*>(grow), s, h);
        const V8<T> o = global_frag<T>(reinterpret_cast<const char*>(orow), s, h);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)g[s][e], (float)o[e], delta);
    }
    delta = half_sum(delta);
    // rows behind the last weigh nothing
    const float ref = row < it.nq ? lse_log2(a.lse[(int64_t)head * a.q_rows + qr]) : __builtin_inff();
    if (h == 0 && row < it.nq) a.delta[(int64_t)head * a.q_rows + qr] = delta;

    const int hk = head / a.group;
    const char* kbase = reinterpret_cast<const char*>(row_ptr<T>(a.k, it.k0, hk));
    const char* vbase = reinterpret_cast<const char*>(row_ptr<T>(a.v, it.k0, hk));
    const int64_t kstep = a.k.row * (int)sizeof(T), vstep = a.v.row * (int)sizeof(T);
    Stage<T, D, kBK, NW * 64> sk(kstep, tid), sv(vstep, tid);
    auto fetch = [&](const KeyWalk& at) {
        sk.load(kbase + at.j0 * kstep, at.end - at.j0, tid);
        sv.load(vbase + at.j0 * vstep, at.end - at.j0, tid);
    };
    const Sight sight(win, rw.pmin, rw.pmax), whole(win, it.pos0, it.pos0 + it.nq - 1);
    const int above_from = rw.pmax + reach, below_to = rw.pmin - reach - 31;     // tiles of one bucket
    unsigned odd = 0;
    auto put = [&](const KeyWalk& at, int buf) {
        sk.store(smem + buf * kBytes, tid);
        sv.store(smem + (2 + buf) * kBytes, tid);
        if (a.has_pos | !whole.all(at.j0, kBK)) odd |= sk.not_finite();
    };
    f32x16_a acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    f32x16_a less_delta;                // dP starts from -delta, kept in registers of its own where there are some to spare
    auto keep_delta = [&] {
        if constexpr (D <= 64) {
#pragma unroll
            for (int r = 0; r < 16; ++r) less_delta[r] = -delta;
        }
    };
    keep_delta();
    int lift = 0;
    if constexpr (Lift<T>::kOn) {
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < ST; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf((float)g[s][e]));
        lift = min(4 + 127 - (int)(__float_as_uint(half_max(top)) >> 23), 40);
    }
    auto off = [&](float x) { return Lift<T>::kOn ? __builtin_amdgcn_ldexpf(x, -lift) : x; };
    float over = 0.f;                   // sum of the row's dS, which is what delta lacks
    float below = 0.f, above = 0.f;     // dS of distances up to -reach, from reach on
    KeyWalk walk(it);
    if (walk.more()) fetch(walk);
    if constexpr (BIAS) {
        load_bias<T>(bias, a.bias, 1.f / a.scale, a.heads, head, tid, NW * 64);
        if constexpr (POS) {
            for (int i = tid; i < NW * nb * 64; i += NW * 64) more[i] = 0.f;
            for (int i = tid; i < bias_room(reach); i += NW * 64)
                bucket[i] = (unsigned char)min(max(a.bias.buckets[min(max(i - kBiasPad, 0), 2 * reach)], 0), nb - 1);
        }
    }
#pragma unroll 1
    for (int pass = kTwice ? 0 : 1;; ++pass) {
        if (walk.more()) put(walk, 0);
        __syncthreads();
        for (int buf = 0; walk.more(); buf ^= 1) {
            const KeyWalk after = walk.next(kBK);
            if (after.more()) fetch(after);
            const char* kt = smem + buf * kBytes;
            const char* vt = smem + (2 + buf) * kBytes;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const int a0 = walk.j0 + 32 * k;
                if (active & (a0 < walk.end) & !sight.none(a0, 32)) {
                    const bool full = (a0 + 32 <= walk.end) & sight.all(a0, 32);
                    const bool is_above = a0 >= above_from, is_below = a0 <= below_to;   // one bucket for the tile
                    const bool near = BIAS & !(is_above | is_below);
                    f32x16_a s, p;
                    if constexpr (D <= 64) {
                        p = less_delta;
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) p[r] = -delta;
                    }
                    float less = (float)lift - ref;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = 0.f;
                    if constexpr (BIAS) {
                        if (near) init_bias(s, bias, reach, a0 + 4 * h - rw.pos);
                        else less += c * bias[is_above ? 2 * reach + kBiasPad : 0];
                    }
                    row_products<T, D, kEarly ? 4 : 1>(s, p, kt, vt, 32 * k, q, g, lane);
                    Cols<T, D> cols;
                    if constexpr (kEarly) {
                        cols.read(kt, 32 * k, lane);
                        after_reads<T>();
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, less)) * p[r];
                    if (!full) hide(s, lane_mask(win, rw.pos, a0 + 4 * h, walk.end), 0.f);
                    float sum = 0.f;
                    if (sizeof(T) == 2 || (POS && !near)) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) sum += s[r];
                    }
                    over += sum;
                    if (kTwice && pass == 0) continue;
                    if constexpr (POS) {
                        if (!near) {
                            above += is_above ? sum : 0.f;
                            below += is_above ? 0.f : sum;
                        } else if (row < it.nq) {
                            const int at = bias_at(a0 + 4 * h - rw.pos, reach);
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                __hip_atomic_fetch_add(bins + bucket[at + reg_row(r)] * 64 + lane, off(s[r]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        }
                    }
                    if constexpr (!kEarly) cols.read(kt, 32 * k, lane);
                    cols.product_more_bits(acc, s);
                }
            }
            if (after.more()) put(after, buf ^ 1);
            __syncthreads();
            walk = after;
        }
        over = half_sum(over);
        if (pass) break;
        delta += finite(over) ? off(over) : 0.f;      // a NaN may be a pair's that the table hides
        keep_delta();
        over = 0.f;
        walk = KeyWalk(it);
        if (walk.more()) fetch(walk);
    }
    over = off(over), below = off(below), above = off(above);
    // this lane's row once more, from the lane's number: kept over the loop it would take the place of operands (heads of 128)
    const int mine = 32 * w + (__lane_id() & 31);
    const bool first_half = __lane_id() < 32;
    float* const delta_at = a.delta + (int64_t)head * a.q_rows + it.q0 + mine;
    bool redo = __syncthreads_or((int)odd);
    if constexpr (BIAS || Lift<T>::kOn) {
        const bool lost = !finite(over + sum_of_all(acc));
        if (!redo && __ballot(lost)) {
            if constexpr (Lift<T>::kOn) redo = __ballot(lost & finite(delta));
            if constexpr (BIAS) redo |= table_hides<T>(a.bias, a.heads, head, 1);
        }
    }
    if (__builtin_expect(redo, 0)) {
        float t[16 * DT];
        const int i = min(mine, it.nq - 1);
        dq_by_pairs<T, D, DT, BIAS>(kernel_args(), t, sizeof(T) == 2 && first_half && mine < it.nq, item, head, i,
                                    row_position(a.plan, a.has_pos, a.pos_at, it.pos0, it.q0, i), bias, first_half ? 0 : 1);
        take<DT>(acc, t);
        lift = 0;
    } else if (sizeof(T) == 2 && first_half && mine < it.nq) {
        *delta_at = delta + over;
    }
    if (mine < it.nq) {
        const float by = off(a.scale);
        T* o = const_cast<T*>(row_ptr<T>(a.dq, (int64_t)it.q0 + mine, head)) + (first_half ? 0 : 4);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < (D >= 32 ? 4 : 2); ++x) {
                V4<T> y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (T)(acc[d][4 * x + e] * by);
                *reinterpret_cast<V4<T>*>(o + 32 * d + 8 * x) = y;
            }
    }
    if constexpr (POS) {
#pragma unroll
        for (int k = 32; k; k >>= 1) {
            above += __shfl_xor(above, k);
            below += __shfl_xor(below, k);
        }
        if (lane == 0) {
            bins[bucket[2 * reach + kBiasPad] * 64] += above;
            bins[bucket[0] * 64] += below;
        }
        __syncthreads();
        for (int b = w; b < nb; b += NW) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) sum += more[(i * nb + b) * 64 + lane];
#pragma unroll
            for (int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k);
            if (lane == 0) a.part_bias[((int64_t)head * a.n_items + item) * nb + b] = sum;
        }
    }
}

// The bias gradient from the tiles' sums, in 64 bits and in a fixed order.  First the tiles of a head in up to 64 groups, one
// thread a word, then one block a head adds the groups up and takes the words of each bucket together.
__global__ __launch_bounds__(256) void attn_dtable_groups_kernel(const float* part, double* groups, int n_items, int words, int per) {
    const int head = blockIdx.y, first = blockIdx.x * per, last = min(first + per, n_items);
    for (int i = threadIdx.x; i < words; i += 256) {
        const float* p = part + ((int64_t)head * n_items + first) * words + i;
        double x = 0.0;
#pragma unroll 8
        for (int k = 0; k < last - first; ++k) x += (double)p[(int64_t)k * words];
        groups[((int64_t)head * gridDim.x + blockIdx.x) * words + i] = x;
    }
}
template <typename T>
__global__ __launch_bounds__(1024) void attn_dtable_kernel(AttnArgs a, const double* groups, int n, int words) {
    __shared__ double word[2 * 1024 + 1 + 2 * kFarPad];
    __shared__ int of[2 * 1024 + 1 + 2 * kFarPad];
    __shared__ double part[1024];
    const int nb = a.bias.n_buckets, reach = a.bias.reach, head = blockIdx.x, tid = threadIdx.x;
    for (int i = tid; i < words; i += 1024) {
        const double* p = groups + (int64_t)head * n * words + i;
        double x = 0.0;
#pragma unroll 8
        for (int k = 0; k < n; ++k) x += p[(int64_t)k * words];
        word[i] = x;
        of[i] = a.has_pos ? i : min(max(a.bias.buckets[min(max(i - kFarPad, 0), 2 * reach)], 0), nb - 1);
    }
    __syncthreads();
    const int b = tid & 63, w = tid >> 6;     // the sixteen wavefronts take every sixteenth word
    double x = 0.0;
    for (int i = w; i < words; i += 16) x += of[i] == b ? word[i] : 0.0;
    part[tid] = x;
    __syncthreads();
    if (tid < nb) {
        for (int k = 1; k < 16; ++k) x += part[64 * k + tid];
        const int64_t at = (int64_t)tid * a.heads + head;
        // the pairs of a bucket that is hidden have no gradient, whatever their operands hold; no other bucket's sum holds theirs
        const bool hidden = bias_value((float)static_cast<const T*>(a.bias.table)[at], 1.f) == kMinusInf;
        static_cast<T*>(a.dtable)[at] = (T)(hidden ? 0.f : (float)x);
    }
}
template <typename T>
hipError_t dtable_of(const AttnArgs& a, int n_items, hipStream_t s) {
    const int words = dtable_words(a.has_pos, a.bias.n_buckets, a.bias.reach), n = dtable_groups(n_items);
    if (n) {
        const int per = (n_items + n - 1) / n;
        const hipError_t e = launch(attn_dtable_groups_kernel, dim3(n, a.heads), dim3(256), 0, s, a.part_bias, a.part_groups, n_items, words, per);
        if (e != hipSuccess) return e;
    }
    return launch(attn_dtable_kernel<T>, dim3(a.heads), dim3(1024), 0, s, a, a.part_groups, n, words);
}

// A wavefront's keys of dk and dv once more, pair by pair (see Stage::not_finite).
template <typename T, int D, int DT, bool BIAS>
DPTM_COLD void dkv_by_pairs(const AttnArgs& a, float* dk, float* dv, int items_at, int item, int hk, int key, int h) {
    const KItem& it = reinterpret_cast<const KItem*>(a.plan + items_at)[item];
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;
    const int j = it.j0 + key;
    const T* k = row_ptr<T>(a.k, (int64_t)it.k0 + key, hk);
    const T* v = row_ptr<T>(a.v, (int64_t)it.k0 + key, hk);
#pragma unroll 1
    for (int i = 0; i < 16 * DT; ++i) dk[i] = dv[i] = 0.f;
    for (int head = hk * a.group; head < (hk + 1) * a.group; ++head)
        for (int i = it.qb; i < it.qe; ++i) {
            const int64_t row = (int64_t)it.q0 + i;
            const int pos = row_position(a.plan, a.has_pos, a.pos_at, it.pos0, it.q0, i);
            const T* q = row_ptr<T>(a.q, row, head);
            const T* g = row_ptr<T>(a.dout, row, head);
            float s = dot_rows<T, D>(q, k);
            bool see = visible(win, j - pos, j);
            if constexpr (BIAS) {
                const int at = min(max(a.bias.buckets[min(max(j - pos, -a.bias.reach), a.bias.reach) + a.bias.reach], 0), a.bias.n_buckets - 1);
                const float b = bias_value((float)static_cast<const T*>(a.bias.table)[(int64_t)at * a.heads + head], 1.f / a.scale);
                s += b;
                see &= b != kMinusInf;
            }
            const float p = __builtin_amdgcn_exp2f(s * c - lse_log2(a.lse[(int64_t)head * a.q_rows + row]));
            const float ds = p * (dot_rows<T, D>(g, v) - a.delta[(int64_t)head * a.q_rows + row]);
#pragma unroll 1
            for (int x = 0; x < 16 * DT; ++x) {
                const int col = reg_col<D>(x >> 4, x & 15, h);
                dk[x] += see ? ds * (float)q[col] : 0.f;
                dv[x] += see ? p * (float)g[col] : 0.f;
            }
        }
}

// Heads of 128 of the 16-bit types take two launches, one for dk and one for dv (8 products then, the scores a third time):
// together their operands and sums leave room for one wavefront a SIMD, and the two launches took 2,392 us where the one took
// 3,018 (32,768 rows in sequences of 2,048, 20 heads); the two take 2,160 now.
//
// Tiles of 64 rows with heads of 64: the 32 that one barrier's second half works on are a loop of its own and columns are read
// when they are needed, which keeps the sums of the bias gradient (SUMS) out of scratch: 48 proteins 291 us; unrolled with early
// reads 401, tiles of 32 rows 303.  Without a bias all of these are the same (558 to 563 us, 32 x 1,024 residues).
// fp32 scores start from zero (or the bias) and lse is taken off by the multiply-add in front of the exponential: sums that start
// from -lse / scale round where that is, which made dk of 2,000 keys 1.7 times as far off as it has to be.  The weights of
// the 16-bit types are rounded far above that, and there the start is free.
template <typename T> constexpr bool kLseLast = sizeof(T) == 4;
enum { kBoth, kOnlyDk, kOnlyDv };
template <typename T, int D> constexpr bool kTwoLaunches = sizeof(T) == 2 && D == 128;

template <typename T, int D, int NW, bool BIAS, bool SUMS, int PART>
__global__ __launch_bounds__(NW * 64, D * sizeof(T) <= 128 || PART != kBoth ? 2 : 1) void attn_dkv_kernel(AttnArgs a) {
    constexpr bool DK = PART != kOnlyDv, DV = PART != kOnlyDk;
    constexpr int kBQ = kRowsPerTile<T, D>, NQ = kBQ / 32, DT = D >= 32 ? D / 32 : 1, ST = D / 16;
    constexpr bool kEarly = D < 64;
    constexpr int kGroup = D <= 64 ? 4 : 2;
    constexpr int kBytes = kBQ * D * (int)sizeof(T);
    extern __shared__ char smem[];
    float* rowref = reinterpret_cast<float*>(smem + 4 * kBytes);   // [2][kBQ] each
    float* rowdelta = rowref + 2 * kBQ;
    int* rowpos = reinterpret_cast<int*>(rowdelta + 2 * kBQ);
    float* bias = reinterpret_cast<float*>(rowpos + 2 * kBQ);
    const int reach = a.bias.reach, words = 2 * reach + 1 + 2 * kFarPad, room = diagonal_room(reach);
    float* more = bias + (BIAS ? bias_room(reach) : 0);             // SUMS
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = a.heads / a.group;
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int hk = id / a.n_items, item = id - hk * a.n_items;
    const KItem it = reinterpret_cast<const KItem*>(a.plan + a.items_at)[item];
    float* shear = more + w * kShear;
    float* sums = more + NW * kShear + w * room;                    // by distance, from -reach - kFarPad
    float below = 0.f, above = 0.f;                                 // dS of distances up to -reach, from reach on
    const Window win{a.left, a.right, a.sinks};
    const float c = a.scale * kLog2e;
    const bool active = 32 * w < it.nk;
    const int key = 32 * w + (lane & 31), keyc = min(key, it.nk - 1);
    const int j = it.j0 + key;                                      // index in the sequence
    const int j0 = it.j0 + 32 * w;
    const T* krow = row_ptr<T>(a.k, (int64_t)it.k0 + keyc, hk);
    const T* vrow = row_ptr<T>(a.v, (int64_t)it.k0 + keyc, hk);
    V8<T> kf[ST], vf[ST];
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        kf[s] = global_frag<T>(reinterpret_cast<const char*>(krow), s, h);
        if constexpr (DK) vf[s] = global_frag<T>(reinterpret_cast<const char*>(vrow), s, h);
    }
    f32x16_a dk[DT], dv[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;
    const int nt = (it.qe - it.qb + kBQ - 1) / kBQ;
    const int64_t qstep = a.q.row * (int)sizeof(T), gstep = a.dout.row * (int)sizeof(T);
    Stage<T, D, kBQ, NW * 64> sq(qstep, tid), sg(gstep, tid);
    unsigned odd = 0;
    float nref = 0.f, ndelta = 0.f;
    int npos = 0;
    const float from_lse = kLseLast<T> ? -1.f : -1.f / c;
    Lift<T> lift;
    // the next tile of rows: its addresses move on with it
    const char *qat = nullptr, *gat = nullptr;
    auto fetch = [&](int head, int t) {
        const int i0 = it.qb + t * kBQ;
        const int64_t r0 = (int64_t)it.q0 + i0;
        const int valid = it.qe - i0;
        if (t == 0) {
            qat = reinterpret_cast<const char*>(row_ptr<T>(a.q, r0, head));
            gat = reinterpret_cast<const char*>(row_ptr<T>(a.dout, r0, head));
        }
        sq.load(qat, valid, tid);
        sg.load(gat, valid, tid);
        qat += kBQ * qstep;
        gat += kBQ * gstep;
        if (tid < kBQ) {
            const int64_t at = (int64_t)head * a.q_rows + r0 + min(tid, valid - 1);
            nref = a.lse[at];       // as they are: a value worked on here would be waited for here
            ndelta = a.delta[at];
            npos = a.has_pos ? a.plan[a.pos_at + it.q0 + i0 + min(tid, valid - 1)] : 0;
        }
    };
    auto put = [&](int t) {
        const int buf = t & 1, i0 = it.qb + t * kBQ, i1 = min(i0 + kBQ, it.qe);
        sq.store(smem + buf * kBytes, tid);
        sg.store(smem + (2 + buf) * kBytes, tid);
        if (a.has_pos | !Sight(win, it.pos0 + i0, it.pos0 + i1 - 1).all(it.j0, it.nk)) odd |= sq.not_finite() | sg.not_finite();
        if (tid < kBQ) {
            // rows behind the last weigh nothing: their scores start from -inf
            rowref[buf * kBQ + tid] = tid < i1 - i0 ? lse_log2(nref) * from_lse : kMinusInf;
            rowdelta[buf * kBQ + tid] = tid < i1 - i0 ? -ndelta : 0.f;
            rowpos[buf * kBQ + tid] = npos;
        }
    };
    if constexpr (SUMS) {
        for (int i = tid; i < NW * (kShear + room); i += NW * 64) more[i] = 0.f;
        if (nt == 0)
            for (int i = tid; i < a.group * words; i += NW * 64)
                a.part_bias[((int64_t)(hk * a.group + i / words) * a.n_items + item) * words + i % words] = 0.f;
    }
    for (int head = hk * a.group; head < (hk + 1) * a.group && nt > 0; ++head) {
        fetch(head, 0);
        if constexpr (BIAS) load_bias<T>(bias, a.bias, 1.f / a.scale, a.heads, head, tid, NW * 64);
        put(0);
        __syncthreads();
        for (int t = 0; t < nt; ++t) {
            if (t + 1 < nt) fetch(head, t + 1);
            const int buf = t & 1, i0 = it.qb + t * kBQ;
            const char* qt = smem + buf * kBytes;
            const char* gt = smem + (2 + buf) * kBytes;
#pragma unroll D == 64 ? 1 : NQ
            for (int u = 0; u < NQ; ++u) {
                const int r0 = i0 + 32 * u;
                int pmin = it.pos0 + r0, pmax = it.pos0 + min(r0 + 31, it.nseq - 1);
                if (a.has_pos) {
                    const int tile = it.tile0 + (min(r0, it.nseq - 1) >> 5);
                    pmin = a.plan[a.tiles_at + 2 * tile];
                    pmax = a.plan[a.tiles_at + 2 * tile + 1];
                }
                const Sight sight(win, pmin, pmax);
                if (active & (r0 < it.qe) & !sight.none(j0, 32)) {
                    // with SUMS lanes behind the last key and rows behind the last count as hidden
                    const bool full = sight.all(j0, 32) & (!SUMS || ((32 * w + 32 <= it.nk) & (r0 + 32 <= it.qe)));
                    bool near = false;
                    const int* pos = rowpos + buf * kBQ + 32 * u + 4 * h;
                    const int far = j - (it.pos0 + r0 + 4 * h);      // to the row of register 0, where the plan lists no positions
                    const float up = lift.log2();
                    // The products start from what is taken off them: the scores from -lse (fp32: see kLseLast) and the bias, dP from -delta
                    f32x16_a s, p;
                    const V4<float>* less = reinterpret_cast<const V4<float>*>(rowref + buf * kBQ + 32 * u + 4 * h);
                    const V4<float>* del = reinterpret_cast<const V4<float>*>(rowdelta + buf * kBQ + 32 * u + 4 * h);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const V4<float> y = kLseLast<T> ? V4<float>{0.f, 0.f, 0.f, 0.f} : less[2 * x];
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * x + e] = y[e];
                        if constexpr (DK) {
                            const V4<float> z = del[2 * x];
#pragma unroll
                            for (int e = 0; e < 4; ++e) p[4 * x + e] = z[e];
                        }
                    }
                    const bool is_above = j0 - pmax >= reach, is_below = j0 + 31 - pmin <= -reach;
                    if constexpr (BIAS) {
                        near = !(is_above | is_below);
                        if (!near) {
                            const float b = bias[is_above ? 2 * reach + kBiasPad : 0];
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[r] += b;
                        } else if (a.has_pos) {
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[r] += bias[bias_at(j - pos[reg_row(r)], reach)];
                        } else {
                            const float* b = bias + bias_at(far - kBiasPad, reach) + kBiasPad;
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[r] += b[-reg_row(r)];
                        }
                    }
                    if constexpr (DK) row_products<T, D, kGroup>(s, p, qt, gt, 32 * u, kf, vf, lane);
                    else row_product<T, D, D <= 64 ? 4 : 2>(s, qt, 32 * u, kf, lane);
                    Cols<T, D> gc, qc;
                    if constexpr (kEarly) {
                        gc.read(gt, 32 * u, lane);
                        qc.read(qt, 32 * u, lane);
                        after_reads<T>();
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        V4<float> y{0.f, 0.f, 0.f, 0.f};
                        if constexpr (kLseLast<T>) y = less[2 * x];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = 4 * x + e;
                            s[r] = __builtin_amdgcn_exp2f(kLseLast<T> ? fmaf(s[r], c, y[e]) : Lift<T>::kOn ? fmaf(s[r], c, up) : s[r] * c);
                            if constexpr (DK) p[r] *= s[r];
                        }
                    }
                    if (!full) {
                        if (a.has_pos) {
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const bool see = visible(win, j - pos[reg_row(r)], j);
                                if constexpr (DV) s[r] = see ? s[r] : 0.f;
                                if constexpr (DK) p[r] = see ? p[r] : 0.f;
                            }
                        } else {
                            // row c is seen if far - c <= right and far - c >= -left, or the key is one of the first
                            const int lo = far - win.right;
                            int hi = j < win.sinks ? kFar : far + win.left;
                            if constexpr (SUMS) hi = min(hi, it.qe - 1 - r0 - 4 * h);
                            const int m = !SUMS || key < it.nk ? max(hi - lo + 1, 0) : 0;
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const bool see = (unsigned)(reg_row(r) - lo) < (unsigned)m;
                                if constexpr (DV) s[r] = see ? s[r] : 0.f;
                                if constexpr (DK) p[r] = see ? p[r] : 0.f;
                            }
                        }
                    }
                    if constexpr (SUMS) {
                        if (near) {
                            auto put_sheared = [&](const f32x16_a& d) {
                                float* mine = shear + 32 + (lane & 31) * kShearRow + 4 * h;
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const V4<float> y{d[4 * x], d[4 * x + 1], d[4 * x + 2], d[4 * x + 3]};
                                    *reinterpret_cast<V4<float>*>(mine + 8 * x) = y;
                                }
                            };
                            if (Lift<T>::kOn && lift.moved) {     // keys meet in a sum
                                f32x16_a d = p;
                                Lift<T>::down(d, lift.e - Lift<T>::kFirst);
                                put_sheared(d);
                            } else {
                                put_sheared(p);
                            }
                        } else {
                            float sum = 0.f;
#pragma unroll
                            for (int r = 0; r < 16; ++r) sum += p[r];
                            sum = lift.off(sum);
                            above += is_above ? sum : 0.f;
                            below += is_above ? 0.f : sum;
                        }
                    }
                    if constexpr (DK && DV) {
                        // P and dS of a key by one power of two
                        if constexpr (Lift<T>::kOn) {
                            const int before = lift.e;
                            lift.settle(p, dk, dv);
                            if (lift.moved) Lift<T>::down(s, before - lift.e);
                        }
                    } else if constexpr (DK) {
                        lift.settle(p, dk);
                    }
                    if constexpr (DV) {
                        if constexpr (!kEarly) {
                            gc.read(gt, 32 * u, lane);
                            after_reads<T>();
                        }
                        gc.product(dv, s);
                    }
                    if constexpr (DK) {
                        if constexpr (!kEarly) {
                            qc.read(qt, 32 * u, lane);
                            after_reads<T>();
                        }
                        qc.product(dk, p);
                    }
                    if constexpr (SUMS) {
                        if (near) {     // while the matrix instructions run
                            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                            __builtin_amdgcn_wave_barrier();
                            // lane l: row - key = l - 31, which is the distance 31 - l + (j0 - position of row r0)
                            const float* from = shear + 32 + lane - 31;
                            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int i = 0; i < 32; ++i) part[i & 3] += from[i * (kShearRow + 1)];
                            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                            __builtin_amdgcn_wave_barrier();
                            const int dist = j0 + 31 - lane - (it.pos0 + r0) + reach + kFarPad;
                            if (lane < 63) sums[dist] += Lift<T>::off_first((part[0] + part[1]) + (part[2] + part[3]));
                        }
                    }
                }
            }
            if (t + 1 < nt) put(t + 1);
            __syncthreads();
        }
        if constexpr (SUMS) {
#pragma unroll
            for (int k = 32; k; k >>= 1) {
                above += __shfl_xor(above, k);
                below += __shfl_xor(below, k);
            }
            if (lane == 0) {
                sums[words - 1] += above;
                sums[0] += below;
            }
            above = below = 0.f;
            __syncthreads();
            float* all = more + NW * kShear;
            float* out = a.part_bias + ((int64_t)head * a.n_items + item) * words;
            for (int i = tid; i < words; i += NW * 64) {
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < NW; ++k) {
                    sum += all[k * room + i];
                    all[k * room + i] = 0.f;
                }
                out[i] = sum;
            }
        }
    }
    float dk_by = lift.off(a.scale), dv_by = lift.off(1.f);
    bool redo = __syncthreads_or((int)odd);
    if constexpr (BIAS)
        if (!redo && __ballot(!finite((DK ? sum_of_all(dk) : 0.f) + (DV ? sum_of_all(dv) : 0.f)))) redo = table_hides<T>(a.bias, a.heads, hk * a.group, a.group);
    if (redo) {
        float x[16 * DT], y[16 * DT];
        dkv_by_pairs<T, D, DT, BIAS>(kernel_args(), x, y, a.items_at, item, hk, keyc, h);
        if constexpr (DK) take<DT>(dk, x);
        if constexpr (DV) take<DT>(dv, y);
        dk_by = a.scale, dv_by = 1.f;
    }
    if (key < it.nk) {
        if (it.slot < 0) {
            T* ok = const_cast<T*>(row_ptr<T>(a.dk, (int64_t)it.k0 + key, hk));
            T* ov = const_cast<T*>(row_ptr<T>(a.dv, (int64_t)it.k0 + key, hk));
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int x = 0; x < (D >= 32 ? 4 : 2); ++x) {
                    V4<T> y, z;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = (T)(dk[d][4 * x + e] * dk_by);
                        z[e] = (T)(dv[d][4 * x + e] * dv_by);
                    }
                    if constexpr (DK) *reinterpret_cast<V4<T>*>(ok + 32 * d + 8 * x + 4 * h) = y;
                    if constexpr (DV) *reinterpret_cast<V4<T>*>(ov + 32 * d + 8 * x + 4 * h) = z;
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
                        y[e] = dk[d][4 * x + e] * dk_by;
                        z[e] = dv[d][4 * x + e] * dv_by;
                    }
                    if constexpr (DK) *reinterpret_cast<V4<float>*>(ok + 32 * d + 8 * x + 4 * h) = y;
                    if constexpr (DV) *reinterpret_cast<V4<float>*>(ov + 32 * d + 8 * x + 4 * h) = z;
                }
        }
    }
}

// dk, dv of a tile of keys from the parts of several workgroups (grid.y: keys and values, and groups of eight rows)
template <typename T, int D>
__global__ __launch_bounds__(kJoinRows * (D / 4)) void attn_dkv_join_kernel(AttnArgs a, int n_join, int join_at, int tile_keys) {
    const int kvh = a.heads / a.group, hk = blockIdx.x / n_join, which = blockIdx.y & 1;
    const Join jn = reinterpret_cast<const Join*>(a.plan + join_at)[blockIdx.x - hk * n_join];
    const int r = (blockIdx.y >> 1) * kJoinRows + threadIdx.x / (D / 4), d = (threadIdx.x % (D / 4)) * 4;
    if (r >= jn.n) return;
    V4<float> x{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < jn.slots; ++k)
        x += *reinterpret_cast<const V4<float>*>(a.part_o + ((((int64_t)(jn.slot0 + k) * kvh + hk) * 2 + which) * tile_keys + r) * D + d);
    V4<T> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)x[e];
    *reinterpret_cast<V4<T>*>(const_cast<T*>(row_ptr<T>(which ? a.dv : a.dk, (int64_t)jn.row0 + r, hk)) + d) = y;
}

template <typename T, int D, int NW>
hipError_t dq_waves(const AttnArgs& a, hipStream_t s) {
    const int64_t blocks = (int64_t)a.n_items * a.heads;
    const size_t tiles = 4 * kDqKeys<T, D, false> * D * sizeof(T), tiles_pos = 4 * kDqKeys<T, D, true> * D * sizeof(T), bias = bias_floats(a) * 4;
    if (!a.bias.table) return start(attn_dq_kernel<T, D, NW, false, false>, blocks, NW * 64, tiles, s, a);
    if (!a.has_pos) return start(attn_dq_kernel<T, D, NW, true, false>, blocks, NW * 64, tiles + bias, s, a);
    return start(attn_dq_kernel<T, D, NW, true, true>, blocks, NW * 64, tiles_pos + bias + 4 * bin_floats(NW, a.bias.n_buckets, a.bias.reach), s, a);
}
template <typename T, int D>
hipError_t dq_dim(const AttnArgs& a, int waves, hipStream_t s) {
    return waves == 2 ? dq_waves<T, D, 2>(a, s) : dq_waves<T, D, 4>(a, s);
}

template <typename T, int D, int NW, bool BIAS, bool SUMS, int PART>
hipError_t dkv_start(const AttnArgs& a, hipStream_t s) {
    const int64_t blocks = (int64_t)a.n_items * (a.heads / a.group);
    constexpr int kRows = kRowsPerTile<T, D>;
    const size_t lds = 4 * kRows * D * sizeof(T) + 6 * kRows * 4 + (bias_floats(a) + (SUMS ? diagonal_floats(NW, a.bias.reach) : 0)) * 4;
    return start(attn_dkv_kernel<T, D, NW, BIAS, SUMS, PART>, blocks, NW * 64, lds, s, a);
}
template <typename T, int D, int NW, int PART>
hipError_t dkv_part(const AttnArgs& a, hipStream_t s) {
    if (!a.bias.table) return dkv_start<T, D, NW, false, false, PART>(a, s);
    if constexpr (PART != kOnlyDv)
        if (!a.has_pos) return dkv_start<T, D, NW, true, true, PART>(a, s);
    return dkv_start<T, D, NW, true, false, PART>(a, s);
}
template <typename T, int D, int NW>
hipError_t dkv_waves(const AttnArgs& a, hipStream_t s) {
    if constexpr (kTwoLaunches<T, D>) {
        const hipError_t e = dkv_part<T, D, NW, kOnlyDk>(a, s);
        return e != hipSuccess ? e : dkv_part<T, D, NW, kOnlyDv>(a, s);
    } else {
        return dkv_part<T, D, NW, kBoth>(a, s);
    }
}
template <typename T, int D>
hipError_t dkv_dim(const AttnArgs& a, int waves, hipStream_t s) {
    return waves == 2 ? dkv_waves<T, D, 2>(a, s) : dkv_waves<T, D, 4>(a, s);
}

template <typename T, int D>
hipError_t dkv_join_dim(const AttnArgs& a, int n_join, int join_at, int tile_keys, hipStream_t s) {
    if (n_join == 0) return hipSuccess;
    return launch(attn_dkv_join_kernel<T, D>, dim3((unsigned)n_join * (a.heads / a.group), 2 * (tile_keys / kJoinRows)), dim3(kJoinRows * (D / 4)), 0, s, a,
                  n_join, join_at, tile_keys);
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
    hipError_t attn_join_##NAME(const AttnArgs& a, int dim, int n, int at, hipStream_t s) { return DPTM_ATTN_BY_DIM(join_dim, a, n, at, s); } \
    hipError_t attn_dkv_join_##NAME(const AttnArgs& a, int dim, int n, int at, int keys, hipStream_t s) {                  \
        return DPTM_ATTN_BY_DIM(dkv_join_dim, a, n, at, keys, s);                                                          \
    }                                                                                                                      \
    hipError_t attn_short_grad_##NAME(const AttnArgs& a, int dim, int waves, int k_items_at, hipStream_t s) {                \
        return DPTM_ATTN_BY_DIM(short_grad_dim, a, waves, k_items_at, s);                                                 \
    }                                                                                                                      \
    hipError_t attn_dtable_##NAME(const AttnArgs& a, int n_items, hipStream_t s) { return dtable_of<E>(a, n_items, s); }   \
    }
