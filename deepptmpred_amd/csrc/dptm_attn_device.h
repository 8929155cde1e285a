// Device helpers of the attention kernels: operand fragments of the 32x32 matrix instructions for the three element
// types, tiles in LDS on the way there, visibility of a pair, the relative position bias.
//
// Layout.  v_mfma_f32_32x32x16 leaves D[row][col] with col = lane % 32 and row = 8 (r / 4) + 4 (lane / 32) + r % 4 for
// register r.  Taken as S^T = K Q^T a lane holds one query's scores of 16 keys, so row sums and maxima are in-lane but for
// one exchange between the half-waves, and registers 8s..8s+7 ARE the B operand of the next product (contraction over
// the keys 16 s + {4h..4h+3, 8+4h..8+4h+3}), whose order within a step is free as long as the A operand uses it too.
// Products chain register to register; the A operand of the second product is read from LDS transposed.
#pragma once
#include <hip/hip_runtime.h>

#include "dptm_layers.h"

namespace dptm {

typedef float f32x16_a __attribute__((ext_vector_type(16)));
typedef short s16x4_a __attribute__((ext_vector_type(4)));
typedef short s16x8_a __attribute__((ext_vector_type(8)));
typedef unsigned u32x4_a __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kMinusInf = -__builtin_inff();

template <typename T> struct Elem;
template <> struct Elem<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    static constexpr unsigned kExp = 0x7f80;
};
template <> struct Elem<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    static constexpr unsigned kExp = 0x7c00;
};
template <> struct Elem<float> {
    static constexpr unsigned kExp = 0x7f80;
    typedef float v8 __attribute__((ext_vector_type(8)));
    typedef float v4 __attribute__((ext_vector_type(4)));
};
template <typename T> using V8 = typename Elem<T>::v8;
template <typename T> using V4 = typename Elem<T>::v4;

// one step of 16 along the contraction; lane: index lane % 32, contraction elements 8 (lane / 32) .. +7.  In fp32 the step is
// eight 32x32x2 instructions, element e of both operands in the e-th.
__device__ __forceinline__ void mma(f32x16_a& c, const V8<__bf16>& a, const V8<__bf16>& b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16_a& c, const V8<_Float16>& a, const V8<_Float16>& b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16_a& c, const V8<float>& a, const V8<float>& b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ V8<T> pack8(const f32x16_a& x, int s) {   // registers 8s..8s+7
    V8<T> r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = (T)x[8 * s + e];
    return r;
}

// ---- a tile of rows in LDS: 16-byte chunks, chunk index XORed with a function of the row so that both the row reads
// ---- (32 rows, one chunk) and the transposed reads (8 rows, four chunks) spread over the banks
template <typename T, int D>
struct Tile {
    static constexpr int kChunks = D * (int)sizeof(T) / 16;   // of a row
    __device__ static __forceinline__ int swz(int row) {
        if constexpr (kChunks >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        else if constexpr (kChunks == 8) return ((row >> 1 & 1) << 2) | (row >> 2 & 3);
        else if constexpr (kChunks == 4) return row >> 2 & 3;
        else return row >> 3 & 1;
    }
    // A or B operand with the row on the lane: contraction elements 16 step + 8h ..
    __device__ static __forceinline__ V8<T> row_frag(const char* t, int row, int step, int h) {
        const char* p = t + row * (kChunks * 16);
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const V8<T>*>(p + (((2 * step + h) ^ swz(row)) << 4));
        } else {
            const V4<T> lo = *reinterpret_cast<const V4<T>*>(p + (((4 * step + 2 * h) ^ swz(row)) << 4));
            const V4<T> hi = *reinterpret_cast<const V4<T>*>(p + (((4 * step + 2 * h + 1) ^ swz(row)) << 4));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // A operand with the column 32 dt + lane % 32 on the lane: contraction rows row0 + {4h..4h+3, 8+4h..8+4h+3}.
    // 16-bit types: each group of 16 lanes hands in 4 rows x 16 columns and takes a column of 4 (ds_read_b64_tr_b16).
    // Head dimension 16 has half a tile of columns: the other lanes repeat them, and their results are not used.
    __device__ static __forceinline__ V8<T> col_frag(const char* t, int row0, int dt, int lane) {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            const int q = lane & 15;
            const int col = 32 * dt + (D >= 32 ? (lane & 16) : 0) + 4 * (q & 3);
            s16x4_a r[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = row0 + 8 * i + 4 * h + (q >> 2);
                const char* p = t + row * (kChunks * 16) + (((col >> 3) ^ swz(row)) << 4) + (col & 7) * 2;
                r[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_a*)(p));
            }
            return __builtin_bit_cast(V8<T>, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int col = (32 * dt + (lane & 31)) & (D - 1);
            V8<T> f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = row0 + 8 * (e >> 2) + 4 * h + (e & 3);
                f[e] = *reinterpret_cast<const float*>(t + row * (kChunks * 16) + (((col >> 2) ^ swz(row)) << 4) + (col & 3) * 4);
            }
            return f;
        }
    }
};

// Left to itself the compiler reads one LDS fragment, waits, and feeds it, to spare registers: a wavefront then stands for
// the LDS latency of every fragment (56 % of its time in the dk, dv kernel).  For the 16-bit types a product's fragments are
// therefore asked for as a group in front of a scheduling barrier in the backward kernels.  (The forward kernel has three
// wavefronts a SIMD that cover for each other, and loses one or spills with more fragments in registers: 127 us for 48
// proteins as it is, 153 to 166 with groups.)  In fp32 a fragment feeds eight instructions and is
// twice as large, and the order is left alone.
template <typename T> __device__ __forceinline__ void after_reads() {
    if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
}
// the row fragments of one lane.  Left to itself the compiler keeps the places of all steps over the loop around them: eight registers
// with 16-bit heads of 128, whose kernels spill operands for them.  There they are formed from one, which it cannot see through.
template <typename T, int D>
struct RowFrags {
    static constexpr bool kFresh = sizeof(T) == 2 && D == 128;
    int row, h;
    unsigned place = 0;
    __device__ __forceinline__ RowFrags(int row, int h) : row(row), h(h) {
        if constexpr (kFresh) {
            place = row * (D * (int)sizeof(T)) + ((h ^ Tile<T, D>::swz(row)) << 4);      // of step 0; step s flips bits 5 to 7
            asm volatile("" : "+v"(place));
        }
    }
    __device__ __forceinline__ V8<T> get(const char* t, int step) const {
        if constexpr (kFresh) return *reinterpret_cast<const V8<T>*>(t + (place ^ (unsigned)(step << 5)));
        else return Tile<T, D>::row_frag(t, row, step, h);
    }
};
// c0 += A0 B0 and c1 += A1 B1 over the whole head dimension, A rows row0 .. row0 + 31 of two tiles; MOST steps at a time
template <typename T, int D, int MOST>
__device__ __forceinline__ void row_products(f32x16_a& c0, f32x16_a& c1, const char* t0, const char* t1, int row0, const V8<T> (&b0)[D / 16],
                                             const V8<T> (&b1)[D / 16], int lane) {
    constexpr int G = D / 16 < MOST ? D / 16 : MOST;
    const RowFrags<T, D> rows(row0 + (lane & 31), lane >> 5);
#pragma unroll
    for (int g = 0; g < D / 16; g += G) {
        V8<T> f0[G], f1[G];
#pragma unroll
        for (int s = 0; s < G; ++s) {
            f0[s] = rows.get(t0, g + s);
            f1[s] = rows.get(t1, g + s);
        }
        after_reads<T>();
#pragma unroll
        for (int s = 0; s < G; ++s) {
            mma(c0, f0[s], b0[g + s]);
            mma(c1, f1[s], b1[g + s]);
        }
    }
}
// c0 += A0 B0 alone
template <typename T, int D, int MOST>
__device__ __forceinline__ void row_product(f32x16_a& c0, const char* t0, int row0, const V8<T> (&b0)[D / 16], int lane) {
    constexpr int G = D / 16 < MOST ? D / 16 : MOST;
    const RowFrags<T, D> rows(row0 + (lane & 31), lane >> 5);
#pragma unroll
    for (int g = 0; g < D / 16; g += G) {
        V8<T> f0[G];
#pragma unroll
        for (int s = 0; s < G; ++s) f0[s] = rows.get(t0, g + s);
        after_reads<T>();
#pragma unroll
        for (int s = 0; s < G; ++s) mma(c0, f0[s], b0[g + s]);
    }
}
// the transposed fragments of 32 rows of a tile
template <typename T, int D>
struct Cols {
    static constexpr int DT = D >= 32 ? D / 32 : 1;
    V8<T> f[2][DT];
    __device__ __forceinline__ void read(const char* t, int row0, int lane) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int d = 0; d < DT; ++d) f[s][d] = Tile<T, D>::col_frag(t, row0 + 16 * s, d, lane);
    }
    // acc += rows^T w, w a 32 x 32 tile with the rows on its registers
    __device__ __forceinline__ void product(f32x16_a (&acc)[DT], const f32x16_a& w) const {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const V8<T> b = pack8<T>(w, s);
#pragma unroll
            for (int d = 0; d < DT; ++d) mma(acc[d], f[s][d], b);
        }
    }
    // the same, 16-bit weights of every other 16 rows in twice as many bits: what their rounding leaves goes through again
    __device__ __forceinline__ void product_more_bits(f32x16_a (&acc)[DT], const f32x16_a& w) const {
        product(acc, w);
        if constexpr (sizeof(T) == 2) {
            V8<T> left;
#pragma unroll
            for (int e = 0; e < 8; ++e) left[e] = (T)(w[e] - (float)(T)w[e]);
#pragma unroll
            for (int d = 0; d < DT; ++d) mma(acc[d], f[0][d], left);
        }
    }
};

// ROWS rows of a strided tensor on the way to LDS through registers; rows from `valid` on become zeros.  Offsets within
// the rows are kept as 32 bits behind a uniform address (row strides are refused from 2^25 bytes on).
template <typename T, int D, int ROWS, int NT>
struct Stage {
    static constexpr int kChunks = Tile<T, D>::kChunks;
    static constexpr int kAll = ROWS * kChunks, kMine = (kAll + NT - 1) / NT, kRowStep = NT / kChunks;
    u32x4_a r[kMine];
    unsigned at, step;     // this thread's first chunk, the next ones lie `step` bytes on
    __device__ __forceinline__ Stage(int64_t row_bytes, int tid) {
        at = (unsigned)(tid / kChunks) * (unsigned)row_bytes + (tid % kChunks) * 16;
        step = kRowStep * (unsigned)row_bytes;
    }
    __device__ __forceinline__ void load(const char* base, int valid, int tid) {
        if (valid >= ROWS && kAll % NT == 0) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) r[i] = *reinterpret_cast<const u32x4_a*>(base + i * step + at);
        } else {
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int row = tid / kChunks + i * kRowStep;
                r[i] = u32x4_a{0, 0, 0, 0};
                if (row < min(valid, ROWS)) r[i] = *reinterpret_cast<const u32x4_a*>(base + i * step + at);
            }
        }
    }
    __device__ __forceinline__ void store(char* t, int tid) const {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int c = tid + i * NT, row = c / kChunks;
            if (kAll % NT == 0 || c < kAll)
                *reinterpret_cast<u32x4_a*>(t + row * (kChunks * 16) + (((c % kChunks) ^ Tile<T, D>::swz(row)) << 4)) = r[i];
        }
    }
    // not 0 if an element of this thread's part is an infinity or a NaN: adding 1 to an exponent of all ones reaches the sign
    __device__ __forceinline__ unsigned not_finite() const {
        constexpr unsigned kMask = sizeof(T) == 4 ? 0x7f800000u : Elem<T>::kExp * 0x10001u;
        constexpr unsigned kOne = sizeof(T) == 4 ? 0x00800000u : (0x8000u - Elem<T>::kExp) * 0x10001u;
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) bits |= (r[i][e] & kMask) + kOne;
        return bits & (sizeof(T) == 4 ? 0x80000000u : 0x80008000u);
    }
};

// operand straight from memory: row on the lane
template <typename T>
__device__ __forceinline__ V8<T> global_frag(const char* row, int step, int h) {
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const V8<T>*>(row + (2 * step + h) * 16);
    } else {
        const V4<T> lo = *reinterpret_cast<const V4<T>*>(row + (4 * step + 2 * h) * 16);
        const V4<T> hi = *reinterpret_cast<const V4<T>*>(row + (4 * step + 2 * h + 1) * 16);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

__device__ __forceinline__ float half_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = min(v, __shfl_xor(v, m));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = max(v, __shfl_xor(v, m));
    return __builtin_amdgcn_readfirstlane(v);
}

// key index of register r of a 32-key score tile, without the 4h
__device__ __forceinline__ constexpr int reg_row(int r) { return 8 * (r >> 2) + (r & 3); }

// pair of a query and a key `far` = key - position behind it: within the window, or one of the first keys.  Without short
// circuits, so that a mask is compares and selects: as branches it is slow, and hipcc 7.2 has dropped the select of a
// score register whose condition it had turned into control flow.
struct Window { int left, right, sinks; };
__device__ __forceinline__ bool visible(const Window& w, int far, int key) {
    return (far <= w.right) & ((far >= -w.left) | (key < w.sinks));
}
// The same for the 16 keys of a lane's score registers: register r is visible if reg_row(r) - lo < n unsigned, or
// reg_row(r) < first.  Three or four instructions an element.
struct LaneMask { int lo, n, first; };
__device__ __forceinline__ LaneMask lane_mask(const Window& w, int pos, int key0, int key_end) {
    const int lo = pos - w.left - key0, hi = min(pos + w.right, key_end - 1) - key0;
    return LaneMask{lo, max(hi - lo + 1, 0), min(w.sinks - key0, hi + 1)};
}
__device__ __forceinline__ bool in_window(const LaneMask& m, int c) { return (unsigned)(c - m.lo) < (unsigned)m.n; }
// registers of hidden pairs become `value`
__device__ __forceinline__ void hide(f32x16_a& s, const LaneMask& m, float value) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = (in_window(m, reg_row(r)) | (reg_row(r) < m.first)) ? s[r] : value;
}
// What rows at positions [pmin, pmax] see of keys [j0, j0 + span), from limits that are formed once: a wavefront asks for
// every tile, and scalar arithmetic with branches per tile costs as much as the tile's exponentials.
struct Sight {
    int none_from, none_to, full_to, full_from, sinks;
    __device__ __forceinline__ Sight(const Window& w, int pmin, int pmax)
        : none_from(pmax + w.right), none_to(pmin - w.left), full_to(pmin + w.right), full_from(pmax - w.left), sinks(w.sinks) {}
    __device__ __forceinline__ bool none(int j0, int span) const {
        return (j0 > none_from) | ((j0 + span <= none_to) & (j0 >= sinks));
    }
    __device__ __forceinline__ bool all(int j0, int span) const {
        return (j0 + span - 1 <= full_to) & ((j0 >= full_from) | (j0 + span <= sinks));
    }
};
// The keys of a tile of rows: first [0, sink_end), then [kb, ke), `step` keys at a time
struct KeyWalk {
    int j0, end;          // this tile's first key, end of its piece
    int kb, ke;
    bool first_keys;
    __device__ __forceinline__ KeyWalk(const QItem& it)
        : j0(it.sink_end > 0 ? 0 : it.kb), end(it.sink_end > 0 ? it.sink_end : it.ke), kb(it.kb), ke(it.ke), first_keys(it.sink_end > 0) {}
    __device__ __forceinline__ bool more() const { return j0 < end; }
    __device__ __forceinline__ KeyWalk next(int step) const {
        KeyWalk n = *this;
        n.j0 += step;
        if (first_keys && n.j0 >= end) n.j0 = kb, n.end = ke, n.first_keys = false;
        return n;
    }
};

// A hidden pair's weight is 0, but 0 * inf and 0 * NaN are NaN.  Where a tile holds hidden pairs its threads look, on the way
// to LDS, whether its rows hold such an element (Stage::not_finite), and workgroups that found one do their rows over at the
// end, pair by pair.  Pairs that the bias table hides are not looked for tile by tile: a score of -inf takes up any NaN, so that a
// result that came out finite met none.  Where one did not and the table hides something, the rows are done over as well.

// ---- relative position bias in LDS: value per distance, divided by the scale of the scores, because the score products start
// ---- from it (init_bias) instead of from zero: the bias costs no arithmetic per element, and no branch touches a score.
// ---- Entries at or below -2^100 hide their pairs, so that a table of the type's lowest value works as a mask does
// The table goes on for 31 distances on either side with the last value: a lane clamps the distance of its first key of a
// tile alone (bias_at), and the others lie behind it.
constexpr int kBiasPad = 31;
__host__ __device__ inline int bias_room(int reach) { return (2 * reach + 1 + 2 * kBiasPad + 3) & ~3; }   // floats
__device__ __forceinline__ int bias_at(int far, int reach) { return min(max(far, -reach - kBiasPad), reach) + reach + kBiasPad; }
__device__ __forceinline__ float bias_value(float v, float inv_scale) { return v <= -0x1p100f ? kMinusInf : v * inv_scale; }
// whether the table hides a bucket of the heads [head, head + n); the same answer in every lane.  64 buckets at most, one a lane
template <typename T>
__device__ __forceinline__ bool table_hides(const BiasArgs& b, int heads, int head, int n) {
    const int lane = threadIdx.x & 63;
    bool any = false;
    for (int i = 0; i < n; ++i)
        any |= lane < b.n_buckets && bias_value((float)static_cast<const T*>(b.table)[(int64_t)lane * heads + head + i], 1.f) == kMinusInf;
    return __ballot(any) != 0;
}
// not finite if one of the accumulators is not
template <int DT>
__device__ __forceinline__ float sum_of_all(const f32x16_a (&acc)[DT]) {
    float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r & 3] += acc[d][r];
    return (z[0] + z[1]) + (z[2] + z[3]);
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < __builtin_inff(); }
template <typename T>
__device__ __forceinline__ void load_bias(float* lds, const BiasArgs& b, float inv_scale, int heads, int head, int tid, int nt) {
    const T* table = static_cast<const T*>(b.table);
    const int n = 2 * b.reach + 1 + 2 * kBiasPad;
    // four entries at a time: the second load of an entry waits for its first
    for (int i0 = tid; i0 < n; i0 += 4 * nt) {
        int k[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) k[u] = b.buckets[min(max(i0 + u * nt - kBiasPad, 0), 2 * b.reach)];
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = (float)table[(int64_t)min(max(k[u], 0), b.n_buckets - 1) * heads + head];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * nt < n) lds[i0 + u * nt] = bias_value(v[u], inv_scale);
    }
}

// accumulators of 32 keys, the first of a lane `far` behind its query
__device__ __forceinline__ void init_bias(f32x16_a& s, const float* bias, int reach, int far) {
    const float* b = bias + bias_at(far, reach);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = b[reg_row(r)];
}

// blocks of one key head's tiles on one XCD, which has an L2 of its own: block b runs on XCD b % 8, and each XCD takes a
// contiguous piece of the (head-major) order
__device__ __forceinline__ int xcd_order(int b, int n) {
    const int per = n >> 3, rest = n & 7, x = b & 7, i = b >> 3;
    return x * per + min(x, rest) + i;
}

__device__ __forceinline__ int row_position(const int* plan, int has_pos, int pos_at, int pos0, int q0, int i) {
    return has_pos ? plan[pos_at + q0 + i] : pos0 + i;
}

}  // namespace dptm
