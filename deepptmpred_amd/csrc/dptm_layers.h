// Layer operators on device tensors (attention over packed sequences, per-head norm with rotation): argument blocks and
// launchers shared by the entry points (dptm_layers.hip) and the kernels (dptm_attn_*.hip, dptm_norm_rope.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>

namespace dptm {

// A kernel's launch with its own result: the last error of the thread may be another call's.
template <typename... P, typename... A>
inline hipError_t launch(void (*kernel)(P...), dim3 blocks, dim3 threads, size_t lds, hipStream_t s, const A&... args) {
    std::tuple<P...> kept(args...);
    return std::apply(
        [&](P&... p) {
            void* at[] = {static_cast<void*>(&p)...};
            return hipLaunchKernel(reinterpret_cast<const void*>(kernel), blocks, threads, at, lds, s);
        },
        kept);
}

// The attention plan is one array of 32-bit words that dptm_attention_plan fills on the host; the caller keeps one copy
// there (the launchers read the header) and one on the device (the kernels read the lists behind it).
enum PlanWord {
    kPlanMagicAt = 0, kPlanWords, kPlanHeads, kPlanKvHeads, kPlanHeadDim, kPlanLeft, kPlanRight, kPlanSinks, kPlanSeqs,
    kPlanQRows, kPlanKRows, kPlanMode, kPlanFwd, kPlanFwdAt, kPlanSlots, kPlanJoin, kPlanJoinAt, kPlanDq, kPlanDqAt,
    kPlanDqWaves, kPlanDkv, kPlanDkvAt, kPlanDkvWaves, kPlanDkvSlots, kPlanDkvJoin, kPlanDkvJoinAt, kPlanHasPos, kPlanPosAt,
    kPlanTiles, kPlanTilesAt, kPlanPack, kPlanCheck, kPlanHeader = 32
};
constexpr int kPlanMagic = 0x31544144;   // "DAT1"
constexpr int kFar = 1 << 29;            // a window side without limit; lengths and positions stay below it

// forward modes: rows of a workgroup's tile, and whether its wavefronts share the keys or split them
enum { kWide128 = 0, kWide64 = 1, kSplitKeys = 2 };

// kPlanDqWaves of a plan whose dq and dk, dv are formed together (dptm_attn_short.h): no sequence has more than 64 rows or keys,
// heads are not larger than this, and entry i of both lists is sequence i of those that are not empty
constexpr int kTogether = 1, kShortDim = 64;

struct QItem {       // a tile of query rows: forward and dq
    int q0, nq;      // first row of the packed q, rows
    int k0;          // first row of the sequence in the packed k
    int pos0;        // position of row q0 when the plan holds no position list
    int kb, ke;      // keys [kb, ke) of the sequence, and
    int sink_end;    // keys [0, sink_end), sink_end <= kb
    int slot;        // partial result to write, -1: the result itself
};
struct KItem {       // a tile of keys: dk and dv
    int k0, nk;      // first row of the packed k, rows
    int j0;          // index of the first key in its sequence
    int q0;          // first row of the sequence in the packed q
    int qb, qe;      // rows [qb, qe) of the sequence, qb a multiple of 32
    int pos0;        // position of the sequence's row 0 when the plan holds no position list
    int slot;        // partial result to write, -1: the result itself
    int tile0;       // entry of the sequence's first 32 rows in the list of position bounds
    int nseq;        // query rows of the sequence
    int pad[2];
};
struct Join { int row0, n, slot0, slots; };   // rows, and the partial results that add up to them

struct Strided { void* p; int64_t row, head; };   // elements of the type between rows and between heads

struct BiasArgs {
    const void* table;     // [n_buckets][heads], the tensors' type; NULL: no bias
    const int* buckets;    // [2 * reach + 1]
    int n_buckets, reach;
};

struct AttnArgs {
    Strided q, k, v, out, dout, dq, dk, dv;
    float* lse;            // [heads][q_rows]
    float* delta;          // [heads][q_rows]
    float* part_o;         // forward partials [slot * heads + h][32][D]; backward: dk | dv partials
    float* part_ml;        // the same [32][2]
    float* part_bias;      // [heads][tiles][dtable_words]
    double* part_groups;   // [heads][dtable_groups][dtable_words]
    void* dtable;          // [n_buckets][heads]
    const int* plan;       // device copy
    BiasArgs bias;
    float scale;           // of the scores
    int heads, group;      // query heads, query heads per key head
    int left, right, sinks, q_rows, n_items, items_at, has_pos, pos_at, tiles_at;
    int by_sequence;       // the wide forward kernel takes the heads of a tile one behind the other, not the tiles of a head
    int pack;              // heads of a group that share a tile of rows where the keys are split
};

// one set of launchers per element type; dim is one of 16, 32, 64, 128
#define DPTM_ATTN_LAUNCHERS(T)                                                                          \
    hipError_t attn_forward_##T(const AttnArgs& a, int dim, int mode, hipStream_t s);                   \
    hipError_t attn_dq_##T(const AttnArgs& a, int dim, int waves, hipStream_t s);                       \
    hipError_t attn_dkv_##T(const AttnArgs& a, int dim, int waves, hipStream_t s);                      \
    hipError_t attn_join_##T(const AttnArgs& a, int dim, int n_join, int join_at, hipStream_t s);       \
    hipError_t attn_dkv_join_##T(const AttnArgs& a, int dim, int n_join, int join_at, int tile_keys, hipStream_t s); \
    hipError_t attn_short_grad_##T(const AttnArgs& a, int dim, int waves, int k_items_at, hipStream_t s); \
    hipError_t attn_dtable_##T(const AttnArgs& a, int n_items, hipStream_t s);
DPTM_ATTN_LAUNCHERS(bf16)
DPTM_ATTN_LAUNCHERS(f16)
DPTM_ATTN_LAUNCHERS(f32)

// words of a dq tile's sums for the bias gradient: by distance (with 62 on either side, see dptm_attn_grad.h), or by
// bucket where the plan lists positions
constexpr int kFarPad = 62;
inline int dtable_words(int has_pos, int n_buckets, int reach) { return has_pos ? n_buckets : 2 * reach + 1 + 2 * kFarPad; }

inline int dtable_groups(int n_items) { return n_items < 64 ? n_items : 64; }

struct NormRopeArgs {
    Strided x[2], y[2], dy[2], dx[2];   // q and k
    int heads[2];
    const float* gain[2];               // NULL: no norm
    const float* cosv;                  // [n_pos][D / 2]
    const float* sinv;
    const int* positions;               // NULL: row r stands at position r
    float* part[2];                     // [blocks][D] partial gain gradients
    float* dgain[2];
    int64_t rows;
    int n_pos, dim, interleaved;
    float eps;
};
hipError_t norm_rope_forward(const NormRopeArgs& a, int dtype, hipStream_t s);
hipError_t norm_rope_backward(const NormRopeArgs& a, int dtype, hipStream_t s);
int norm_rope_blocks(int64_t rows, int heads, int dim);

}  // namespace dptm
