// What the kernels of tree speculation share: their parameters, how the work of a launch is dealt out to its CTAs from
// lengths that only the device knows, and which drafted rows a node sees.
#pragma once

#include "params.cuh"

namespace hipml {

constexpr int kTreeNodes = 256;                      // most nodes of a slot's tree
constexpr int kTreeWords = kTreeNodes / 32;
constexpr int kTreeKeyTile = 64;                     // cache rows that runs are counted in
constexpr int kTreeBadTree = 41;                     // device status: a parent that is no earlier node, a token past the vocabulary
constexpr int kTreeBadPath = 42;                     // device status: a path that does not ascend within its tree

// Attention of drafted nodes. A CTA has `tile_rows` query rows of one KV head of one slot (row r of them is head r % group
// of node r / group) and one run of the slot's rows.
struct TreeParams {
    const int *pos;        // [slots] {prefix rows, prefix and drafted rows}
    const int *parents;    // [slots][nodes]
    const float *q;        // [slots][nodes][n_heads * head_dim]
    const unsigned char *k, *v;
    float *out;            // as q
    float *part_acc;       // [grid][tile_rows][head_dim]
    float *part_ml;        // [grid][tile_rows] {maximum in log2 units, sum}
    int4 *shares;          // [slots] {first CTA, runs, tiles}: how a slot was dealt out, for the fold
    int *status;
    int n_heads, n_kv, group, head_dim, stride, nodes, slots;
    int kv_dtype;          // 0 f32 [row][n_kv * head_dim], 1 q8_0, 2 q4_0 (head-major)
    float scale_log2;
    size_t slot_bytes;
    int grid, tile_rows;
    unsigned group_inverse;   // 65536 / group, rounded up: exact for groups of at most 8 and the rows of 256 nodes
    // row / group, of the rows of a slot (fewer than 65536 / 8)
    __device__ __forceinline__ int node_of(int row) const { return (int)((unsigned)row * group_inverse >> 16); }
};

// Prefix rows and live nodes of a slot; whatever `pos` says, no row lies past the cache and no node past `nodes`.
struct TreeSlot {
    int base, live;
};

// The CTAs that a launch gets: one round of the device, or as many as there are (slot, KV head, tile) triples at least.
// tree_part_bytes(...) of scratch hold the partials of all of them.
inline int tree_grid(int n_heads, int n_kv, int nodes, int slots, int tile_rows, int round) {
    const int group = n_heads / n_kv;
    const long long triples = (long long)slots * n_kv * (((long long)nodes * group + tile_rows - 1) / tile_rows);
    const long long rounds = (triples + round - 1) / round;
    const long long grid = (rounds < 1 ? 1 : rounds) * round;
    return grid > 0x7fffffff ? -1 : (int)grid;
}

#ifdef __CUDACC__

__device__ __forceinline__ TreeSlot tree_slot(const int *pos, int slot, int stride, int nodes) {
    const int from = __ldcg(pos + 2 * (size_t)slot), to = __ldcg(pos + 2 * (size_t)slot + 1);
    TreeSlot s;
    s.base = min(max(from, 0), stride);
    s.live = min(max(min(max(to, 0), stride) - s.base, 0), nodes);   // (of numbers that are not negative: no difference wraps)
    return s;
}

// One CTA's share: the query rows [tile * tile_rows, ...) of KV head kvh of a slot, over key tiles of run `run` of `runs`.
struct TreeItem {
    int slot, kvh, tile, run, runs;
    int base, live, quota;
    // the run's rows; no row past the slot's last is formed, which may be the largest int
    __device__ __forceinline__ int first_row() const { return run * quota * kTreeKeyTile; }
    __device__ __forceinline__ int end_row() const {
        return run + 1 < runs ? first_row() + quota * kTreeKeyTile : base + live;
    }
};

// The slots as a warp's lanes hold them: the first 32 stay in registers, so that the plan is one trip to memory.
// kRows: rows of a tile.
template <int kRows>
struct TreeSlots {
    const TreeParams &p;
    TreeSlot mine;
    __device__ __forceinline__ explicit TreeSlots(const TreeParams &params) : p(params), mine({0, 0}) {
        const int lane = threadIdx.x & 31;
        if (lane < p.slots) mine = tree_slot(p.pos, lane, p.stride, p.nodes);
    }
    __device__ __forceinline__ TreeSlot at(int s) const {   // s % 32 == lane
        return s < 32 ? mine : tree_slot(p.pos, s, p.stride, p.nodes);
    }
    static __device__ __forceinline__ unsigned keys(const TreeSlot &t) {   // key tiles
        return ((unsigned)(t.base + t.live) + kTreeKeyTile - 1) / kTreeKeyTile;
    }
    __device__ __forceinline__ unsigned tiles(const TreeSlot &t) const {   // of rows
        return (unsigned)(t.live * p.group + kRows - 1) / kRows;
    }
};

// Key tiles per run, the same for all: the fewest with which the runs fit the grid. Called by a whole warp. (One loop over
// the slots: this runs once, and every line of it comes through an empty instruction cache.)
template <int kRows>
__device__ __forceinline__ int tree_quota(const TreeParams &p, const TreeSlots<kRows> &slots) {
    const int lane = threadIdx.x & 31;
    const unsigned fit = (unsigned)p.grid / (unsigned)p.n_kv;   // runs per KV head
    // question 0: the tiles of all; then the runs that quota q makes
    unsigned lo = 1, hi = 0, q = 1;
#pragma unroll 1
    for (int asked = 0;; asked++) {
        unsigned runs = 0, rows = 0;
#pragma unroll 1
        for (int s = lane; s < p.slots; s += 32) {
            const TreeSlot t = slots.at(s);
            const unsigned r = slots.tiles(t);
            runs += r * ((slots.keys(t) + q - 1) / q);
            rows += r;
        }
        runs = __reduce_add_sync(0xffffffffu, runs);
        if (asked == 0) {   // (q was 1)
            rows = __reduce_add_sync(0xffffffffu, rows);
            if (runs <= fit) return 1;
            lo = (runs + fit - 1) / fit;
            // sum(rows * ceil(keys / q)) <= runs / q + rows; with one run each, every triple has its CTA
            hi = fit > rows ? (runs + fit - rows - 1) / (fit - rows) : ((unsigned)p.stride + kTreeKeyTile - 1) / kTreeKeyTile;
            q = lo;
            lo--;       // (does not fit; hi does)
            if (hi <= q) return (int)q;
            continue;
        }
        if (runs <= fit) hi = q; else lo = q;
        if (hi - lo <= 1) return (int)hi;
        q = asked == 1 ? q + 1 : lo + (hi - lo) / 2;   // (most often the least that may do, or the next, does)
        if (q >= hi) q = lo + (hi - lo) / 2;
    }
}

// CTA `cta`'s item (slot < 0: none); a slot's first CTA leaves its share for the fold. Called by a whole warp.
template <int kRows>
__device__ __forceinline__ TreeItem tree_item(const TreeParams &p, int cta) {
    const int lane = threadIdx.x & 31;
    const TreeSlots<kRows> slots(p);
    const int quota = tree_quota<kRows>(p, slots);
    TreeItem it;
    it.slot = -1;
    it.quota = quota;
    unsigned before = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < p.slots && it.slot < 0; s0 += 32) {
        TreeSlot t = {0, 0};
        if (s0 + lane < p.slots) t = slots.at(s0 + lane);
        const unsigned tiles = slots.tiles(t), runs = (slots.keys(t) + quota - 1) / (unsigned)quota;
        const unsigned mine = p.n_kv * tiles * runs;
        unsigned upto = mine;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, (unsigned)cta < before + upto);
        if (past) {
            const int at = __ffs(past) - 1;
            const unsigned first = before + __shfl_sync(0xffffffffu, upto - mine, at);
            it.slot = s0 + at;
            it.base = __shfl_sync(0xffffffffu, t.base, at);
            it.live = __shfl_sync(0xffffffffu, t.live, at);
            it.runs = (int)__shfl_sync(0xffffffffu, runs, at);
            const unsigned of_slot = __shfl_sync(0xffffffffu, tiles, at), in_slot = cta - first;
            const unsigned triple = in_slot / (unsigned)it.runs;
            it.run = (int)(in_slot - triple * it.runs);
            it.kvh = (int)(triple / of_slot);
            it.tile = (int)(triple - it.kvh * of_slot);
            if (in_slot == 0 && lane == 0) p.shares[it.slot] = make_int4(cta, it.runs, (int)of_slot, 0);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return it;
}

// Bits of the drafted rows that `node` sees, its own and those of its ancestors, into words[kTreeWords]. A parent that is no
// earlier node ends the walk (and is reported).
__device__ __forceinline__ void tree_ancestors(const int *parents, int node, unsigned *words, int *status) {
#pragma unroll 1
    for (int w = 0; w < kTreeWords; w++) words[w] = 0;
#pragma unroll 1
    for (int i = node; i >= 0;) {
        words[i >> 5] |= 1u << (i & 31);
        const int up = parents[i];
        if (up >= i || up < -1) {
            atomicCAS(status, 0, kTreeBadTree);
            break;
        }
        i = up;
    }
}
#endif

// attn_tree.cu: the CUDA-core kernel (any head size and alignment) and the fold of the runs.
int launch_tree_scalar(cudaStream_t stream, const TreeParams &p);
constexpr int kTreeScalarRows = 32;
// attn_tree_tc.cu: head_dim 256, caches (and slots) on 16 bytes.
int launch_tree_tc(cudaStream_t stream, const TreeParams &p);
constexpr int kTreeTcRows = 128;
int launch_tree_fold(cudaStream_t stream, const TreeParams &p);

// tree_verify.cu
constexpr int kVerifyVocab = 1 << 20;   // most tokens of a vocabulary
struct VerifyParams {
    const int *pos, *parents, *tokens;
    const float *target, *draft, *uniform;
    int *path, *count, *next;
    int *status;
    int nodes, slots, vocab;
    long long row_stride;
    int stride;            // rows of the cache that the nodes' rows lie in
};
int launch_tree_verify(cudaStream_t stream, const VerifyParams &p);

// kv_path.cu
constexpr int kPathLayers = 64;   // of one launch
struct PathParams {
    const int *pos, *path, *count;
    int *status;
    int n_kv, stride, nodes, which;   // which: 2 * layers caches
    long long slot_bytes;
    long long head_pitch, row_pitch;  // bytes from one KV head's row to the next head's, and to the next row
    int row_bytes;                    // of one KV head's row
    unsigned char *cache[2 * kPathLayers];
};
int launch_kv_path_keep(cudaStream_t stream, const PathParams &p, int slots);

}  // namespace hipml
