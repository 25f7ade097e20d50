// What the kernels of tree speculation share: their parameters, how the work of a launch is dealt out to its CTAs from
// lengths that only the device knows, and which drafted rows a node sees.
#pragma once

#include "params.cuh"

namespace hipml {

__host__ __device__ __forceinline__ int div_up_int(int a, int b) { return (a + b - 1) / b; }

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
    s.live = min(max(min(to, stride) - s.base, 0), nodes);
    return s;
}

// One CTA's share: the query rows [tile * tile_rows, ...) of KV head kvh of a slot, over key tiles of run `run` of `runs`.
struct TreeItem {
    int slot, kvh, tile, run, runs;
    int base, live, quota;
};

// The slots as a warp's lanes hold them: the first 32 stay in registers, so that the plan is one trip to memory.
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
};

// Key tiles per run, the same for all: the fewest with which the runs fit the grid. Called by a whole warp.
__device__ __forceinline__ int tree_quota(const TreeParams &p, const TreeSlots &slots) {
    const int lane = threadIdx.x & 31;
    auto each = [&](auto f) {   // sum over the slots of f(key tiles, row tiles)
        int n = 0;
        for (int s = lane; s < p.slots; s += 32) {
            const TreeSlot t = slots.at(s);
            n += f(div_up_int(t.base + t.live, kTreeKeyTile), div_up_int(t.live * p.group, p.tile_rows));
        }
        return (int)__reduce_add_sync(0xffffffffu, n);
    };
    const int fit = p.grid / p.n_kv;   // runs per KV head
    const int total = each([](int keys, int rows) { return keys * rows; });
    auto runs_at = [&](int q) { return each([&](int keys, int rows) { return rows * div_up_int(keys, q); }); };
    int lo = max(1, div_up_int(total, fit));
    if (runs_at(lo) <= fit) return lo;
    // sum(rows * ceil(keys / q)) <= total / q + few; with one run each, every triple has its CTA
    const int few = each([](int, int rows) { return rows; });
    int hi = fit > few ? div_up_int(total, fit - few) : div_up_int(p.stride, kTreeKeyTile);
    hi = max(hi, lo + 1);
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (runs_at(mid) <= fit) hi = mid; else lo = mid;
    }
    return hi;
}

__device__ __forceinline__ int tree_ctas(const TreeParams &p, const TreeSlot &t, int quota) {
    return p.n_kv * div_up_int(t.live * p.group, p.tile_rows) * div_up_int(t.base + t.live, kTreeKeyTile * quota);
}

// CTA `cta`'s item (slot < 0: none); a slot's first CTA leaves its share for the fold. Called by a whole warp.
__device__ __forceinline__ TreeItem tree_item(const TreeParams &p, int cta) {
    const int lane = threadIdx.x & 31;
    const TreeSlots slots(p);
    const int quota = tree_quota(p, slots);
    TreeItem it;
    it.slot = -1;
    it.quota = quota;
    int before = 0;
    for (int s0 = 0; s0 < p.slots && it.slot < 0; s0 += 32) {
        TreeSlot t = {0, 0};
        if (s0 + lane < p.slots) t = slots.at(s0 + lane);
        const int mine = tree_ctas(p, t, quota);
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, cta < before + upto);
        if (past) {
            const int at = __ffs(past) - 1;
            const int first = before + __shfl_sync(0xffffffffu, upto - mine, at);
            it.slot = s0 + at;
            it.base = __shfl_sync(0xffffffffu, t.base, at);
            it.live = __shfl_sync(0xffffffffu, t.live, at);
            it.runs = div_up_int(it.base + it.live, kTreeKeyTile * quota);
            const int in_slot = cta - first, tiles = div_up_int(it.live * p.group, p.tile_rows);
            const int triple = in_slot / it.runs;
            it.run = in_slot - triple * it.runs;
            it.kvh = triple / tiles;
            it.tile = triple - it.kvh * tiles;
            if (in_slot == 0 && lane == 0) p.shares[it.slot] = make_int4(cta, it.runs, tiles, 0);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return it;
}

// Bits of the drafted rows that `node` sees, its own and those of its ancestors, into words[kTreeWords]. A parent that is no
// earlier node ends the walk (and is reported).
__device__ __forceinline__ void tree_ancestors(const int *parents, int node, unsigned *words, int *status) {
    for (int w = 0; w < kTreeWords; w++) words[w] = 0;
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
