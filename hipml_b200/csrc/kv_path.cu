// The rows of an accepted path move together: in every cache of a step (K and V of all layers) row base + path[i] of a slot
// becomes row base + i, i < count. One launch for all of them; bytes are moved as they are, so every cache format is alike.
// No counterpart in the reference, whose drafts are chains and stay where they were appended.
//
// In place: a path's nodes ascend, so path[i] >= i and a row is a source only of itself or of a lower one. A CTA has one KV
// head's rows of one cache and slot and takes them in pieces, row after row: all sources of a piece are read before any of
// its rows is written, and no later source lies among them. A latency-bound launch: two trips to memory (the path, then the
// rows) and the stores; 16 layers, one slot, 70 KB.
#include "tree.cuh"

namespace hipml {

namespace {

constexpr int kThreads = 256, kEach = 8;

// grid (2 * layers * n_kv, slots). Word: the widest type that rows and pitches are whole numbers of.
template <class Word>
__global__ void __launch_bounds__(kThreads) kv_path_keep(const __grid_constant__ PathParams p) {
    __shared__ int s_path[kTreeNodes];
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x, slot = blockIdx.y;
    const int which = blockIdx.x / p.n_kv, head = blockIdx.x - which * p.n_kv;
    // (the path is fetched whole, beside its length: one trip to memory)
    static_assert(kThreads >= kTreeNodes, "a thread per node");
    int node = -1, before = -1;
    if (tid < p.nodes) {
        const int *const at = p.path + (size_t)slot * p.nodes + tid;
        node = __ldcg(at);
        if (tid > 0) before = __ldcg(at - 1);
    }
    const TreeSlot t = tree_slot(p.pos, slot, p.stride, p.nodes);
    const int kept = __ldcg(p.count + slot);
    const int count = t.live == 0 ? 0 : kept;   // (of an idle slot verification has left path and count as they were)
    bool bad = count < 0 || count > t.live;
    if (tid < count) {
        bad = bad || node <= before || node < 0 || node >= t.live;
        s_path[tid] = node;
    }
    if (__syncthreads_or(bad)) {   // the slot's rows stay as they are
        if (tid == 0) atomicCAS(p.status, 0, kTreeBadPath);
        return;
    }
    const int words = p.row_bytes / (int)sizeof(Word);
    unsigned char *const rows = p.cache[which] + slot * p.slot_bytes + head * p.head_pitch + (long long)t.base * p.row_pitch;
    auto word = [&](int row, int w) { return reinterpret_cast<Word *>(rows + row * p.row_pitch) + w; };
    const int all = count * words;
    for (int e0 = 0; e0 < all; e0 += kThreads * kEach) {
        Word x[kEach];
        int row[kEach], w[kEach];
#pragma unroll
        for (int j = 0; j < kEach; j++) {
            const int e = e0 + j * kThreads + tid;
            row[j] = e < all ? e / words : -1;
            w[j] = e - row[j] * words;
            if (row[j] >= 0 && s_path[row[j]] == row[j]) row[j] = -1;   // (already there)
            if (row[j] >= 0) x[j] = *word(s_path[row[j]], w[j]);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kEach; j++)
            if (row[j] >= 0) *word(row[j], w[j]) = x[j];
    }
}

}  // namespace

int launch_kv_path_keep(cudaStream_t stream, const PathParams &p, int slots) {
    size_t align = (size_t)p.row_bytes | (size_t)p.slot_bytes | (size_t)p.head_pitch | (size_t)p.row_pitch;
    for (int i = 0; i < p.which; i++) align |= reinterpret_cast<size_t>(p.cache[i]);
    const dim3 grid(p.which * p.n_kv, slots), block(kThreads);
    if ((align & 15) == 0) return launch_pdl(kv_path_keep<uint4>, grid, block, 0, stream, 1, p);
    if ((align & 3) == 0) return launch_pdl(kv_path_keep<unsigned>, grid, block, 0, stream, 1, p);
    return launch_pdl(kv_path_keep<unsigned short>, grid, block, 0, stream, 1, p);
}

}  // namespace hipml
