// Attention of a tree of drafted tokens over a cache (f32, q8_0, q4_0; several slots), on the CUDA cores, and the fold of
// the runs' partials. For node i of a slot, with `base` prefix rows and the drafted rows behind them:
//     out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(scale log2(e) q_i . k_j - m_i),
//     j over [0, base) and base + {i and its ancestors}.
// No counterpart in the reference, whose verify columns are a chain (crates/hipml-kernels/src/launch_kv.rs:320-400).
//
// This kernel takes the head sizes and alignments that the tensor-core kernel does not. A CTA has 32 query rows, four to a
// warp, and walks its run 32 cache rows at a time: the tile is dequantised once to f32 in shared memory for all of them
// (scores: lane = cache row; values: lane = dims), so the cache is read once per 32 query rows and the products are plain
// f32 FMAs, which bound it.
#include <atomic>

#include "q8_pack.cuh"
#include "tree.cuh"

namespace hipml {

namespace {

constexpr int kRows = kTreeScalarRows, kWarpRows = 4, kWarps = 8, kKeys = 32;

// x, or not a number where it is not finite: a key of -infinity would leave a row with a weight of 0. (Looked at here, once per
// value or scale; where a score is -infinity it cost 8 % of 12 nodes at 60,000 rows, heads of 64.)
__device__ __forceinline__ float finite_or_nan(float x) { return fabsf(x) < INFINITY ? x : __int_as_float(0x7fffffff); }

// Values [32 * blk, +32) of one KV head's cache row, as f32 into dst[0 .. 31]; rows that are not finite are not numbers there.
__device__ __forceinline__ void load_block(const TreeParams &p, const unsigned char *cache, int kvh, int row, int blk,
                                           float *dst) {
    if (p.kv_dtype == 0) {
        const float *src = reinterpret_cast<const float *>(cache) + ((size_t)row * p.n_kv + kvh) * p.head_dim + 32 * blk;
#pragma unroll
        for (int j = 0; j < 32; j++) dst[j] = finite_or_nan(src[j]);
    } else if (p.kv_dtype == 1) {
        const unsigned short *src = reinterpret_cast<const unsigned short *>(
            cache + q8_row_offset(kvh, p.stride, row, p.head_dim) + (size_t)blk * kQ8BlockBytes);
        const float d = finite_or_nan(half_bits_to_float(src[0]));
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const unsigned short w = src[1 + j];
            dst[2 * j] = d * (float)(signed char)(w & 0xff);
            dst[2 * j + 1] = d * (float)(signed char)(w >> 8);
        }
    } else {
        const unsigned short *src = reinterpret_cast<const unsigned short *>(
            cache + q4_row_offset(kvh, p.stride, row, p.head_dim) + (size_t)blk * kQ4BlockBytes);
        const float d = finite_or_nan(half_bits_to_float(src[0]));
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const unsigned short w = src[1 + j];
            dst[2 * j] = d * ((float)(w & 15) - 8.0f);
            dst[2 * j + 1] = d * ((float)((w >> 8) & 15) - 8.0f);
            dst[2 * j + 16] = d * ((float)((w >> 4) & 15) - 8.0f);
            dst[2 * j + 17] = d * ((float)(w >> 12) - 8.0f);
        }
    }
}

// grid as tree_grid, block 256, kB = head_dim / 32.
template <int kB>
__global__ void __launch_bounds__(256) attn_tree_scalar(TreeParams p) {
    constexpr int kD = 32 * kB, kPitch = kD + 1;
    extern __shared__ float smem[];
    float *const ks = smem, *const vs = ks + kKeys * kPitch, *const qs = vs + kKeys * kPitch;
    __shared__ TreeItem s_item;
    __shared__ int s_parents[kTreeNodes];
    __shared__ unsigned s_sees[kRows][kTreeWords];
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (warp == 0) {
        const TreeItem it = tree_item<kRows>(p, blockIdx.x);
        if (lane == 0) s_item = it;
    }
    __syncthreads();
    const TreeItem it = s_item;
    if (it.slot < 0) return;
    const int rows = min(kRows, it.live * p.group - it.tile * kRows);
    const unsigned lo = it.first_row(), hi = it.end_row();   // (k0 + 31 below may be past the largest int)
    for (int i = tid; i < it.live; i += 256) s_parents[i] = p.parents[(size_t)it.slot * p.nodes + i];
    const size_t slot_row = (size_t)it.slot * p.nodes;
    // a row of the tile as a row of q and out, in heads
    auto head_row = [&](int r) {
        const int at = it.tile * kRows + r, node = p.node_of(at);
        return (slot_row + node) * p.n_heads + it.kvh * p.group + (at - node * p.group);
    };
    for (int i = tid; i < kRows * kD; i += 256) {
        const int r = i / kD;
        qs[i] = r < rows ? p.q[head_row(r) * kD + (i - r * kD)] * p.scale_log2 : 0.0f;
    }
    __syncthreads();
    if (tid < rows) {
        tree_ancestors(s_parents, p.node_of(it.tile * kRows + tid), s_sees[tid], p.status);
    }
    const unsigned char *const kc = p.k + (size_t)it.slot * p.slot_bytes, *const vc = p.v + (size_t)it.slot * p.slot_bytes;
    float acc[kWarpRows][kB], m[kWarpRows], l[kWarpRows];
#pragma unroll
    for (int a = 0; a < kWarpRows; a++) {
        m[a] = -INFINITY;
        l[a] = 0.0f;
#pragma unroll
        for (int b = 0; b < kB; b++) acc[a][b] = 0.0f;
    }
    for (unsigned k0 = lo; k0 < hi; k0 += kKeys) {
        __syncthreads();
        for (int i = warp; i < 2 * kB; i += kWarps) {   // lane = cache row: the stores fall into different banks
            const int blk = i % kB;
            float *const dst = (i < kB ? ks : vs) + lane * kPitch + 32 * blk;
            if (k0 + lane < hi) {
                load_block(p, i < kB ? kc : vc, it.kvh, k0 + lane, blk, dst);
            } else {
#pragma unroll
                for (int j = 0; j < 32; j++) dst[j] = 0.0f;
            }
        }
        __syncthreads();
        float s[kWarpRows] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float *const krow = ks + lane * kPitch, *const qrow = qs + warp * kWarpRows * kD;
#pragma unroll 4
        for (int d = 0; d < kD; d += 4) {
            const float k0v = krow[d], k1v = krow[d + 1], k2v = krow[d + 2], k3v = krow[d + 3];
#pragma unroll
            for (int a = 0; a < kWarpRows; a++) {
                const float4 x = *reinterpret_cast<const float4 *>(qrow + a * kD + d);
                s[a] = fmaf(x.x, k0v, fmaf(x.y, k1v, fmaf(x.z, k2v, fmaf(x.w, k3v, s[a]))));
            }
        }
        unsigned seen[kWarpRows];   // bit j: the row sees cache row k0 + j
#pragma unroll
        for (int a = 0; a < kWarpRows; a++) {
            const int r = warp * kWarpRows + a, drafted = (int)(k0 + lane - it.base);
            bool sees = r < rows && k0 + lane < hi;
            if (sees && drafted >= 0) sees = s_sees[r][drafted >> 5] >> (drafted & 31) & 1;
            seen[a] = __ballot_sync(0xffffffffu, sees);
            // (a row that sees nothing of these keeps what it has: -inf - -inf must not be formed)
            const float mine = sees ? s[a] : -INFINITY;
            const float m_new = fmaxf(m[a], warp_max(mine));
            const float ref = m_new == -INFINITY ? 0.0f : m_new;
            const float corr = exp2f(m[a] - ref);
            s[a] = sees ? exp2f(mine - ref) : 0.0f;
            l[a] = l[a] * corr + warp_sum(s[a]);
            m[a] = m_new;
#pragma unroll
            for (int b = 0; b < kB; b++) acc[a][b] *= corr;
        }
#pragma unroll 4
        for (int j = 0; j < kKeys; j++) {
            float x[kB];
#pragma unroll
            for (int b = 0; b < kB; b++) x[b] = vs[j * kPitch + 32 * b + lane];
#pragma unroll
            for (int a = 0; a < kWarpRows; a++) {
                const float w = __shfl_sync(0xffffffffu, s[a], j);
                if (seen[a] >> j & 1) {   // what a row does not see may hold anything
#pragma unroll
                    for (int b = 0; b < kB; b++) acc[a][b] = fmaf(w, x[b], acc[a][b]);
                }
            }
        }
    }
#pragma unroll
    for (int a = 0; a < kWarpRows; a++) {
        const int r = warp * kWarpRows + a;
        if (r >= rows) break;
        const bool whole = it.runs == 1;
        const size_t part = (size_t)blockIdx.x * kRows + r;
        float *const dst = whole ? p.out + head_row(r) * kD : p.part_acc + part * kD;
        const float inv = whole ? 1.0f / l[a] : 1.0f;
#pragma unroll
        for (int b = 0; b < kB; b++) dst[32 * b + lane] = acc[a][b] * inv;
        if (!whole && lane == 0) {
            // (a maximum leaves out what is not a number; -infinity alone would be a run of which the row sees nothing)
            p.part_ml[2 * part] = l[a] == l[a] ? m[a] : 0.0f;
            p.part_ml[2 * part + 1] = l[a];
        }
    }
}

// The runs of a query row, folded: grid (n_heads * nodes, slots), 256 threads. A column of four dims has 1024 / head_dim
// threads, which take the runs in turn, relative to a maximum of their own (so that a run's row and its pair are one trip
// to memory, after that for the slot's share), and meet in shared memory.
__global__ void __launch_bounds__(256) attn_tree_fold(TreeParams p) {
    __shared__ float s_max[256], s_den[256];
    __shared__ float4 s_sum[256];
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x;
    const int slot = blockIdx.y, node = blockIdx.x / p.n_heads, head = blockIdx.x - node * p.n_heads;
    const int4 share = __ldcg(p.shares + slot);
    const TreeSlot t = tree_slot(p.pos, slot, p.stride, p.nodes);
    const int runs = share.y;
    if (node >= t.live || runs == 1) return;   // (one run has written the row itself)
    const int kvh = head / p.group, at = node * p.group + head - kvh * p.group;
    const int tile = at / p.tile_rows, r = at - tile * p.tile_rows;
    const size_t first = (size_t)share.x + (size_t)(kvh * share.z + tile) * runs;
    const int cols = p.head_dim / 4, groups = 256 / cols;
    const int col = tid % cols, g = tid / cols;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float den = 0.0f, big = -INFINITY;
    if (g < groups) {
        const float2 *const ml = reinterpret_cast<const float2 *>(p.part_ml) + first * p.tile_rows + r;
        const float4 *const acc = reinterpret_cast<const float4 *>(p.part_acc + (first * p.tile_rows + r) * p.head_dim) + col;
        const size_t step = (size_t)p.tile_rows * cols;
        constexpr int kAtOnce = 5;
        for (int j0 = g; j0 < runs; j0 += groups * kAtOnce) {
            float2 x[kAtOnce];
            float4 a[kAtOnce];
            float most = big;
#pragma unroll
            for (int k = 0; k < kAtOnce; k++) {
                const int j = j0 + k * groups;
                x[k] = make_float2(-INFINITY, 0.0f);
                if (j < runs) {
                    x[k] = __ldcg(ml + (size_t)j * p.tile_rows);
                    a[k] = __ldcg(acc + (size_t)j * step);
                }
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; k++) most = fmaxf(most, x[k].x);
            const float corr = big == -INFINITY ? 0.0f : exp2f(big - most);
            sum.x *= corr;
            sum.y *= corr;
            sum.z *= corr;
            sum.w *= corr;
            den *= corr;
            big = most;
#pragma unroll
            for (int k = 0; k < kAtOnce; k++) {
                if (x[k].x == -INFINITY) continue;   // (no run, or one of which the row sees nothing)
                const float w = exp2f(x[k].x - big);
                sum.x = fmaf(a[k].x, w, sum.x);
                sum.y = fmaf(a[k].y, w, sum.y);
                sum.z = fmaf(a[k].z, w, sum.z);
                sum.w = fmaf(a[k].w, w, sum.w);
                den = fmaf(x[k].y, w, den);
            }
        }
    }
    s_max[tid] = big;
    s_sum[tid] = sum;
    s_den[tid] = den;
    __syncthreads();
    if (g == 0) {
        for (int i = 1; i < groups; i++) big = fmaxf(big, s_max[i * cols + col]);
        sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        den = 0.0f;
        for (int i = 0; i < groups; i++) {
            const float m = s_max[i * cols + col];
            if (m == -INFINITY) continue;
            const float w = exp2f(m - big);
            const float4 a = s_sum[i * cols + col];
            sum.x = fmaf(a.x, w, sum.x);
            sum.y = fmaf(a.y, w, sum.y);
            sum.z = fmaf(a.z, w, sum.z);
            sum.w = fmaf(a.w, w, sum.w);
            den = fmaf(s_den[i * cols + col], w, den);
        }
        const float inv = 1.0f / den;
        reinterpret_cast<float4 *>(p.out + (((size_t)slot * p.nodes + node) * p.n_heads + head) * p.head_dim)[col] =
            make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
    }
}

template <int kB>
int launch_scalar(cudaStream_t stream, const TreeParams &p) {
    constexpr int kD = 32 * kB;
    constexpr size_t kNeed = (2 * (size_t)kKeys * (kD + 1) + (size_t)kRows * kD) * sizeof(float);
    // Two CTAs to an SM and no more: launches start early, while others' CTAs are there, and then the few that have work came
    // together on a few SMs (12 nodes of eight heads of 64 over 1,000 rows, calls in a row: 30.5 us).
    constexpr size_t kSmem = kNeed > 80 * 1024 ? kNeed : 80 * 1024;
    static std::atomic<bool> configured[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev].load()) {
        const cudaError_t e = cudaFuncSetAttribute(attn_tree_scalar<kB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) configured[dev].store(true);
    }
    return launch_pdl(attn_tree_scalar<kB>, dim3(p.grid), dim3(256), kSmem, stream, 1, p);
}

}  // namespace

int launch_tree_scalar(cudaStream_t stream, const TreeParams &p) {
    switch (p.head_dim / 32) {
        case 1: return launch_scalar<1>(stream, p);
        case 2: return launch_scalar<2>(stream, p);
        case 3: return launch_scalar<3>(stream, p);
        case 4: return launch_scalar<4>(stream, p);
        case 5: return launch_scalar<5>(stream, p);
        case 6: return launch_scalar<6>(stream, p);
        case 7: return launch_scalar<7>(stream, p);
        default: return launch_scalar<8>(stream, p);
    }
}

int launch_tree_fold(cudaStream_t stream, const TreeParams &p) {
    return launch_pdl(attn_tree_fold, dim3(p.n_heads * p.nodes, p.slots), dim3(256), 0, stream, 1, p);
}

}  // namespace hipml
