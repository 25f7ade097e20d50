// Which drafted nodes a step keeps, and the token that follows them, from the target's probabilities, the drafter's and
// given random numbers. The walk of a slot begins at node 0 (the last token of the sequence) with r = the target row of that
// node. The children of the node that was kept last are tried in order: child c with token x is kept where
//     u_c q(x) < r(x)            (q: the draft row of the parent; without draft rows q is 1 at x and 0 elsewhere),
// and r becomes the target row of c; a child that is not kept leaves
//     r <- max(r - q, 0) / Z,  Z its sum (r stays where Z is 0).
// Where no child is kept the next token is drawn from r: the first x whose running sum exceeds u_0 times the whole.
// Accepted tokens and the drawn one are distributed as the target's own (the drafter's errors cost speed only).
// No counterpart in the reference, which compares greedy tokens on the host (crates/hipml-model/src/gpu/spec.rs).
//
// A slot is one cluster of CTAs; each has a part of the vocabulary. What the walk asks of single tokens, r(x) and q(x) of
// every node, is fetched by all nodes at once in the beginning (one trip to memory instead of one per level); a rejected
// child costs one pass over the target and the draft row, all CTAs together, and the pass of the last rejection leaves the
// sums by which the next token is found (no rejection: one pass over the target row). Differences, sums and comparisons are
// in 64 bits: over 150,000 probabilities a 32-bit running sum moves some thousandth of the drawn tokens by one place. r of
// the second and later rejections is computed from the rows again, so nothing is kept per probability.
#include "sm100_ptx.cuh"
#include "tree.cuh"

namespace hipml {

namespace {

using namespace ptx;

constexpr int kCtas = 8, kThreads = 512, kWarps = kThreads / 32;
constexpr int kPiece = kThreads * 4;      // probabilities that a CTA takes at once
constexpr int kSegment = 128;             // of a warp: what the sums are kept of
constexpr int kSegments = kVerifyVocab / kCtas / kSegment;

// The rejections since a node was kept, by which what is left of its target row is computed.
struct Left {
    double inverse[kTreeNodes];   // one over the sum that rejection j left
    int token[kTreeNodes];        // of the child that was rejected
};

__device__ __forceinline__ double probability(float p) {   // what is no probability counts as 0
    return p > 0.0f && p < INFINITY ? (double)p : 0.0;
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__global__ void __launch_bounds__(kThreads) __cluster_dims__(kCtas, 1, 1) tree_verify(VerifyParams p) {
    __shared__ int s_parent[kTreeNodes], s_token[kTreeNodes];
    __shared__ float s_u[kTreeNodes], s_p[kTreeNodes], s_q[kTreeNodes];
    __shared__ Left s_left;
    __shared__ double s_segment[kSegments];   // of this CTA's part
    __shared__ double s_sum[2];               // this CTA's part of a pass, read by the others (the passes take turns)
    __shared__ double s_all[kCtas];
    __shared__ double s_warp[kWarps];
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank(), slot = blockIdx.x / kCtas;
    const TreeSlot t = tree_slot(p.pos, slot, 0x7fffffff, p.nodes);
    if (t.live == 0) return;   // (the whole cluster) nothing is written
    const size_t first = (size_t)slot * p.nodes;
    bool bad = false;
    for (int i = tid; i < t.live; i += kThreads) {
        int up = i == 0 ? -1 : p.parents[first + i], x = i == 0 ? 0 : p.tokens[first + i];
        if (up >= i || up < -1) bad = true, up = -1;
        if (x < 0 || x >= p.vocab) bad = true, up = -1;   // (is not reached)
        s_parent[i] = up;
        s_token[i] = x;
        s_u[i] = p.uniform[first + i];
        if (up >= 0) {
            const long long at = (long long)(first + up) * p.row_stride + x;
            s_p[i] = p.target[at];
            s_q[i] = p.draft ? p.draft[at] : 1.0f;
        }
    }
    if (bad && rank == 0) atomicCAS(p.status, 0, kTreeBadTree);
    __syncthreads();

    // this CTA's part of the vocabulary, in whole pieces of four
    const int quads = (p.vocab + 3) / 4, part = (quads + kCtas - 1) / kCtas * 4;
    const int v0 = min(rank * part, p.vocab), v1 = min(v0 + part, p.vocab);
    const bool wide = ((reinterpret_cast<size_t>(p.target) | reinterpret_cast<size_t>(p.draft)) & 15) == 0 &&
                      (p.row_stride & 3) == 0;
    int here = 0;   // the node that was kept last

    // what is left of p.target's row `here` at x, before the division by the last sum; `tried` rejections
    auto left_of = [&](double r, double q, int x, int tried) {
        if (p.draft) {
            for (int j = 0; j < tried; j++) r = fmax((j == 0 ? r : r * s_left.inverse[j - 1]) - q, 0.0);
        } else {
            for (int j = 0; j < tried; j++)
                if (s_left.token[j] == x) r = 0.0;
        }
        return r;
    };
    // four probabilities from x on
    auto load4 = [&](const float *row, int x, float (&v)[4]) {
        if (wide && x + 4 <= v1) {
            const float4 w = __ldg(reinterpret_cast<const float4 *>(row + x));
            v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = x + e < v1 ? __ldg(row + x + e) : 0.0f;
        }
    };
    // One pass over the row: the sums of this CTA's segments, and the sum of all (in the order of the CTAs, everywhere the
    // same bits).
    int passes = 0;
    auto pass = [&](int tried) {
        const float *const target = p.target + (long long)(first + here) * p.row_stride;
        const float *const draft = p.draft ? p.draft + (long long)(first + here) * p.row_stride : nullptr;
        double mine = 0.0;
        for (int x0 = v0, n = 0; x0 < v1; x0 += kPiece, n++) {
            const int x = x0 + 4 * tid;
            float a[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (x < v1) {
                load4(target, x, a);
                if (draft && tried > 0) load4(draft, x, b);
            }
            double sum = 0.0;
#pragma unroll
            for (int e = 0; e < 4; e++) sum += left_of(probability(a[e]), probability(b[e]), x + e, tried);
            sum = warp_sum_f64(sum);
            if (lane == 0) s_segment[n * kWarps + warp] = sum;
            mine += sum;
        }
        if (lane == 0) s_warp[warp] = mine;
        __syncthreads();
        if (tid == 0) {
            double all = 0.0;
            for (int w = 0; w < kWarps; w++) all += s_warp[w];
            s_sum[passes & 1] = all;
        }
        cluster_sync_all();
        if (tid < kCtas) {
            const unsigned at = map_to_cta(smem_u32(&s_sum[passes & 1]), tid);
            double v;
            asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
            s_all[tid] = v;
        }
        __syncthreads();
        passes++;
        double all = 0.0;
        for (int c = 0; c < kCtas; c++) all += s_all[c];
        return all;
    };

    // The walk, the same in every thread. An accepted child lies behind its parent and its siblings are tried in order, so
    // one run over the nodes meets them all.
    int count = 1, tried = 0;
    bool summed = false;      // the last pass was over what is left now
    double whole = 1.0;       // what r is divided by
    if (rank == 0 && tid == 0) p.path[first] = 0;
    for (int i = 1; i < t.live; i++) {
        if (s_parent[i] != here) continue;
        const int x = s_token[i];
        const double q = p.draft ? probability(s_q[i]) : 1.0;
        const double r = left_of(probability(s_p[i]), q, x, tried);
        if ((double)s_u[i] * q * whole < r) {
            here = i;
            if (rank == 0 && tid == 0) p.path[first + count] = i;
            count++;
            tried = 0;
            whole = 1.0;
            summed = false;
            continue;
        }
        __syncthreads();
        if (tid == 0) {
            s_left.token[tried] = x;
            if (tried > 0) s_left.inverse[tried - 1] = 1.0 / whole;
        }
        __syncthreads();
        const double sum = pass(tried + 1);
        if (sum > 0.0) {
            tried++;
            whole = sum;
            summed = true;
        } else {
            summed = false;   // (the segments' sums are of nothing)
        }
    }
    if (!summed) whole = pass(tried);
    if (rank == 0) {
        for (int i = count + tid; i < p.nodes; i += kThreads) p.path[first + i] = -1;
        if (tid == 0) p.count[slot] = count;
    }
    // The next token: the part, the segment in it, the place in that.
    const double bar = (double)s_u[0] * whole;
    if (!(whole > 0.0)) {
        if (rank == 0 && tid == 0) p.next[slot] = -1;
    } else {
        double before = 0.0;
        int owner = -1, last = 0;   // last: the part that ends the mass, where rounding leaves no running sum above the bar
        double upto = 0.0, before_last = 0.0;
        for (int c = 0; c < kCtas; c++) {
            if (s_all[c] > 0.0) {
                last = c;
                before_last = upto;
            }
            if (owner < 0 && upto + s_all[c] > bar && s_all[c] > 0.0) {
                owner = c;
                before = upto;
            }
            upto += s_all[c];
        }
        const bool end = owner < 0;   // the last token that has mass
        if (end) {
            owner = last;
            before = before_last;
        }
        if (rank == owner && warp == 0) {
            const int segments = (v1 - v0 + kSegment - 1) / kSegment;
            int at = -1, at_last = 0;
            double start = before, start_last = before;
            for (int s0 = 0; s0 < segments; s0 += 32) {
                const double mine = s0 + lane < segments ? s_segment[s0 + lane] : 0.0;
                double incl = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double w = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += w;
                }
                const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
                const unsigned past = end ? 0 : __ballot_sync(0xffffffffu, mine > 0.0 && before + incl > bar);
                if (past && at < 0) {
                    const int l = __ffs(past) - 1;
                    at = s0 + l;
                    start = before + __shfl_sync(0xffffffffu, incl - mine, l);
                }
                if (some) {
                    const int l = 31 - __clz(some);
                    at_last = s0 + l;
                    start_last = before + __shfl_sync(0xffffffffu, incl - mine, l);
                }
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (at < 0) {
                at = at_last;
                start = start_last;
            }
            const float *const target = p.target + (long long)(first + here) * p.row_stride;
            const float *const draft = p.draft ? p.draft + (long long)(first + here) * p.row_stride : nullptr;
            const int x = v0 + at * kSegment + 4 * lane;
            float a[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (x < v1) {
                load4(target, x, a);
                if (draft && tried > 0) load4(draft, x, b);
            }
            double w[4], incl = 0.0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                w[e] = left_of(probability(a[e]), probability(b[e]), x + e, tried);
                incl += w[e];
            }
            const double mine = incl;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            double c = start + incl - mine;
            int found = 0x7fffffff, ends = -1;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                c += w[e];
                if (w[e] > 0.0) {
                    ends = x + e;
                    if (c > bar && found == 0x7fffffff) found = x + e;
                }
            }
            found = __reduce_min_sync(0xffffffffu, found);
            ends = __reduce_max_sync(0xffffffffu, ends);
            if (lane == 0) p.next[slot] = !end && found != 0x7fffffff ? found : ends;
        }
    }
    cluster_sync_all();   // no CTA leaves while another may still read its sum
}

}  // namespace

int launch_tree_verify(cudaStream_t stream, const VerifyParams &p) {
    return launch_pdl(tree_verify, dim3(p.slots * kCtas), dim3(kThreads), 0, stream, 1, p);
}

}  // namespace hipml
