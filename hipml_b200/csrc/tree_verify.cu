// Which drafted nodes a step keeps, and the token that follows them, from the target's probabilities, the drafter's and
// given random numbers. The walk of a slot begins at node 0 (the last token of the sequence) with r = the target row of that
// node. The children of the node that was kept last are tried in order: child c with token x is kept where
//     u_c q(x) < r(x)            (q: the draft row of the parent; without draft rows q is 1 at x and 0 elsewhere),
// and r becomes the target row of c; a child that is not kept leaves
//     r <- max(r - q, 0) / Z,  Z its sum (r stays where Z is 0).
// Where no child is kept the next token is drawn from r: the first x whose running sum exceeds u_0 times the whole.
// Accepted tokens and the drawn one are distributed as the target's own (the drafter's errors cost speed only): with draft
// rows if siblings were drawn from their parent's row independently of one another, without them however they were chosen.
// No counterpart in the reference, which compares greedy tokens on the host (crates/hipml-model/src/gpu/spec.rs).
//
// A slot is one cluster of CTAs; each has a part of the vocabulary, each warp a run of that. What the walk asks of single
// tokens, r(x) and q(x) of every node, is fetched by all nodes at once in the beginning (one trip to memory instead of one
// per level). A rejected child costs one pass over the target and the draft row, all CTAs together; without draft rows only
// the first one of a node does: it leaves out the tokens of all its children, what was not tried yet is added back, and if
// the walk ends there these are the sums that it needs. The sums of the last pass are those by which the next token is found.
// Differences, sums and comparisons are in 64 bits: over 150,000 probabilities a 32-bit running sum moves some thousandth of
// the drawn tokens by one place. r after the second and later rejections is computed from the rows again, so nothing is kept
// per probability.
#include <atomic>

#include "sm100_ptx.cuh"
#include "tree.cuh"

namespace hipml {

namespace {

using namespace ptx;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kAtOnce = 8;                // a lane's probabilities that are on their way together

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

// The sum of a few non-negative f32 values, with their rounding errors beside it; sums of more go on in 64 bits. The errors
// are exact and at most 2^-24 of the sum's power of two for each add; what is lost is the rounding of their own running sum,
// half a last place of 2, 4, 4 and four times 8 of that unit: 21 * 2^-48 of the sum for eight values. Differences come with
// errors of their own, at most as much as two more such units for all of them: 21 * 2^-48 for four of them (six roundings of
// 2^-24 of a unit each before they meet, then sums of four, five and six). With the sums in 64 bits less than 2^-43 of the
// whole is lost, whatever the vocabulary. (One such sum for all of a lane's values lost 2^-38 of rows of 2^20 tokens.)
struct LongSum {
    float hi = 0.0f, lo = 0.0f;
    __device__ __forceinline__ void add(float x, float error) {
        const float s = hi + x, b = s - hi;
        lo += ((hi - (s - b)) + (x - b)) + error;
        hi = s;
    }
    __device__ __forceinline__ void move_to(double &sum) {
        sum += (double)hi + (double)lo;
        hi = lo = 0.0f;
    }
};

// grid slots * kCtas, clusters of kCtas.
template <int kCtas>
__global__ void __launch_bounds__(kThreads, 2) tree_verify(VerifyParams p) {
    __shared__ int s_parent[kTreeNodes], s_token[kTreeNodes];
    __shared__ float s_u[kTreeNodes], s_p[kTreeNodes], s_q[kTreeNodes];
    __shared__ Left s_left;
    // without draft rows: a child's probability where its token is first tried, else 0; the sum of those of the children behind
    __shared__ float s_c[kTreeNodes];
    __shared__ double s_after[kTreeNodes];
    __shared__ double s_sum[2];               // this CTA's part of a pass, read by the others (the passes take turns)
    __shared__ double s_all[kCtas];           // the sums of the parts
    __shared__ double s_warp[kWarps];         // of this part, by warp
    __shared__ double s_segment[kWarps];
    static_assert(kThreads >= kTreeNodes, "a thread per node");
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank(), slot = blockIdx.x / kCtas;
    const size_t first = (size_t)slot * p.nodes;
    // (a thread per node, dead ones too: the slot's length comes with the same trip to memory)
    int up = -1, x_of = 0;
    if (tid < p.nodes) {
        up = tid == 0 ? -1 : __ldcg(p.parents + first + tid);
        x_of = tid == 0 ? 0 : __ldcg(p.tokens + first + tid);
        s_u[tid] = __ldcg(p.uniform + first + tid);
    }
    const TreeSlot t = tree_slot(p.pos, slot, p.stride, p.nodes);
    if (t.live == 0) return;   // (the whole cluster) nothing is written
    if (tid < t.live) {
        if (up >= tid || up < -1 || x_of < 0 || x_of >= p.vocab) {
            if (rank == 0) atomicCAS(p.status, 0, kTreeBadTree);
            up = -1;           // (is not reached)
            x_of = 0;
        }
        s_parent[tid] = up;
        s_token[tid] = x_of;
        if (up >= 0) {
            const long long at = (long long)(first + up) * p.row_stride + x_of;
            s_p[tid] = __ldg(p.target + at);
            s_q[tid] = p.draft ? __ldg(p.draft + at) : 1.0f;
        }
    }
    __syncthreads();

    // this CTA's part of the vocabulary and the warps' runs of it (rows may lie anywhere: a lane loads single values)
    const int run = (p.vocab + kCtas * kWarps - 1) / (kCtas * kWarps), part = run * kWarps;
    const int v0 = min(rank * part, p.vocab), v1 = min(v0 + part, p.vocab);
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
    // One pass over the row: the sums of the warps' runs, and the sum of all (everywhere the same bits).
    int passes = 0;
    auto pass = [&](int tried) {
        const float *const target = p.target + (long long)(first + here) * p.row_stride;
        const float *const draft = p.draft && tried > 0 ? p.draft + (long long)(first + here) * p.row_stride : nullptr;
        const int w0 = min(v0 + warp * run, v1), w1 = min(w0 + run, v1);
        // Most often what is left is p or max(p - q, 0): in f32 with the rounding error beside it, which is as exact here and
        // an eighth of the instructions in 64 bits. (The loops are loops: this code runs once or twice a launch, and its
        // lines come from beyond the instruction cache: unrolled in 64 bits 8 nodes of 151,936 took 30 us, so 10. Sixteen
        // values at once take 80 registers, which leaves an SM one CTA: 32 slots of 8 nodes 62 us, with eight 33.)
        double sum = 0.0;
        if (!p.draft || tried <= 1) {
            LongSum s;
#pragma unroll 1
            for (int x0 = w0 + lane; x0 < w1; x0 += 32 * kAtOnce) {
                float a[kAtOnce], b[kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; k++) {
                    const int x = x0 + 32 * k;
                    a[k] = x < w1 ? __ldg(target + x) : 0.0f;
                    b[k] = draft && x < w1 ? __ldg(draft + x) : 0.0f;
                }
                if (!p.draft) {   // what was rejected is no longer there
#pragma unroll 1
                    for (int j = 0; j < tried; j++) {
                        const int gone = s_left.token[j] - x0;
                        if (gone < -lane || gone >= 32 * kAtOnce - lane) continue;   // (the same in every lane)
#pragma unroll
                        for (int k = 0; k < kAtOnce; k++)
                            if (gone == 32 * k) a[k] = 0.0f;
                    }
                }
#pragma unroll
                for (int k = 0; k < kAtOnce; k++) {   // as probability(): below infinity's bits, which every negative is above
                    a[k] = __float_as_uint(a[k]) < 0x7f800000u ? a[k] : 0.0f;
                    b[k] = __float_as_uint(b[k]) < 0x7f800000u ? b[k] : 0.0f;
                }
                static_assert(kAtOnce == 8, "eight values, or two times four differences, to a sum");
                if (!draft) {
#pragma unroll
                    for (int k = 0; k < kAtOnce; k++) s.add(a[k], 0.0f);
                } else {
#pragma unroll
                    for (int k = 0; k < kAtOnce; k++) {
                        const float d = a[k] - b[k], e = d - a[k];
                        if (d > 0.0f) s.add(d, (a[k] - (d - e)) - (b[k] + e));
                        if (k == kAtOnce / 2 - 1) s.move_to(sum);
                    }
                }
                s.move_to(sum);
            }
        } else {
            constexpr int kFew = 4;
#pragma unroll 1
            for (int x0 = w0 + lane; x0 < w1; x0 += 32 * kFew) {
                float a[kFew], b[kFew];
#pragma unroll
                for (int k = 0; k < kFew; k++) {
                    const int x = x0 + 32 * k;
                    a[k] = x < w1 ? __ldg(target + x) : 0.0f;
                    b[k] = x < w1 ? __ldg(draft + x) : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < kFew; k++) sum += left_of(probability(a[k]), probability(b[k]), x0 + 32 * k, tried);
            }
        }
        sum = warp_sum_f64(sum);
        if (lane == 0) s_warp[warp] = sum;
        __syncthreads();
        if (warp == 0) {
            const double all = warp_sum_f64(lane < kWarps ? s_warp[lane] : 0.0);
            if (lane == 0) s_sum[passes & 1] = all;
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
        return warp_sum_f64(lane < kCtas ? s_all[lane] : 0.0);
    };

    // The walk, the same in every thread. An accepted child lies behind its parent and its siblings are tried in order, so
    // one run over the nodes meets them all.
    int count = 1, tried = 0;
    int known = -1;           // rejections that the sums of the last pass have in them
    bool apart = false;       // without draft rows: the last pass left out the tokens of all children, and
    double others = 0.0;      // this is its sum
    bool plain = p.draft;     // a rejection is a pass
    double whole = 1.0;       // what r is divided by
    if (rank == 0 && tid == 0) p.path[first] = 0;
    for (int i = 1; i < t.live; i++) {
        if (s_parent[i] != here) continue;
        const int x = s_token[i];
        const double q = p.draft ? probability(s_q[i]) : 1.0;
        const double r = apart ? (double)s_c[i] : left_of(probability(s_p[i]), q, x, tried);
        if ((double)s_u[i] * q * whole < r) {
            here = i;
            if (rank == 0 && tid == 0) p.path[first + count] = i;
            count++;
            tried = 0;
            whole = 1.0;
            apart = false;
            plain = p.draft;
            known = -1;
            continue;
        }
        __syncthreads();
        if (!plain && !apart) {
            // the children, in order: their tokens, their own part of the mass, that of those behind them
            const bool child = tid < t.live && s_parent[tid] == here;
            const int kids = __syncthreads_count(child);
            if (child) {
                int before = 0;
                bool again = false;
                for (int k = here + 1; k < tid; k++) {
                    if (s_parent[k] != here) continue;
                    before++;
                    again = again || s_token[k] == s_token[tid];
                }
                s_left.token[before] = s_token[tid];
                s_c[tid] = again ? 0.0f : (float)probability(s_p[tid]);
            }
            __syncthreads();
            if (child) {
                double after = 0.0;
                for (int k = t.live - 1; k > tid; k--)
                    if (s_parent[k] == here) after += (double)s_c[k];
                s_after[tid] = after;
            }
            others = pass(kids);
            apart = true;
            known = tried = kids;
        }
        if (apart) {
            const double sum = others + s_after[i];
            if (sum > 0.0) {
                whole = sum;
                continue;
            }
            // Nothing would be left: r stays what it was before this child, the mass of this child's token alone. (From here on
            // as with draft rows.)
            apart = false;
            plain = true;
            known = -1;
            tried = 0;
            for (int k = here + 1; k < i; k++) tried += s_parent[k] == here;
            continue;
        }
        if (tid == 0) {
            s_left.token[tried] = x;
            if (tried > 0) s_left.inverse[tried - 1] = 1.0 / whole;
        }
        __syncthreads();
        const double sum = pass(tried + 1);
        known = sum > 0.0 ? tried + 1 : -1;
        if (sum > 0.0) {
            tried++;
            whole = sum;
        }
    }
    if (known != tried) whole = pass(tried);
    if (rank == 0) {
        for (int i = count + tid; i < p.nodes; i += kThreads) p.path[first + i] = -1;
        if (tid == 0) p.count[slot] = count;
    }
    // The next token: the part, the segment in it, the place in that.
    const double bar = (double)s_u[0] * whole;
    if (!(whole > 0.0)) {
        if (rank == 0 && tid == 0) p.next[slot] = -1;
    } else {
        // Of up to 32 sums (a lane has one) the first within which the running sum, from `before` on, passes the bar, or the
        // last that is not 0 where none does; `before` becomes the running sum in front of it.
        auto choose = [&](double mine, double &before, bool &past) {
            double incl = mine;
#pragma unroll 1
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const unsigned over = __ballot_sync(0xffffffffu, mine > 0.0 && before + incl > bar);
            const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
            const int at = over ? __ffs(over) - 1 : 31 - __clz(some);
            before += __shfl_sync(0xffffffffu, incl - mine, at);
            past = over != 0;
            return at;
        };
        double start = 0.0;
        bool past;
        const int owner = choose(lane < kCtas ? s_all[lane] : 0.0, start, past);
        if (rank == owner) {
            // the warp's run in the part; every warp of the CTA finds it alike
            const int at = choose(lane < kWarps ? s_warp[lane] : 0.0, start, past);
            const float *const target = p.target + (long long)(first + here) * p.row_stride;
            const float *const draft = p.draft && tried > 0 ? p.draft + (long long)(first + here) * p.row_stride : nullptr;
            const int w0 = min(v0 + at * run, v1), w1 = min(w0 + run, v1);
            int found = 0x7fffffff, ends = -1;
            // its segments of 32, one to a warp and round: their sums, then the one in which the running sum passes the bar
#pragma unroll 1
            for (int x0 = w0; x0 < w1; x0 += 32 * kWarps) {
                const int x = x0 + 32 * warp + lane;
                double w = 0.0;
                if (x < w1) w = left_of(probability(__ldg(target + x)), draft ? probability(__ldg(draft + x)) : 0.0, x, tried);
                double incl = w;
#pragma unroll 1
                for (int o = 1; o < 32; o <<= 1) {
                    const double v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                if (lane == 31) s_segment[warp] = incl;
                __syncthreads();
                double sums = lane < kWarps ? s_segment[lane] : 0.0;
#pragma unroll 1
                for (int o = 1; o < kWarps; o <<= 1) {
                    const double v = __shfl_up_sync(0xffffffffu, sums, o);
                    if (lane >= o) sums += v;
                }
                double c = start + incl;
                const double ahead = __shfl_sync(0xffffffffu, sums, warp > 0 ? warp - 1 : 0);
                if (warp > 0) c += ahead;
                start += __shfl_sync(0xffffffffu, sums, kWarps - 1);
                __syncthreads();
                if (w > 0.0) {
                    ends = x;
                    if (c > bar && found == 0x7fffffff) found = x;
                }
            }
            found = __reduce_min_sync(0xffffffffu, found);
            ends = __reduce_max_sync(0xffffffffu, ends);
            // (s_parent and s_token have been read for the last time)
            if (lane == 0) {
                s_parent[warp] = found;
                s_token[warp] = ends;
            }
            __syncthreads();
            if (tid == 0) {
                for (int k = 0; k < kWarps; k++) {
                    found = min(found, s_parent[k]);
                    ends = max(ends, s_token[k]);
                }
                p.next[slot] = found != 0x7fffffff ? found : ends;
            }
        }
    }
    cluster_sync_all();   // no CTA leaves while another may still read its sum
}

}  // namespace

namespace {

// How many clusters of sixteen CTAs of the kernel the current device runs at a time.
int sixteen_together() {
    if (cudaFuncSetAttribute(tree_verify<16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    cudaLaunchAttribute size = {};
    size.id = cudaLaunchAttributeClusterDimension;
    size.val.clusterDim.x = 16;
    size.val.clusterDim.y = size.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(16);
    config.blockDim = dim3(kThreads);
    config.attrs = &size;
    config.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, tree_verify<16>, &config) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return clusters;
}

}  // namespace

// Clusters of sixteen, which is more than every device must have and is asked for once, as long as all of them fit; more slots
// take eights (10 slots of 8 nodes of 151,936 with draft rows: 37 us, with eights 60).
// What bounds it is latency, not memory: a trip for the tree, one for what the walk asks, one pass, the exchange of its sums
// and the segment of the drawn token follow one another. 8 nodes of 151,936 take 9.7 us, 8 slots of 16 nodes of 50,257 with
// draft rows 14.5 to 20 (rejections in a row, a pass each), 32 slots of 8 nodes of 151,936 without draft rows 18 to 20 (their
// rows pass in 3).
int launch_tree_verify(cudaStream_t stream, const VerifyParams &p) {
    static std::atomic<int> sixteen[64];   // one more than clusters; 0: not asked yet
    int dev = 0;
    cudaGetDevice(&dev);
    const bool known = dev >= 0 && dev < 64;
    int most = known ? sixteen[dev].load() : 0;
    if (most == 0) {
        most = sixteen_together() + 1;
        if (known) sixteen[dev].store(most);
    }
    if (p.slots < most) return launch_pdl(tree_verify<16>, dim3(p.slots * 16), dim3(kThreads), 0, stream, 16, p);
    return launch_pdl(tree_verify<8>, dim3(p.slots * 8), dim3(kThreads), 0, stream, 8, p);
}

}  // namespace hipml
