// Attention of a tree of drafted tokens on the 5th-generation tensor cores, head_dim 256, straight from the cache.
// The definition stands in attn_tree.cu.
//
// A CTA has 128 query rows (nodes x heads of the group) of one KV head and a run of cache rows, which it takes in tiles.
// Per tile of 64 rows (32 of the f32 cache):
//     S = Q K^T       tcgen05.mma M = 128, N = 64, K = 256
//     W = 2^(S - m)   eight softmax warps, two threads a row, W written over S in TMEM
//     O += W V        tcgen05.mma M = 128, N = 128 (256), K = 64 (32), W from TMEM
//
// Both products take each operand as two f16 parts, x = hi + lo, and leave out lo lo: three MMAs a product, 22 bits of
// each operand. The planes of K and V are made here, by eight warps that read the rows as they lie (bulk copies into a ring)
// and write hi and lo to shared memory in the layout of the MMAs (rows of 64 dims, 128-byte swizzle): for K^T with the
// dims contiguous along K, for V the same image with them along N. A q8_0 or q4_0 value (11-bit scale times a code of 8
// bits) is exactly hi + lo: hi is its f16 product and lo the f16 FMA's remainder, two instructions for two values.
//
// f16 parts need their operands in range whatever the cache holds. So the rows of a tile are scaled by a power of two, K's
// and V's each by its largest scale (f32: value), and each query row by one of its own. S is multiplied back; the value's
// power 2^E goes into the weight: w = 2^(s + E - m), where m follows the largest s + E, and the denominator takes w 2^-E.
// Where a tile's rows lie so far apart that its smallest would lose bits (a drafted row that most nodes do not see may hold
// anything), each of them has a power of its own (rare; 64 nodes over 100,000 rows with every tile so: 517 us instead of 490).
// A K row that is not finite is not a number in the planes, which reaches the rows that see it and no others; a V row that is
// not finite is zero there, and the weights of those that see it are not a number (a hidden key's weight is 0).
//
// Where the time goes (a quantised tile of 64 rows): the MMAs 3,330 cycles (48 of N = 64, 32 cycles with A from TMEM and 48
// with A from shared memory, and 24 of N = 128, 64 cycles); shared memory as much: the raw bytes in and out (1.1 KB a row),
// the planes (2), K and the low part of Q into the pipe (2.5), V (1.5), 55 cycles a row. So Q's high part and W come from
// TMEM: Q hi takes 128 of the 512 columns, O 256, two S tiles 128. A tile takes 5,500 to 6,000 cycles, 64 nodes of 24 heads
// (four KV heads) over 100,000 rows 490 us (in a run under the power cap 550): the tensor pipe is 44 % busy and the issue
// slots 47 %, and the planes, Q K^T, the softmax and W V wait for one another. Four more warps for the planes changed
// nothing, nor did a third stage of V.
// Short calls are bound by what comes before the first tile: the launch, the tree, Q's planes, one trip to memory after
// another and the code's own lines (the loops are loops for that reason).
//
// Sums: the tensor cores cut their f32 accumulators off instead of rounding them, 3.5e-9 relative per key of an unbroken
// chain, so every kFlushKeys keys O leaves TMEM for the run's partial in memory (added there, in f32).
//
// Warps 0-7 softmax and epilogue, 8-11 planes of K, 12-15 of V, 16 copies, 17 the largest of a tile's V
// rows and their factors, 18 those of K, 19 MMAs
// (the whole warp runs that loop and one elected lane issues: from a branch of a single lane every descriptor went through a
// move to the uniform registers, 46 cycles an MMA of N = 64 and 83 beside the other warps, against 32; the fourth scheduler
// has the fewest other warps). Waits are bounded: one that runs out sets the device
// status and a flag that turns every other wait of the CTA into none; all warps still come to every barrier, nothing is
// written out, and copies and MMAs in flight are waited for (bounded too) before shared memory and TMEM are released.
#include <atomic>

#include "q8_pack.cuh"
#include "sm100_ptx.cuh"
#include "tree.cuh"

namespace hipml {

namespace {

using namespace ptx;

constexpr int kD = 256, kRows = kTreeTcRows;
constexpr int kThreads = 20 * 32;
constexpr int kGroup = 4;                        // warps that make planes: four of K, four of V
constexpr int kQChunk = kRows * 128;             // 128 rows x 64 dims, f16
constexpr int kQBytes = 4 * kQChunk;             // one plane of Q
constexpr int kStages = 2;                       // of K and of V
constexpr int kKStage = 32 * 1024, kVStage = 16 * 1024;
constexpr int kRawBytes = 3 * 64 * 272;
constexpr int kFlushKeys = 512;
constexpr unsigned kSpinLimit = 1u << 22;
constexpr float kThreshold = 5.0f;               // log2: the reference moves when a weight would exceed 2^5 times it,
constexpr float kLift = 10.0f;                   // and weights are kept 2^10 times larger: up to 2^15.5; f16's last bit, 2^-24,
                                                 // is then 2^-34 of the reference (2^-22 of weights down to 2^-12 of it)
constexpr int kLeastPower = -80, kMostPower = 117;   // of a tile or row; smaller values count as 0 (as do zeros)

template <int kType>   // 0 f32, 1 q8_0, 2 q4_0
struct Shape {
    static constexpr int kKeys = kType == 0 ? 32 : 64;         // of a tile
    static constexpr int kParts = kType == 0 ? 1 : 2;          // of a row, by dims
    static constexpr int kChunks = 4 / kParts;                 // of 64 dims, in a part
    // a stage of K has a part of a tile's rows, one of V a part of half of them; hi plane, then lo
    static constexpr int kChunkBytes = kKeys * 128;
    static constexpr int kPlaneBytes = kChunks * kChunkBytes;
    static constexpr int kVKeys = kKeys / 2;
    static constexpr int kVChunkBytes = kVKeys * 128;
    static constexpr int kVPlaneBytes = kChunks * kVChunkBytes;
    static_assert(kParts <= kStages && 2 * kPlaneBytes == kKStage && 2 * kVPlaneBytes == kVStage, "a stage is two planes");
    // the raw ring has half tiles (f32 rows padded apart so that eight rows' 16-byte words fall into different banks)
    static constexpr int kRowPitch = kType == 0 ? 1040 : (kType == 1 ? 272 : 144);
    static constexpr int kRawRows = kKeys / 2;
    static constexpr int kRawSlot = kRawRows * kRowPitch;
    static constexpr int kRawSlots = kRawBytes / kRawSlot < 8 ? kRawBytes / kRawSlot : 8;
    static constexpr int kHalf = kKeys / 2;                    // keys of a softmax thread
    // the 32 dims that make block b of part h of a row. Quantised blocks come in pairs (an odd block begins inside a word):
    // a part has one block of each pair, so that eight rows' four pairs fall into different banks.
    __host__ __device__ static constexpr int block(int h, int b) { return kType == 0 ? b : 2 * b + h; }
};

constexpr int kOffQ = 0;                                   // Q lo
constexpr int kOffK = kOffQ + kQBytes;
constexpr int kOffV = kOffK + kStages * kKStage;
constexpr int kOffRaw = kOffV + kStages * kVStage;
// What is known of a tile's rows ahead of their planes: the power of two of K, that of V, and which rows are not finite. A
// ring of eight tiles: a tile's rows are in the raw ring at the earliest when planes were made that needed Q K^T of three
// tiles before, and that came after the softmax of two more.
constexpr int kScouts = 8;
struct __align__(16) Scout {
    int power;
    unsigned bad[2];   // a bit per row
    int wide;          // whether the rows have powers of their own
};
constexpr int kOffScout = kOffRaw + kRawBytes;             // [K, V][kScouts]
constexpr int kOffFactors = kOffScout + 2 * kScouts * 16;   // [K, V][kScouts][64]: what each row is multiplied by
constexpr int kOffMeet = kOffFactors + 2 * kScouts * 64 * 4;   // [2][2][128]: the halves of a row meet
constexpr int kOffRowFac = kOffMeet + 2 * 2 * 128 * 4;     // [128]
constexpr int kOffSees = kOffRowFac + kRows * 4;           // [128][kTreeWords + 1]
constexpr int kOffParents = kOffSees + kRows * (kTreeWords + 1) * 4;
constexpr int kOffBars = kOffParents + kTreeNodes * 4;
constexpr int kBars = 55;
constexpr int kSmemNeed = kOffBars + kBars * 8;
constexpr int kSmemBytes = (kSmemNeed + 15) / 16 * 16 + 1024;               // (the planes lie on 1 KB boundaries)
static_assert(kSmemBytes <= 227 * 1024, "one CTA per SM");
constexpr int kOutPitch = kD + 4;                          // floats of a staged output row
static_assert(kRows * kOutPitch * 4 <= kOffRaw, "the output rows are staged over Q and the planes");
static_assert(kQBytes <= kStages * kKStage, "Q hi passes through K's stages");

constexpr unsigned kTmemO = 0, kTmemS = 256, kTmemQ = 384;   // columns; S: two tiles of 64

// MN-major operand of 64-dim chunks `pitch` bytes apart, each of rows of 128 bytes (8-row groups 1 KB apart), swizzled.
__device__ __forceinline__ unsigned desc_lo_mn(unsigned addr, unsigned pitch) {
    return ((addr & 0x3ffff) >> 4) | (pitch >> 4) << 16;
}

// The kernel's code is kept small: its roles together, and what runs once, come through one instruction cache (with every
// loop unrolled a tile of 64 rows took 10,000 cycles and Q 6,700). Loops over blocks, rows and chunks are loops.
__device__ __noinline__ bool wait_long(unsigned bar, unsigned parity, volatile int *abort, int *status, int code) {
    for (unsigned i = 0; i < kSpinLimit; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255) == 255 && *abort) return false;
        if (i > 4096) __nanosleep(64);
    }
    atomicCAS(status, 0, code);
    *abort = 1;
    return false;
}
__device__ __forceinline__ bool elect_one() {
    unsigned p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
struct Waits {
    volatile int *abort;
    int *status;
    __device__ __forceinline__ bool operator()(unsigned bar, unsigned parity, int code) const {
        return mbar_try_wait(bar, parity) || wait_long(bar, parity, abort, status, code);
    }
};

__device__ __forceinline__ __half2 as_half2(unsigned x) { return *reinterpret_cast<__half2 *>(&x); }
__device__ __forceinline__ unsigned as_bits(__half2 x) { return *reinterpret_cast<unsigned *>(&x); }

// hi and lo of code times scale, two values: hi is the rounded product, lo exactly what it lacks.
__device__ __forceinline__ void split_product(__half2 code, __half2 scale, unsigned &hi, unsigned &lo) {
    const __half2 h = __hmul2(code, scale);
    hi = as_bits(h);
    lo = as_bits(__hfma2(code, scale, __hneg2(h)));
}
__device__ __forceinline__ void split_pair(float a, float b, unsigned &hi, unsigned &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = as_bits(h);
    lo = as_bits(__floats2half2_rn(a - f.x, b - f.y));
}

// 2^n for whole n of [-126, 127]
__device__ __forceinline__ float power(int n) { return __int_as_float((n + 127) << 23); }

// The largest |value| of half of an f32 row, or |scale| of a quantised row, as bits; `least`: less one, the smallest scale that
// is not 0 (2^32 - 1: none).
template <int kType>
__device__ __forceinline__ unsigned row_most(const unsigned char *row, int half, unsigned &least) {
    unsigned most = 0;
    least = 0xffffffffu;
    if constexpr (kType == 0) {
#pragma unroll 4
        for (int k = 0; k < 32; k++) {
            const uint4 x = reinterpret_cast<const uint4 *>(row)[32 * half + k];
            most = max(max(most, x.x & 0x7fffffffu), max(max(x.y & 0x7fffffffu, x.z & 0x7fffffffu), x.w & 0x7fffffffu));
        }
    } else {
#pragma unroll
        for (int b = 0; b < 8; b++) {
            const unsigned x = *reinterpret_cast<const unsigned short *>(row + b * (kType == 1 ? 34 : 18)) & 0x7fff;
            most = max(most, x);
            least = min(least, x - 1);
        }
    }
    return most;
}
// The power of two that brings rows into range, from their largest |value| or |scale| as bits: values come to [2^10, 2^11),
// scales to [8, 16), so that codes times them stay below 2^11 and lo is exact.
template <int kType>
__device__ __forceinline__ int power_of(unsigned most) {
    if (kType == 0) return min(max((int)(most >> 23) - 127 - 10, kLeastPower), kMostPower);
    return most == 0 ? kLeastPower : max((int)most >> 10, 1) - 15 - 3;
}

// A quantised block's 32 values times scale, as hi and lo words in the order of the dims. `w`: its words from the one that
// holds its scale on. An even block's codes begin in the middle of that word (take = 0x5432), an odd one's behind it (0x7654).
template <int kType>
__device__ __forceinline__ void block_planes(const unsigned *w, unsigned take, __half2 s, unsigned (&hi)[16], unsigned (&lo)[16]) {
    if constexpr (kType == 1) {
        const __half2 bias = __float2half2_rn(1152.0f);   // 0x6400 | byte is 1024 + byte
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const unsigned c = __byte_perm(w[j], w[j + 1], take) ^ 0x80808080u;
            split_product(__hsub2(as_half2(__byte_perm(c, 0x64646464u, 0x4140)), bias), s, hi[2 * j], lo[2 * j]);
            split_product(__hsub2(as_half2(__byte_perm(c, 0x64646464u, 0x4342)), bias), s, hi[2 * j + 1], lo[2 * j + 1]);
        }
    } else {
        const __half2 bias = __float2half2_rn(1032.0f);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned c = __byte_perm(w[j], w[j + 1], take);
#pragma unroll
            for (int e = 0; e < 2; e++) {   // bytes 0, 1 and 2, 3; the low nibbles are values j, the high ones j + 16
                const unsigned x = __byte_perm(c, 0, e ? 0x4342 : 0x4140);
                split_product(__hsub2(as_half2((x & 0x000f000fu) | 0x64006400u), bias), s, hi[2 * j + e], lo[2 * j + e]);
                split_product(__hsub2(as_half2(((x >> 4) & 0x000f000fu) | 0x64006400u), bias), s, hi[8 + 2 * j + e],
                              lo[8 + 2 * j + e]);
            }
        }
    }
}

// grid tree_grid(.., 128 rows, the device's SMs), 20 warps.
template <int kType>
__global__ void __launch_bounds__(kThreads, 1) attn_tree_tc(TreeParams p) {
    using T = Shape<kType>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *const smem =
        reinterpret_cast<unsigned char *>((reinterpret_cast<size_t>(smem_raw) + 1023) & ~(size_t)1023);
    __shared__ TreeItem s_item;
    __shared__ int s_abort;
    __shared__ unsigned s_tmem;
    griddep_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint64_t *const bars = reinterpret_cast<uint64_t *>(smem + kOffBars);
    // raw rows: full by the half tile's number, eight of K and eight of V (whoever waits for one waits for all of its kind, in
    // their order, so no phase is taken for another), empty by the slot
    const unsigned raw_full = smem_u32(bars), raw_empty = smem_u32(bars + 16), k_full = smem_u32(bars + 24),
                   k_empty = smem_u32(bars + 26), v_full = smem_u32(bars + 28), v_empty = smem_u32(bars + 30),
                   s_ready = smem_u32(bars + 32), w_ready = smem_u32(bars + 34), o_done = smem_u32(bars + 36),
                   scouted = smem_u32(bars + 38), all_done = smem_u32(bars + 54);
    static_assert(T::kRawSlots <= 8 && kScouts == 8 && kBars == 55, "barriers");
    auto scout_bar = [&](bool v, int t) { return scouted + 8 * ((v ? 8 : 0) + (t & 7)); };   // of tile t
    Scout *const scouts = reinterpret_cast<Scout *>(smem + kOffScout);
    // of tile t, by row: a power of two, 0 where there is no row, not a number where the row is not finite
    auto factors = [&](bool v, int t) { return reinterpret_cast<float *>(smem + kOffFactors) + 64 * ((v ? 8 : 0) + (t & 7)); };
    auto raw_bar = [&](bool v, int i) { return raw_full + 8 * ((v ? 8 : 0) + (i & 7)); };   // of half tile i
    if (warp == 1) {
        for (int i = lane; i < kBars; i += 32) {
            const int pair = i / 2;   // from 12 on: k_full, k_empty, v_full, v_empty, s_ready, w_ready, o_done
            // (a raw slot is read by four warps that make planes and one that scouts)
            mbar_init(raw_full + 8 * i, i >= 16 && i < 24          ? kGroup + 1
                                        : pair == 12 || pair == 14 ? kGroup
                                        : pair == 17               ? 8
                                                                   : 1);
        }
        if (lane == 0) s_abort = 0;
        mbar_init_fence();
    }
    if (warp == 19) tmem_alloc<1>(smem_u32(&s_tmem), 512);
    tc_fence_before();
    griddep_wait();
    if (warp == 0) {
        const TreeItem it = tree_item<kRows>(p, blockIdx.x);
        if (lane == 0) s_item = it;
    }
    __syncthreads();
    tc_fence_after();
    const TreeItem it = s_item;
    const Waits wait = {&s_abort, p.status};
    const int rows = min(kRows, it.live * p.group - it.tile * kRows);
    const int lo_key = it.first_row(), hi_key = it.end_row();
    const int n = it.slot < 0 ? 0 : (hi_key - lo_key + T::kKeys - 1) / T::kKeys;   // tiles
    const size_t first_node = (size_t)it.slot * p.nodes;
    auto head_row = [&](int r) {   // row r of the tile as a row of q and out, in heads
        const int at = it.tile * kRows + r, node = p.node_of(at);
        return (first_node + node) * p.n_heads + it.kvh * p.group + (at - node * p.group);
    };
    // Half tiles in the raw ring: K0 K1 V0 K2 V1 .. V(n-1). A slot of V is free when its planes are made, in the middle of
    // its W V, and what takes it is then K of two tiles later. (K0 V0 K1 V1: K of the next tile, whose copy everything waited
    // for.)
    auto raw_of = [&](bool v, int t) { return v ? (t == n - 1 ? 4 * t + 2 : 4 * t + 4) : (t == 0 ? 0 : 4 * t - 2); };
    const size_t slot_at = (size_t)it.slot * p.slot_bytes;
    auto tile_rows = [&](int t) { return min(T::kKeys, hi_key - (lo_key + t * T::kKeys)); };

    if (warp == 16 && n > 0) {
        // ------------------------------------------------------------ copies
        unsigned c = 0, c_k = 0, c_v = 0;   // half tiles asked for, of K, of V
        for (int m = 0; m < 2 * n && !*wait.abort; m++) {
            const bool is_v = m == 2 * n - 1 || (m > 0 && (m & 1) == 0);
            const int t = m == 2 * n - 1 ? n - 1 : (is_v ? m / 2 - 1 : (m + 1) / 2), live = tile_rows(t);
            const unsigned char *const cache = (is_v ? p.v : p.k) + slot_at;
            for (int piece = 0; piece < 2; piece++, c++) {
                const unsigned slot = c % T::kRawSlots, round = c / T::kRawSlots;
                wait(raw_empty + 8 * slot, (round & 1) ^ 1, 51);
                const int key = lo_key + t * T::kKeys + piece * T::kRawRows;
                const int here = min(max(live - piece * T::kRawRows, 0), T::kRawRows);
                const unsigned dst = smem_u32(smem + kOffRaw) + slot * T::kRawSlot, bar = raw_bar(is_v, 2 * t + piece);
                const bool go = !*wait.abort;
                if (__any_sync(0xffffffffu, !go)) break;
                (is_v ? c_v : c_k)++;
                if constexpr (kType == 0) {
                    if (lane == 0) mbar_arrive_expect_tx(bar, here * kD * 4);
                    __syncwarp();
                    if (lane < here)
                        bulk_load(dst + lane * T::kRowPitch, cache + ((size_t)(key + lane) * p.n_kv + it.kvh) * (kD * 4), kD * 4,
                                  bar);
                } else if (lane == 0) {
                    mbar_arrive_expect_tx(bar, here * T::kRowPitch);
                    bulk_load(dst, cache + ((size_t)it.kvh * p.stride + key) * T::kRowPitch, here * T::kRowPitch, bar);
                }
            }
        }
        __syncwarp();
        if (*wait.abort) {
            // what is on its way lands before shared memory is released: the last half tiles of both kinds
            for (int i = 0; i < 16; i++) {
                const unsigned used = i < 8 ? c_k : c_v;   // half tiles asked for
                const unsigned last = used > (unsigned)(i & 7) ? (used - 1 - (i & 7)) / 8 : 0;   // uses of the barrier, less one
                if (used > (unsigned)(i & 7))
                    for (unsigned spin = 0; spin < kSpinLimit; spin++)
                        if (mbar_try_wait(raw_full + 8 * i, last & 1)) break;
            }
        }
    }

    // ---------------------------------------------------------------- Q: warps 0-7 and 12-15, a row at a time
    // hi goes to TMEM by way of K's stages.
    if ((warp < 8 || (warp >= 12 && warp < 16)) && n > 0) {
        constexpr int kQWarps = 12;
        const int qw = warp < 8 ? warp : warp - 4;
        // Position of dims 8 * lane .. in the order of the parts: block b of part h stands at 128 h + 32 b (f32: 32 b)
        const int blk = lane >> 2;
        const int at = kType == 0 ? 8 * lane : 128 * (blk & 1) + 32 * (blk >> 1) + 8 * (lane & 3);
        unsigned char *const to = smem + kOffQ + (at >> 6) * kQChunk;
        for (int i = tid < 256 ? tid : tid - 128; i < it.live; i += 384)
            reinterpret_cast<int *>(smem + kOffParents)[i] = p.parents[first_node + i];
        if (tid >= rows && tid < kRows) reinterpret_cast<float *>(smem + kOffRowFac)[tid] = 0.0f;
        auto row_at = [&](int r) { return reinterpret_cast<const float4 *>(p.q + head_row(r) * kD) + 2 * lane; };
        constexpr int kAhead = 4;   // rows on their way
        float4 x[kAhead][2];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const float4 *const src = row_at(min(qw + kQWarps * k, rows - 1));
            x[k][0] = __ldg(src);
            x[k][1] = __ldg(src + 1);
        }
#pragma unroll 1
        for (int r0 = qw; r0 < rows; r0 += kQWarps * kAhead) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int r = r0 + kQWarps * k;
                if (r >= rows) break;
                const float v[8] = {x[k][0].x, x[k][0].y, x[k][0].z, x[k][0].w, x[k][1].x, x[k][1].y, x[k][1].z, x[k][1].w};
                if (r + kQWarps * kAhead < rows) {
                    const float4 *const src = row_at(r + kQWarps * kAhead);
                    x[k][0] = __ldg(src);
                    x[k][1] = __ldg(src + 1);
                }
                unsigned most = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
                most = __reduce_max_sync(0xffffffffu, most);
                const bool bad = most >= 0x7f800000u;
                // the row's largest value comes to [2^10, 2^11)
                const int e = min(max((int)(most >> 23) - 127 - 10, -116), 116);
                const float f = copysignf(power(-e), p.scale_log2);   // (the largest score is the largest S)
                unsigned hi[4], lo[4];
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    split_pair(v[2 * d] * f, v[2 * d + 1] * f, hi[d], lo[d]);
                    if (bad) hi[d] = lo[d] = 0;
                }
                if (lane == 0)
                    reinterpret_cast<float *>(smem + kOffRowFac)[r] = bad ? __int_as_float(0x7fffffff) : power(e) * fabsf(p.scale_log2);
                const int off = sw128_offset(r, at & 63);
                *reinterpret_cast<uint4 *>(to + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                *reinterpret_cast<uint4 *>(to + (kOffK - kOffQ) + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            }
        }
        fence_async_shared();   // Q lo; the barriers below carry it on
        named_sync(1, 32 * kQWarps);
        if (warp < 8) {
            // thread (row, half) takes two chunks of the row's hi plane to TMEM
            const int r = tid & 127, half = tid >> 7;
#pragma unroll 1
            for (int c = 2 * half; c < 2 * half + 2; c++) {
                unsigned q[32];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(smem + kOffK + c * kQChunk + sw128_offset(r, 8 * j));
                    q[4 * j] = w.x;
                    q[4 * j + 1] = w.y;
                    q[4 * j + 2] = w.z;
                    q[4 * j + 3] = w.w;
                }
                tmem_st32(s_tmem + kTmemQ + 32 * c + ((unsigned)((warp & 3) * 32) << 16), q);
            }
            tmem_wait_st();
            named_arrive(7, 12 * 32);   // K's stages are free
            if (tid < kRows && hi_key > it.base) {
                // which drafted rows this row sees (rows past the last: those of the last)
                unsigned *const sees = reinterpret_cast<unsigned *>(smem + kOffSees) + tid * (kTreeWords + 1);
                tree_ancestors(reinterpret_cast<const int *>(smem + kOffParents), p.node_of(it.tile * kRows + min(tid, rows - 1)),
                               sees, p.status);
                sees[kTreeWords] = 0;
            }
        }
    }
    tc_fence_before();
    if (warp < 8 || warp == 19) named_sync(6, 9 * 32);   // Q is there (the planes are under way meanwhile)
    tc_fence_after();
    const unsigned tmem = s_tmem;

    if (warp == 19) {
        // ------------------------------------------------------------ MMAs
        if (n > 0) {
            constexpr unsigned kMn = 1u << 16;   // B with N contiguous
            constexpr unsigned kIdescS = idesc_f16(128, T::kKeys), kIdescO = idesc_f16(128, 64 * T::kChunks) | kMn;
            const unsigned q_lo = desc_lo_sw128(smem_u32(smem + kOffQ));
            unsigned kc = 0, vc = 0;   // stages consumed
            // A stage's MMAs are one straight run from one election: every instruction between two of them competes with four
            // other warps for the scheduler (looped by fours, beside busy warps: 3,093 cycles a Q K^T, so 2,051).
            bool ok = true;
            auto stage = [&](unsigned bar, unsigned parity, int code) {
                ok = __all_sync(0xffffffffu, wait(bar, parity, code));
                tc_fence_after();
            };
            auto qk = [&](int i) {
                const unsigned d = tmem + kTmemS + 64 * (i & 1), planes = desc_lo_sw128(smem_u32(smem + kOffK));
                // The small terms of the whole row first, the large ones last: each MMA cuts the sum off, relative to what it
                // has come to. (By parts, each with its small and large terms, the error of S was twice as large.)
#pragma unroll 1
                for (int h = 0; h < T::kParts; h++) {
                    const unsigned slot = (kc + h) % kStages;
                    stage(k_full + 8 * slot, ((kc + h) / kStages) & 1, 52);
                    if (!ok) return;
                    const unsigned hi = planes + slot * (kKStage >> 4), lo = hi + (T::kPlaneBytes >> 4);
                    const unsigned ql = q_lo + h * T::kChunks * (kQChunk >> 4), qh = tmem + kTmemQ + 32 * T::kChunks * h;
                    const unsigned more = h != 0;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4 * T::kChunks; k++)
                            tc_mma_ts<1>(d, qh + 8 * k, desc_from(lo + (k / 4) * (T::kChunkBytes >> 4) + 2 * (k % 4)), kIdescS,
                                         k == 0 ? more : 1);
#pragma unroll
                        for (int k = 0; k < 4 * T::kChunks; k++)
                            tc_mma_ss<1>(d, desc_from(ql + (k / 4) * (kQChunk >> 4) + 2 * (k % 4)),
                                         desc_from(hi + (k / 4) * (T::kChunkBytes >> 4) + 2 * (k % 4)), kIdescS, 1);
                    }
                    __syncwarp();
                }
#pragma unroll 1
                for (int h = 0; h < T::kParts; h++, kc++) {
                    const unsigned hi = planes + (kc % kStages) * (kKStage >> 4);
                    const unsigned qh = tmem + kTmemQ + 32 * T::kChunks * h;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4 * T::kChunks; k++)
                            tc_mma_ts<1>(d, qh + 8 * k, desc_from(hi + (k / 4) * (T::kChunkBytes >> 4) + 2 * (k % 4)), kIdescS, 1);
                        tc_commit<1>(k_empty + 8 * (kc % kStages));
                        if (h + 1 == T::kParts) tc_commit<1>(s_ready + 8 * (i & 1));
                    }
                    __syncwarp();
                }
            };
            auto pv = [&](int i) {
                const unsigned later = (i * T::kKeys) % kFlushKeys != 0;   // 0: O starts afresh
#pragma unroll
                for (int s = 0; s < 2 * T::kParts; s++) {   // half of the rows, part of the dims
                    const int half = s / T::kParts, h = s % T::kParts;
                    stage(v_full + 8 * (vc % kStages), (vc / kStages) & 1, 53);
                    if (!ok) return;
                    const unsigned a = tmem + kTmemS + 64 * (i & 1) + T::kVKeys * half, d = tmem + kTmemO + 128 * h;
                    const unsigned hi = desc_lo_mn(smem_u32(smem + kOffV) + (vc % kStages) * kVStage, T::kVChunkBytes);
                    const unsigned lo = hi + (T::kVPlaneBytes >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < T::kVKeys / 16; k++) {   // 16 keys: two groups of eight rows
                            tc_mma_ts<1>(d, a + 16 * k, desc_from(lo + 128 * k), kIdescO, (half | k) == 0 ? later : 1);
                            tc_mma_ts<1>(d, a + 16 * k + 8, desc_from(hi + 128 * k), kIdescO, 1);
                            tc_mma_ts<1>(d, a + 16 * k, desc_from(hi + 128 * k), kIdescO, 1);
                        }
                        tc_commit<1>(v_empty + 8 * (vc % kStages));
                        if (s + 1 == 2 * T::kParts) tc_commit<1>(o_done + 8 * (i & 1));
                    }
                    __syncwarp();
                    vc++;
                }
            };
            qk(0);
            for (int i = 0; i < n && ok; i++) {
                if (i + 1 < n) qk(i + 1);
                if (!ok) break;
                stage(w_ready + 8 * (i & 1), (i >> 1) & 1, 54);
                if (ok) pv(i);
            }
            if (!ok) {
                if (elect_one()) tc_commit<1>(all_done);
                for (unsigned spin = 0; spin < kSpinLimit && !mbar_try_wait(all_done, 0); spin++) {}
            }
        }
    } else if (warp == 17 || warp == 18) {
        // ------------------------------------------------------------ scouts: warp 17 of V, 18 of K
        const bool is_v = warp == 17;
#pragma unroll 1
        for (int t = 0; t < n; t++) {
            const int live = tile_rows(t);
            Scout found = {0, {0, 0}, 0};
            unsigned most = 0;                                        // of the rows that are finite:
            unsigned least = 0xffffffffu, least_scale = 0xffffffffu;  // of those that are not 0, less one
#pragma unroll 1
            for (int j = 0; j < 2; j++) {
                const unsigned u = raw_of(is_v, t) + j;
                wait(raw_bar(is_v, 2 * t + j), ((2 * t + j) >> 3) & 1, 56);
                const unsigned char *const from = smem + kOffRaw + (u % T::kRawSlots) * T::kRawSlot;
                // f32: a lane has half of a row; quantised: a lane has a row
                const int r = kType == 0 ? lane & 15 : lane;
                unsigned mine = 0, small = 0xffffffffu;
                if (T::kRawRows * j + r < live) mine = row_most<kType>(from + r * T::kRowPitch, kType == 0 ? lane >> 4 : 0, small);
                if constexpr (kType == 0) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 16));
                const bool bad = mine >= (kType == 0 ? 0x7f800000u : 0x7c00u);
                const unsigned bits = __ballot_sync(0xffffffffu, bad);
                if (kType == 0)
                    found.bad[0] |= (bits & 0xffff) << (16 * j);
                else
                    found.bad[j] = bits;
                if (!bad) {
                    most = max(most, mine);
                    least = min(least, mine - 1);
                    least_scale = min(least_scale, small);
                }
                if (kType != 0 || lane < 16)
                    factors(is_v, t)[T::kRawRows * j + r] = bad ? __int_as_float(0x7fffffff)
                                                            : T::kRawRows * j + r < live ? power(-power_of<kType>(mine))
                                                                                         : 0.0f;
                if (lane == 0) mbar_arrive(raw_empty + 8 * (u % T::kRawSlots));
            }
            most = __reduce_max_sync(0xffffffffu, most);
            least = __reduce_min_sync(0xffffffffu, least);
            found.power = power_of<kType>(most);
            // Against f16's 2^-24 a scale of [8, 16) has 17 powers to spare until a product loses a bit, the largest value of an
            // f32 row, of [2^10, 2^11), has 12 until fewer than 22 are left. A tile of V whose power is that of a row that a
            // query hardly sees costs the weights of the other tiles as many bits: 7 at most.
            const int spread = least < most ? found.power - power_of<kType>(least + 1) : 0;
            found.wide = spread > (is_v ? 7 : 12);
            if (kType != 0) {
                least_scale = __reduce_min_sync(0xffffffffu, least_scale);
                if (least_scale < most && found.power - power_of<kType>(least_scale + 1) > 17) found.wide = 1;
            }
            if (!found.wide) {   // one power for all
                for (int k = lane; k < T::kKeys; k += 32) {
                    float *const by = factors(is_v, t) + k;
                    if (*by > 0.0f) *by = power(-found.power);
                }
            }
            __syncwarp();
            if (lane == 0) {
                scouts[(is_v ? kScouts : 0) + (t & 7)] = found;
                mbar_arrive(scout_bar(is_v, t));
            }
        }
    } else if (warp >= 8 && warp < 16) {
        // ------------------------------------------------------------ planes: warps 8-11 of K, 12-15 of V
        const bool is_v = warp >= 12;
        const int w4 = warp & 3;
        constexpr int kPair = kType == 1 ? 17 : 9, kOdd = kType == 1 ? 8 : 4;   // words of two blocks; the odd block's first
        // Thread's row of half tile j. f32: block lane / 4 of row 4 (warp % 4) + lane % 4 (of 16). Quantised: pair lane / 8 of
        // row 8 (warp % 4) + lane % 8 (of 32), one block of it in each part.
        const int row = kType == 0 ? 4 * w4 + (lane & 3) : 8 * w4 + (lane & 7);
        const int blk = lane >> 2, pair = lane >> 3;
        auto free_raw = [&](unsigned u) {
            if (lane == 0) mbar_arrive(raw_empty + 8 * (u % T::kRawSlots));
        };
        unsigned c = 0;                               // stages written
#pragma unroll 1
        for (int t = 0; t < n; t++) {
            const int live = tile_rows(t);
            const unsigned u0 = raw_of(is_v, t);   // the tile's first raw slot
            wait(raw_bar(is_v, 2 * t), ((2 * t) >> 3) & 1, 56);
            wait(raw_bar(is_v, 2 * t + 1), ((2 * t + 1) >> 3) & 1, 56);
            wait(scout_bar(is_v, t), (t >> 3) & 1, 58);
            // K: both halves of a part, then the other part; V: both parts of a half, then the other half
#pragma unroll 1
            for (int s = 0; s < 2 * T::kParts; s++) {
                const int j = kType == 0 ? s : (is_v ? s >> 1 : s & 1), h = kType == 0 ? 0 : (is_v ? s & 1 : s >> 1);
                const int key = T::kRawRows * j + row;
                const unsigned full = (is_v ? v_full : k_full) + 8 * (c % kStages);
                const unsigned char *const raw_row = smem + kOffRaw + ((u0 + j) % T::kRawSlots) * T::kRawSlot + row * T::kRowPitch;
                float by = factors(is_v, t)[key];
                const bool bad = by != by;
                if (bad) by = 0.0f;
                unsigned hi[16], lo[16];
                if constexpr (kType == 0) {
                    // (an odd block's halves are swapped: eight lanes' words fall into different banks)
                    const float4 *const src = reinterpret_cast<const float4 *>(raw_row + blk * 128);
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const float4 a = src[k ^ ((blk & 1) << 2)];
                        split_pair(a.x * by, a.y * by, hi[2 * k], lo[2 * k]);
                        split_pair(a.z * by, a.w * by, hi[2 * k + 1], lo[2 * k + 1]);
                    }
                    if (by == 0.0f) {   // (not finite, or no row at all: there may be anything)
#pragma unroll
                        for (int k = 0; k < 16; k++) hi[k] = lo[k] = 0;
                    }
                } else {
                    const unsigned *const src = reinterpret_cast<const unsigned *>(raw_row) + pair * kPair + (h ? kOdd : 0);
                    unsigned w[kOdd + 1];
#pragma unroll
                    for (int k = 0; k <= kOdd; k++) w[k] = src[k];
                    const float scale = half_bits_to_float((uint16_t)(w[0] >> (16 * h)));
                    block_planes<kType>(w, h ? 0x7654 : 0x5432, __float2half2_rn(by == 0.0f ? 0.0f : scale * by), hi, lo);
                }
                if (bad && !is_v) hi[0] = 0x7fff7fff;   // one value is enough: the row's scores are not a number
                if (!is_v && c == 0 && j == 0) named_sync(7, 12 * 32);   // Q hi has left K's stages
                if (is_v || j == 0) wait((is_v ? v_empty : k_empty) + 8 * (c % kStages), ((c / kStages) & 1) ^ 1, 55);
                const int b = kType == 0 ? blk : pair;
                unsigned char *const dst = is_v ? smem + kOffV + (c % kStages) * kVStage + row * 128 + (b >> 1) * T::kVChunkBytes
                                                : smem + kOffK + (c % kStages) * kKStage + key * 128 + (b >> 1) * T::kChunkBytes;
                const int plane = is_v ? T::kVPlaneBytes : T::kPlaneBytes;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int unit = 4 * (b & 1) + (kType == 0 ? k ^ ((b & 1) << 1) : k);
                    const int at = (unit ^ (key & 7)) << 4;
                    *reinterpret_cast<uint4 *>(dst + at) = make_uint4(hi[4 * k], hi[4 * k + 1], hi[4 * k + 2], hi[4 * k + 3]);
                    *reinterpret_cast<uint4 *>(dst + plane + at) =
                        make_uint4(lo[4 * k], lo[4 * k + 1], lo[4 * k + 2], lo[4 * k + 3]);
                }
                const bool done = s + 1 == 2 * T::kParts;
                if (is_v || j == 1) {   // the stage is written
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full);
                    c++;
                }
                // a half's rows were read for the last time
                if (kType == 0) {
                    __syncwarp();
                    free_raw(u0 + j);
                } else if (is_v) {
                    if (h == 1) free_raw(u0 + j);
                } else if (done) {
                    free_raw(u0);
                    free_raw(u0 + 1);
                }
            }
        }
    } else if (warp < 8 && n > 0) {
        // ------------------------------------------------------------ softmax
        const int r = tid & 127, half = tid >> 7;
        const unsigned lane_at = tmem + ((unsigned)((warp & 3) * 32) << 16);
        const float row_factor = reinterpret_cast<const float *>(smem + kOffRowFac)[r];
        const bool live = r < rows, whole = it.runs == 1;
        // m_out: the reference of what is in memory already, which is at most 2^30 above it
        float m = -INFINITY, l = 0.0f, m_out = -INFINITY;
        // the other half's value of the row (the warps w and w + 4 meet)
        auto meet = [&](int x, float mine) {
            float *const buf = reinterpret_cast<float *>(smem + kOffMeet) + (x & 1) * 256;
            buf[128 * half + r] = mine;
            named_sync(2 + (warp & 3), 64);
            return buf[128 * (half ^ 1) + r];
        };
        // dims of column group j (32 columns) of this thread's half of O
        auto dims_of = [&](int j) { return kType == 0 ? 128 * half + 32 * j : 32 * T::block(half, j); };
        const bool idle = 32 * (warp & 3) >= rows;   // (no row of this warp is live: nothing reads its lanes)
        // Values' powers are taken relative to that of the run's first tile, within [-9, 8]: then no weight's share of the
        // denominator, w 2^-E, leaves f32's range, for E of [-80, 117].
        int power0 = 0;
        float *const flushed = p.part_acc + ((size_t)blockIdx.x * kRows * (kD / 4) + r) * 4;   // [64 x four dims][128 rows]
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            const unsigned s_at = lane_at + kTmemS + 64 * (i & 1) + T::kHalf * half;
            wait(s_ready + 8 * (i & 1), (i >> 1) & 1, 57);
            if (idle) {
                __syncwarp();
                if (lane == 0) mbar_arrive(w_ready + 8 * (i & 1));
                continue;
            }
            wait(scout_bar(false, i), (i >> 3) & 1, 58);
            wait(scout_bar(true, i), (i >> 3) & 1, 58);
            const Scout known = scouts[kScouts + (i & 7)];
            if (i == 0) power0 = min(max(known.power, -9), 8);
            float value_power = (float)(known.power - power0), value_inverse = power(power0 - known.power);
            const Scout known_k = scouts[i & 7];
            const bool wide = (known.wide | known_k.wide) != 0;
            float factor = row_factor * power(known_k.power);   // of S; > 0, so that a hidden row's -inf stays that
            if (factor < 1e-30f) factor = 1e-30f;
            __syncwarp();
            tc_fence_after();
            float u[T::kHalf];
            if constexpr (T::kHalf == 32) {
                unsigned v[32];
                tmem_ld32(s_at, v);
#pragma unroll
                for (int e = 0; e < 32; e++) u[e] = __uint_as_float(v[e]);
            } else {
                tmem_ld16(s_at, u);
            }
            const int key0 = lo_key + i * T::kKeys + T::kHalf * half;
            if ((known.bad[0] | known.bad[1]) != 0) {   // rare: a V row that is not finite
                const unsigned bits = T::kHalf == 32 ? known.bad[half] : known.bad[0] >> (16 * half);
#pragma unroll
                for (int e = 0; e < T::kHalf; e++)
                    if (bits >> e & 1) u[e] = __int_as_float(0x7fffffff);
            }
            if (lo_key + (i + 1) * T::kKeys > it.base) {   // drafted rows, and none past the last
                unsigned sees;
                const int from = key0 - it.base;
                const unsigned *const words = reinterpret_cast<const unsigned *>(smem + kOffSees) + r * (kTreeWords + 1);
                if (from <= -32) {
                    sees = 0xffffffffu;
                } else if (from < 0) {
                    sees = (1u << -from) - 1 | words[0] << -from;
                } else if (from < kTreeNodes) {
                    sees = __funnelshift_r(words[from >> 5], words[(from >> 5) + 1], from & 31);
                } else {
                    sees = 0;
                }
#pragma unroll
                for (int e = 0; e < T::kHalf; e++)
                    if (!(sees >> e & 1)) u[e] = -INFINITY;
            }
            // Rows with powers of their own: u becomes s + E here, and the denominator's terms are summed relative to their own
            // largest. (The sums are rounded where they are exact otherwise: 2^-24 of the exponent, which a spread of 2^20 takes
            // to some 30.)
            float most_s = -INFINITY, sum_s = 0.0f;
            if (__builtin_expect(wide, 0)) {
                const float *const by_k = factors(false, i) + T::kHalf * half, *const by_v = factors(true, i) + T::kHalf * half;
                auto power_in = [](float by) { return 127 - (__float_as_int(by) >> 23); };
#pragma unroll
                for (int e = 0; e < T::kHalf; e++) {
                    const float f = row_factor * power(power_in(by_k[e]));
                    u[e] *= f < 1e-30f ? 1e-30f : f;
                    most_s = fmaxf(most_s, u[e]);
                }
                if (most_s > -INFINITY) {
#pragma unroll
                    for (int e = 0; e < T::kHalf; e++) {
                        sum_s += ex2(u[e] - most_s);
                        u[e] += (float)(power_in(by_v[e]) - power0);
                    }
                }
                factor = 1.0f;
                value_power = value_inverse = 0.0f;
            }
            float big[4] = {u[0], u[1], u[2], u[3]};
#pragma unroll
            for (int e = 4; e < T::kHalf; e += 4)
#pragma unroll
                for (int k = 0; k < 4; k++) big[k] = fmaxf(big[k], u[e + k]);
            float m_new = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
            // (a whole number: what is subtracted is exact then, the same in every tile, and O's corrections are powers of two)
            m_new = fmaxf(m, rintf(fmaf(fmaxf(m_new, meet(i, m_new)), factor, value_power)));
            const bool fresh = (i * T::kKeys) % kFlushKeys == 0;   // O starts afresh with this tile
            const bool flush = fresh && i > 0;
            const bool move = !fresh && (m_new > m + kThreshold || (m == -INFINITY && m_new > -INFINITY));
            if (flush || __any_sync(0xffffffffu, move)) {
                wait(o_done + 8 * ((i - 1) & 1), ((i - 1) >> 1) & 1, 59);
                __syncwarp();
                tc_fence_after();
            }
            if (flush) {
                // O, relative to m, is added to what is in memory, relative to m_out (or takes its place, where that is nothing
                // beside it); a warp's 32 rows lie together there
                const bool over = m_out == -INFINITY || m > m_out + 90.0f;
                if (!over && m > m_out + 30.0f && live && !*wait.abort) {   // rare
                    const float down = exp2f(m_out - m);
#pragma unroll 1
                    for (int j = 0; j < 32; j++) {
                        float4 *const at = reinterpret_cast<float4 *>(flushed + (size_t)(32 * half + j) * (kRows * 4));
                        const float4 x = __ldcg(at);
                        *at = make_float4(x.x * down, x.y * down, x.z * down, x.w * down);
                    }
                    m_out = m;
                }
                const float g = over ? 1.0f : exp2f(m - m_out);
#pragma unroll 1
                for (int j = 0; j < 4; j++) {
                    unsigned v[32];
                    __syncwarp();
                    tmem_ld32(lane_at + kTmemO + 128 * half + 32 * j, v);
                    if (live && !*wait.abort) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 w = make_float4(__uint_as_float(v[e]) * g, __uint_as_float(v[e + 1]) * g,
                                                         __uint_as_float(v[e + 2]) * g, __uint_as_float(v[e + 3]) * g);
                            float *const to = flushed + (size_t)(32 * half + 8 * j + e / 4) * (kRows * 4);
                            if (over)
                                *reinterpret_cast<float4 *>(to) = w;
                            else
                                asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(w.x), "f"(w.y),
                                             "f"(w.z), "f"(w.w)
                                             : "memory");
                        }
                    }
                }
                __syncwarp();
                tc_fence_before();
                if (over) m_out = m;
            }
            if (fresh) {
                l *= m == -INFINITY ? 0.0f : exp2f(m - m_new);
                m = m_new;
            } else if (__any_sync(0xffffffffu, move)) {
                const float corr = m == -INFINITY ? 0.0f : exp2f(m - m_new);
                __syncwarp();
#pragma unroll 1
                for (int j = 0; j < 4; j++) {
                    unsigned v[32];
                    tmem_ld32(lane_at + kTmemO + 128 * half + 32 * j, v);
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * corr);
                    tmem_st32(lane_at + kTmemO + 128 * half + 32 * j, v);
                }
                tmem_wait_st();
                l *= corr;
                m = m_new;
            }
            const float shift = value_power - ((m == -INFINITY ? 0.0f : m) - kLift);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            __syncwarp();
#pragma unroll
            for (int e0 = 0; e0 < T::kHalf; e0 += 16) {   // per 16 keys: eight words of hi, eight of lo
                float o[16];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float w0 = ex2(fmaf(u[e0 + e], factor, shift)), w1 = ex2(fmaf(u[e0 + e + 1], factor, shift));
                    sum[e & 2] += w0;
                    sum[(e & 2) + 1] += w1;
                    unsigned hi, lo;
                    split_pair(w0, w1, hi, lo);
                    o[e / 2] = __uint_as_float(hi);
                    o[8 + e / 2] = __uint_as_float(lo);
                }
                tmem_st16(s_at + e0, o);
            }
            l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), value_inverse, l);
            if (sum_s != 0.0f) l = fmaf(sum_s, exp2f(most_s - m + kLift), l);
            __syncwarp();
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(w_ready + 8 * (i & 1));
        }
        // ------------------------------------------------------------ epilogue
        wait(o_done + 8 * ((n - 1) & 1), ((n - 1) >> 1) & 1, 59);
        __syncwarp();
        // O leaves through shared memory, where a thread has half a row, in whole rows of 1 KB (the planes and Q are dead:
        // every MMA is done)
        float *const staged = reinterpret_cast<float *>(smem);
        if (!idle) {
            tc_fence_after();
            l += meet(n, l);
            // (O lacks the power that the values' are relative to)
            const float inv = whole ? power(power0) / l : power(power0);
            // part of the row may be in memory; where the last part outweighs that past all bounds, it is dropped
            const bool join = m_out != -INFINITY && m <= m_out + 90.0f;
            const float g = join ? exp2f(m_out - m) : 0.0f;
#pragma unroll 1
            for (int j = 0; j < 4; j++) {
                unsigned v[32];
                __syncwarp();
                tmem_ld32(lane_at + kTmemO + 128 * half + 32 * j, v);
                float *const at = staged + r * kOutPitch + dims_of(j);
                if (join && live) {
                    // (this thread's own stores and additions)
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 old =
                            __ldcg(reinterpret_cast<const float4 *>(flushed + (size_t)(32 * half + 8 * j + e / 4) * (kRows * 4)));
                        v[e] = __float_as_uint(fmaf(old.x, g, __uint_as_float(v[e])));
                        v[e + 1] = __float_as_uint(fmaf(old.y, g, __uint_as_float(v[e + 1])));
                        v[e + 2] = __float_as_uint(fmaf(old.z, g, __uint_as_float(v[e + 2])));
                        v[e + 3] = __float_as_uint(fmaf(old.w, g, __uint_as_float(v[e + 3])));
                    }
                }
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<float4 *>(at + e) =
                        make_float4(__uint_as_float(v[e]) * inv, __uint_as_float(v[e + 1]) * inv,
                                    __uint_as_float(v[e + 2]) * inv, __uint_as_float(v[e + 3]) * inv);
            }
            if (live && half == 0 && !whole && !*wait.abort) {
                const size_t at = 2 * ((size_t)blockIdx.x * kRows + r);
                p.part_ml[at] = l == l ? m : 0.0f;   // (not a number: -infinity would be a run of which the row sees nothing)
                p.part_ml[at + 1] = l;
            }
        }
        named_sync(1, 256);
        if (!*wait.abort) {
#pragma unroll 2
            for (int rr = warp; rr < rows; rr += 8) {
                float4 *const to = reinterpret_cast<float4 *>(whole ? p.out + head_row(rr) * kD
                                                                    : p.part_acc + ((size_t)blockIdx.x * kRows + rr) * kD);
                const float4 *const from = reinterpret_cast<const float4 *>(staged + rr * kOutPitch);
                to[lane] = from[lane];
                to[lane + 32] = from[lane + 32];
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 19) {
        tc_fence_after();
        tmem_dealloc<1>(tmem, 512);
    }
}

template <int kType>
int launch(cudaStream_t stream, const TreeParams &p) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev].load()) {
        const cudaError_t e = cudaFuncSetAttribute(attn_tree_tc<kType>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) configured[dev].store(true);
    }
    return launch_pdl(attn_tree_tc<kType>, dim3(p.grid), dim3(kThreads), (size_t)kSmemBytes, stream, 1, p);
}

}  // namespace

int launch_tree_tc(cudaStream_t stream, const TreeParams &p) {
    return p.kv_dtype == 0 ? launch<0>(stream, p) : p.kv_dtype == 1 ? launch<1>(stream, p) : launch<2>(stream, p);
}

}  // namespace hipml
