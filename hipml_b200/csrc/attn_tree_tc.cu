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
// f16 parts need their operands in range whatever the cache holds. So each key and each value row is scaled by a power of two
// of its own, by its largest scale (f32: value), and each query row too. S is multiplied back (a factor per key and one
// per row); the value's power 2^E goes into the weight: w = 2^(s + E - m), where m follows the largest s + E, and the
// denominator takes w 2^-E. A row that is not finite is zero in the planes and its factors are not a number, so it reaches
// the rows that see it and no others (a hidden key's weight is 0, and 0 times its plane is 0).
//
// Where the time goes (a quantised tile of 64 rows): tensor pipe 2 x 1,536 cycles; shared memory 7.1 KB a row: the raw
// bytes in and out (1.1), the planes (2), K and the low part of Q into the pipe (2.5), V (1.5), 55 cycles a row at 128
// bytes a cycle. So the pipe and shared memory are about balanced, and Q's high part and W come from TMEM for that reason:
// Q hi takes 128 of the 512 columns, O 256, two S tiles 128.
//
// Sums: the tensor cores cut their f32 accumulators off instead of rounding them, 3.5e-9 relative per key of an unbroken
// chain, so every kFlushKeys keys O leaves TMEM for the run's partial in memory (added there, in f32).
//
// Warps 0-7 softmax and epilogue, 8-15 planes, 16 copies, 17 MMAs. Waits are bounded: one that runs out sets the device
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
constexpr int kThreads = 18 * 32;
constexpr int kPlaneThreads = 256;
constexpr int kQChunk = kRows * 128;             // 128 rows x 64 dims, f16
constexpr int kQBytes = 4 * kQChunk;             // one plane of Q
constexpr int kStages = 3, kStageBytes = 32 * 1024;
constexpr int kRawBytes = 3 * 64 * 272;
constexpr int kFlushKeys = 1024;
constexpr unsigned kSpinLimit = 1u << 22;
constexpr float kThreshold = 8.0f;               // log2: the reference moves when a weight would exceed 2^8 times it,
constexpr float kLift = 7.0f;                    // and weights are kept 2^7 times larger: below 2^15, f16's smallest 2^-24
constexpr float kLeastPower = -100.0f;           // of a value row; smaller values count as 0 (as do rows of zeros)

template <int kType>   // 0 f32, 1 q8_0, 2 q4_0
struct Shape {
    static constexpr int kKeys = kType == 0 ? 32 : 64;         // of a tile
    static constexpr int kParts = kType == 0 ? 1 : 2;          // stages of a K (or V) tile, by dims
    static constexpr int kChunks = 4 / kParts;                 // of 64 dims, in a stage
    static constexpr int kChunkBytes = kKeys * 128;
    static constexpr int kPlaneBytes = kChunks * kChunkBytes;  // hi, then lo
    static_assert(2 * kPlaneBytes == kStageBytes, "a stage is two planes");
    // the raw ring: f32 in pieces of 16 rows, padded apart so that eight rows' 16-byte words fall into different banks
    static constexpr int kRowPitch = kType == 0 ? 1040 : (kType == 1 ? 272 : 144);
    static constexpr int kRawRows = kType == 0 ? 16 : 64;
    static constexpr int kRawSlot = kRawRows * kRowPitch;
    static constexpr int kRawSlots = kRawBytes / kRawSlot;
    static constexpr int kPieces = kKeys / kRawRows;           // raw slots of a tile
    static constexpr int kHalf = kKeys / 2;                    // keys of a softmax thread
    // the 32 dims that make block b of part h of a row. Quantised blocks come in pairs (an odd block begins inside a word):
    // a part has one block of each pair, so that eight rows' four pairs fall into different banks.
    __host__ __device__ static constexpr int block(int h, int b) { return kType == 0 ? b : 2 * b + h; }
};

constexpr int kOffQ = 0;                                   // Q lo
constexpr int kOffStages = kOffQ + kQBytes;
constexpr int kOffRaw = kOffStages + kStages * kStageBytes;
constexpr int kOffKey = kOffRaw + kRawBytes;               // [3][64] factor of S, by key
constexpr int kOffPow = kOffKey + 3 * 64 * 4;              // [2][64] E
constexpr int kOffInv = kOffPow + 2 * 64 * 4;              // [2][64] 2^-E
constexpr int kOffMeet = kOffInv + 2 * 64 * 4;             // [2][2][128]: the halves of a row meet
constexpr int kOffRowFac = kOffMeet + 2 * 2 * 128 * 4;     // [128]
constexpr int kOffSees = kOffRowFac + kRows * 4;           // [128][kTreeWords + 1]
constexpr int kOffParents = kOffSees + kRows * (kTreeWords + 1) * 4;
constexpr int kOffBars = kOffParents + kTreeNodes * 4;
constexpr int kSmemNeed = kOffBars + 256;
constexpr int kSmemBytes = kSmemNeed + 1024;               // (the planes lie on 1 KB boundaries)
static_assert(kSmemBytes <= 227 * 1024, "one CTA per SM");
constexpr int kOutPitch = kD + 4;                          // floats of a staged output row
static_assert(kRows * kOutPitch * 4 <= kOffRaw, "the output rows are staged over Q and the planes");

constexpr unsigned kTmemO = 0, kTmemS = 256, kTmemQ = 384;   // columns; S: two tiles of 64

// MN-major operand of 64-dim chunks `pitch` bytes apart, each of rows of 128 bytes (8-row groups 1 KB apart), swizzled.
__device__ __forceinline__ unsigned desc_lo_mn(unsigned addr, unsigned pitch) {
    return ((addr & 0x3ffff) >> 4) | (pitch >> 4) << 16;
}

struct Waits {
    volatile int *abort;
    int *status;
    __device__ __forceinline__ void operator()(unsigned bar, unsigned parity, int code) const {
        for (unsigned i = 0; i < kSpinLimit; i++) {
            if (mbar_try_wait(bar, parity)) return;
            if ((i & 255) == 255 && *abort) return;
            if (i > 4096) __nanosleep(64);
        }
        atomicCAS(status, 0, code);
        *abort = 1;
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

// A quantised block's 32 values (scale `s` in range), as hi and lo words in the order of the dims.
template <int kType>
__device__ __forceinline__ void block_planes(const unsigned *w, bool odd, __half2 s, unsigned (&hi)[16], unsigned (&lo)[16]) {
    if constexpr (kType == 1) {
        // even: codes in bytes 2 .. 33 of w; odd: in whole words from 1 on (word 0 holds the scale)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const unsigned c = (odd ? w[1 + j] : __byte_perm(w[j], w[j + 1], 0x5432)) ^ 0x80808080u;
            // 0x6400 | byte is 1024 + byte
            const __half2 bias = __float2half2_rn(1152.0f);
            const __half2 a = __hsub2(as_half2(__byte_perm(c, 0x64646464u, 0x4140)), bias);
            const __half2 b = __hsub2(as_half2(__byte_perm(c, 0x64646464u, 0x4342)), bias);
            split_product(a, s, hi[2 * j], lo[2 * j]);
            split_product(b, s, hi[2 * j + 1], lo[2 * j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned c = odd ? w[1 + j] : __byte_perm(w[j], w[j + 1], 0x5432);
            const __half2 bias = __float2half2_rn(1032.0f);
            const unsigned even = __byte_perm(c, 0, 0x4140), next = __byte_perm(c, 0, 0x4342);   // bytes 0, 1 and 2, 3
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const unsigned x = e ? next : even;
                split_product(__hsub2(as_half2((x & 0x000f000fu) | 0x64006400u), bias), s, hi[2 * j + e], lo[2 * j + e]);
                split_product(__hsub2(as_half2(((x >> 4) & 0x000f000fu) | 0x64006400u), bias), s, hi[8 + 2 * j + e],
                              lo[8 + 2 * j + e]);
            }
        }
    }
}

// grid tree_grid(.., 128 rows, the device's SMs), 18 warps.
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
    const unsigned raw_full = smem_u32(bars), raw_empty = smem_u32(bars + 5), st_full = smem_u32(bars + 10),
                   st_empty = smem_u32(bars + 13), s_ready = smem_u32(bars + 16), w_ready = smem_u32(bars + 18),
                   o_done = smem_u32(bars + 20), factors = smem_u32(bars + 22), all_done = smem_u32(bars + 24);
    static_assert(T::kRawSlots <= 5, "raw barriers");
    if (tid == 0) {
        for (int i = 0; i < T::kRawSlots; i++) {
            mbar_init(raw_full + 8 * i, 1);
            mbar_init(raw_empty + 8 * i, kPlaneThreads / 32 / T::kPieces);   // the warps that read the slot
        }
        for (int i = 0; i < kStages; i++) {
            mbar_init(st_full + 8 * i, kPlaneThreads / 32);
            mbar_init(st_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(s_ready + 8 * i, 1);
            mbar_init(w_ready + 8 * i, 8);
            mbar_init(o_done + 8 * i, 1);
            mbar_init(factors + 8 * i, kPlaneThreads / 32);
        }
        mbar_init(all_done, 1);
        s_abort = 0;
        mbar_init_fence();
    }
    if (warp == 17) tmem_alloc<1>(smem_u32(&s_tmem), 512);
    tc_fence_before();
    griddep_wait();
    if (warp == 0) {
        const TreeItem it = tree_item(p, tree_quota(p), blockIdx.x);
        if (lane == 0) s_item = it;
    }
    __syncthreads();
    tc_fence_after();
    const TreeItem it = s_item;
    const Waits wait = {&s_abort, p.status};
    const int rows = min(kRows, it.live * p.group - it.tile * kRows);
    const int len = it.base + it.live;
    const int lo_key = it.run * it.quota * kTreeKeyTile, hi_key = min(lo_key + it.quota * kTreeKeyTile, len);
    const int n = it.slot < 0 ? 0 : (hi_key - lo_key + T::kKeys - 1) / T::kKeys;   // tiles
    const size_t first_node = (size_t)it.slot * p.nodes;
    auto head_row = [&](int r) {   // row r of the tile as a row of q and out, in heads
        const int at = it.tile * kRows + r, node = at / p.group;
        return (first_node + node) * p.n_heads + it.kvh * p.group + (at - node * p.group);
    };
    // The tiles' K and V in the order in which the MMAs take them: K0 K1 V0 K2 V1 ... V(n-1).
    const int units = 2 * n;
    auto unit_is_v = [&](int m) { return n == 1 ? m == 1 : (m >= 2 && (m & 1) == 0) || m == units - 1; };
    auto unit_tile = [&](int m) {
        if (m == units - 1) return n - 1;
        return m == 0 ? 0 : ((m & 1) ? (m + 1) / 2 : (m - 2) / 2);
    };
    const size_t slot_at = (size_t)it.slot * p.slot_bytes;
    auto tile_rows = [&](int t) { return min(T::kKeys, hi_key - (lo_key + t * T::kKeys)); };

    if (warp == 16 && n > 0) {
        // ------------------------------------------------------------ copies
        unsigned c = 0;   // raw slots filled
        for (int m = 0; m < units && !*wait.abort; m++) {
            const int t = unit_tile(m), live = tile_rows(t);
            const unsigned char *const cache = (unit_is_v(m) ? p.v : p.k) + slot_at;
            for (int piece = 0; piece < T::kPieces; piece++, c++) {
                const unsigned slot = c % T::kRawSlots, round = c / T::kRawSlots;
                wait(raw_empty + 8 * slot, (round & 1) ^ 1, 51);
                const int key = lo_key + t * T::kKeys + piece * T::kRawRows;
                const int here = min(max(live - piece * T::kRawRows, 0), T::kRawRows);
                const unsigned dst = smem_u32(smem + kOffRaw) + slot * T::kRawSlot, bar = raw_full + 8 * slot;
                const bool go = !*wait.abort;
                if (__any_sync(0xffffffffu, !go)) break;
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
            // what is on its way lands before shared memory is released
            for (unsigned i = c > (unsigned)T::kRawSlots ? c - T::kRawSlots : 0; i < c; i++)
                for (unsigned spin = 0; spin < kSpinLimit; spin++)
                    if (mbar_try_wait(raw_full + 8 * (i % T::kRawSlots), (i / T::kRawSlots) & 1)) break;
        }
    }

    if (warp < 16 && n > 0) {
        // ------------------------------------------------------------ Q: eight rows a warp
        float4 x[8][2];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = warp * 8 + j;
            x[j][0] = x[j][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r < rows) {
                const float4 *const src = reinterpret_cast<const float4 *>(p.q + head_row(r) * kD) + 2 * lane;
                x[j][0] = __ldg(src);
                x[j][1] = __ldg(src + 1);
            }
        }
        for (int i = tid; i < it.live; i += 512)
            reinterpret_cast<int *>(smem + kOffParents)[i] = p.parents[first_node + i];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = warp * 8 + j;
            const float v[8] = {x[j][0].x, x[j][0].y, x[j][0].z, x[j][0].w, x[j][1].x, x[j][1].y, x[j][1].z, x[j][1].w};
            float most = 0.0f;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                most = fmaxf(most, fabsf(v[e]));
                bad = bad || !(fabsf(v[e]) < INFINITY);
            }
            most = warp_max(most);
            bad = __any_sync(0xffffffffu, bad);
            // the row's largest value comes to [2^10, 2^11)
            const int e = bad ? 0 : min(max(((__float_as_int(most) >> 23) & 255) - 127 - 10, -116), 116);
            const float f = power(-e);
            if (lane == 0)
                reinterpret_cast<float *>(smem + kOffRowFac)[r] =
                    bad ? __int_as_float(0x7fffffff) : power(e) * p.scale_log2;
            unsigned h[4], l[4];
#pragma unroll
            for (int k = 0; k < 4; k++) split_pair(bad ? 0.0f : v[2 * k] * f, bad ? 0.0f : v[2 * k + 1] * f, h[k], l[k]);
            // Position of dims 8 * lane .. in the order of the parts: block b of part h stands at 128 h + 32 b (f32: 32 b)
            const int blk = lane >> 2;
            const int at = kType == 0 ? 8 * lane : 128 * (blk & 1) + 32 * (blk >> 1) + 8 * (lane & 3);
            const int off = (at >> 6) * kQChunk + sw128_offset(r, at & 63);
            *reinterpret_cast<uint4 *>(smem + kOffQ + off) = make_uint4(l[0], l[1], l[2], l[3]);
            // (hi goes to TMEM by way of the first stages)
            *reinterpret_cast<uint4 *>(smem + kOffStages + off) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        named_sync(1, 512);
        if (warp < 8) {
            // thread (row, half) takes half of the row's hi plane to TMEM
            const int r = tid & 127, half = tid >> 7;
            const unsigned to = s_tmem + kTmemQ + 64 * half + ((unsigned)((warp & 3) * 32) << 16);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                unsigned q[32];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(smem + kOffStages + (2 * half + c) * kQChunk +
                                                                     sw128_offset(r, 8 * j));
                    q[4 * j] = w.x;
                    q[4 * j + 1] = w.y;
                    q[4 * j + 2] = w.z;
                    q[4 * j + 3] = w.w;
                }
                tmem_st32(to + 32 * c, q);
            }
            tmem_wait_st();
            if (half == 0 && hi_key > it.base) {
                // which drafted rows this row sees (rows past the last: those of the last)
                unsigned words[kTreeWords];
                tree_ancestors(reinterpret_cast<const int *>(smem + kOffParents), (it.tile * kRows + min(r, rows - 1)) / p.group,
                               words, p.status);
                unsigned *const at = reinterpret_cast<unsigned *>(smem + kOffSees) + r * (kTreeWords + 1);
#pragma unroll
                for (int w = 0; w < kTreeWords; w++) at[w] = words[w];
                at[kTreeWords] = 0;
            }
        }
        fence_async_shared();
    }
    tc_fence_before();
    if (warp != 16) named_sync(6, kThreads - 32);   // (the copies go on meanwhile)
    tc_fence_after();
    const unsigned tmem = s_tmem;

    if (warp == 17) {
        // ------------------------------------------------------------ MMAs
        if (lane == 0 && n > 0) {
            constexpr unsigned kMn = 1u << 16;   // B with N contiguous
            constexpr unsigned kIdescS = idesc_f16(128, T::kKeys), kIdescO = idesc_f16(128, 64 * T::kChunks) | kMn;
            const unsigned q_lo = desc_lo_sw128(smem_u32(smem + kOffQ)), stages = smem_u32(smem + kOffStages);
            unsigned c = 0;   // stages consumed
            auto stage = [&](int code) {
                wait(st_full + 8 * (c % kStages), (c / kStages) & 1, code);
                tc_fence_after();
                return stages + (c % kStages) * kStageBytes;
            };
            auto release = [&]() {
                tc_commit<1>(st_empty + 8 * (c % kStages));
                c++;
            };
            auto qk = [&](int i) {
                const unsigned d = tmem + kTmemS + 64 * (i & 1);
                for (int h = 0; h < T::kParts; h++) {
                    const unsigned at = stage(52);
                    if (*wait.abort) return;
#pragma unroll
                    for (int ch = 0; ch < T::kChunks; ch++) {
                        const unsigned hi = desc_lo_sw128(at + ch * T::kChunkBytes);
                        const unsigned lo = desc_lo_sw128(at + T::kPlaneBytes + ch * T::kChunkBytes);
                        const int chunk = h * T::kChunks + ch;
                        const unsigned qh = tmem + kTmemQ + 32 * chunk, ql = q_lo + chunk * (kQChunk >> 4);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tc_mma_ts<1>(d, qh + 8 * k, desc_from(lo + 2 * k), kIdescS, (h | ch | k) != 0);
#pragma unroll
                        for (int k = 0; k < 4; k++) tc_mma_ss<1>(d, desc_from(ql + 2 * k), desc_from(hi + 2 * k), kIdescS, 1);
#pragma unroll
                        for (int k = 0; k < 4; k++) tc_mma_ts<1>(d, qh + 8 * k, desc_from(hi + 2 * k), kIdescS, 1);
                    }
                    release();
                }
                tc_commit<1>(s_ready + 8 * (i & 1));
            };
            auto pv = [&](int i) {
                const unsigned a = tmem + kTmemS + 64 * (i & 1);
                const unsigned later = (i * T::kKeys) % kFlushKeys != 0;   // 0: O starts afresh
                for (int h = 0; h < T::kParts; h++) {
                    const unsigned at = stage(53);
                    if (*wait.abort) return;
                    const unsigned d = tmem + kTmemO + 128 * h;
                    const unsigned hi = desc_lo_mn(at, T::kChunkBytes), lo = desc_lo_mn(at + T::kPlaneBytes, T::kChunkBytes);
#pragma unroll
                    for (int k = 0; k < T::kKeys / 16; k++) {   // 16 keys: two groups of eight rows
                        tc_mma_ts<1>(d, a + 16 * k, desc_from(lo + 128 * k), kIdescO, k == 0 ? later : 1);
                        tc_mma_ts<1>(d, a + 16 * k + 8, desc_from(hi + 128 * k), kIdescO, 1);
                        tc_mma_ts<1>(d, a + 16 * k, desc_from(hi + 128 * k), kIdescO, 1);
                    }
                    release();
                }
                tc_commit<1>(o_done + 8 * (i & 1));
            };
            qk(0);
            for (int i = 0; i < n && !*wait.abort; i++) {
                if (i + 1 < n) qk(i + 1);
                if (*wait.abort) break;
                wait(w_ready + 8 * (i & 1), (i >> 1) & 1, 54);
                if (*wait.abort) break;
                tc_fence_after();
                pv(i);
            }
            if (*wait.abort) {
                tc_commit<1>(all_done);
                for (unsigned spin = 0; spin < kSpinLimit && !mbar_try_wait(all_done, 0); spin++) {}
            }
        }
    } else if (warp >= 8 && warp < 16) {
        // ------------------------------------------------------------ planes
        const int w8 = warp - 8;
        unsigned c_raw = 0, c = 0;
        float *const key_factor = reinterpret_cast<float *>(smem + kOffKey);
        float *const value_power = reinterpret_cast<float *>(smem + kOffPow);
        float *const value_inverse = reinterpret_cast<float *>(smem + kOffInv);
        auto take_stage = [&]() {
            wait(st_empty + 8 * (c % kStages), ((c / kStages) & 1) ^ 1, 55);
            return smem + kOffStages + (c % kStages) * kStageBytes;
        };
        auto give_stage = [&]() {
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(st_full + 8 * (c % kStages));
            c++;
        };
        for (int m = 0; m < units; m++) {
            const int t = unit_tile(m), live = tile_rows(t);
            const bool is_v = unit_is_v(m);
            if constexpr (kType == 0) {
                // thread: block lane / 4 of row 4 * (warp - 8) + lane % 4
                const int key = 4 * w8 + (lane & 3), blk = lane >> 2;
                const unsigned mine = c_raw + (w8 >> 2), slot = mine % T::kRawSlots;
                wait(raw_full + 8 * slot, (mine / T::kRawSlots) & 1, 56);
                float x[32];   // an odd block's halves are swapped: eight lanes' words fall into different banks
                const float4 *const src = reinterpret_cast<const float4 *>(smem + kOffRaw + slot * T::kRawSlot +
                                                                           (key & 15) * T::kRowPitch + blk * 128);
                float most = 0.0f;
                bool bad = false;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (key < live) w = src[j ^ ((blk & 1) << 2)];
                    x[4 * j] = w.x;
                    x[4 * j + 1] = w.y;
                    x[4 * j + 2] = w.z;
                    x[4 * j + 3] = w.w;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        most = fmaxf(most, fabsf(x[4 * j + e]));
                        bad = bad || !(fabsf(x[4 * j + e]) < INFINITY);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(raw_empty + 8 * slot);
                c_raw += T::kPieces;
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const unsigned whose = 0x11111111u << (lane & 3);
                bad = (__ballot_sync(0xffffffffu, bad) & whose) != 0;
                const int top = (__float_as_int(most) >> 23) & 255;
                int e = min(max(top - 127 - 10, (int)kLeastPower), 116);   // (a row of zeros: the least)
                if (bad) e = 0;
                const float f = bad ? 0.0f : power(-e);
                unsigned char *const st = take_stage();
                if (blk == 0) {
                    if (is_v) {
                        value_power[64 * (t & 1) + key] = (float)e;
                        value_inverse[64 * (t & 1) + key] = bad ? __int_as_float(0x7fffffff) : power(-e);
                    } else {
                        key_factor[64 * (t % 3) + key] = bad ? __int_as_float(0x7fffffff) : power(e);
                    }
                }
                unsigned char *const dst = st + (blk >> 1) * T::kChunkBytes + key * 128;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    unsigned h[4], l[4];
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        split_pair(bad ? 0.0f : x[8 * j + 2 * k] * f, bad ? 0.0f : x[8 * j + 2 * k + 1] * f, h[k], l[k]);
                    const int u = 4 * (blk & 1) + (j ^ ((blk & 1) << 1));
                    const int at = (u ^ (key & 7)) << 4;
                    *reinterpret_cast<uint4 *>(dst + at) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(dst + T::kPlaneBytes + at) = make_uint4(l[0], l[1], l[2], l[3]);
                }
                give_stage();
            } else {
                // thread: pair lane / 8 of row 8 * (warp - 8) + lane % 8; one block of it in each part
                constexpr int kPair = kType == 1 ? 17 : 9, kOdd = kType == 1 ? 8 : 4;   // words; the odd block's first
                const int key = 8 * w8 + (lane & 7), pair = lane >> 3;
                const unsigned slot = c_raw % T::kRawSlots;
                wait(raw_full + 8 * slot, (c_raw / T::kRawSlots) & 1, 56);
                const unsigned *const src = reinterpret_cast<const unsigned *>(smem + kOffRaw + slot * T::kRawSlot +
                                                                               key * T::kRowPitch) + pair * kPair;
                unsigned w[kPair];
#pragma unroll
                for (int j = 0; j < kPair; j++) w[j] = key < live ? src[j] : 0u;
                __syncwarp();
                if (lane == 0) mbar_arrive(raw_empty + 8 * slot);
                c_raw++;
                const unsigned s0 = w[0] & 0xffffu, s1 = w[kOdd] >> 16;   // the scales' bits
                int most = max((int)(s0 & 0x7fffu), (int)(s1 & 0x7fffu));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 8));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 16));
                const bool bad = most >= 0x7c00;
                // the row's largest scale comes to [8, 16): codes times it stay below 2^11 and lo is exact
                int e = most == 0 ? (int)kLeastPower : max(most >> 10, 1) - 15 - 3;
                if (bad) e = 0;
                if (!is_v && most == 0) e = 0;
                const float f = bad || most == 0 ? 0.0f : power(-e);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    unsigned hi[16], lo[16];
                    const float s = half_bits_to_float((uint16_t)(h ? s1 : s0));
                    block_planes<kType>(w + (h ? kOdd : 0), h != 0, __float2half2_rn(bad ? 0.0f : s * f), hi, lo);
                    unsigned char *const st = take_stage();
                    if (h == 0 && pair == 0) {
                        if (is_v) {
                            value_power[64 * (t & 1) + key] = (float)e;
                            value_inverse[64 * (t & 1) + key] = bad ? __int_as_float(0x7fffffff) : power(-e);
                        } else {
                            key_factor[64 * (t % 3) + key] = bad ? __int_as_float(0x7fffffff) : power(e);
                        }
                    }
                    unsigned char *const dst = st + (pair >> 1) * T::kChunkBytes + key * 128;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int at = ((4 * (pair & 1) + j) ^ (key & 7)) << 4;
                        *reinterpret_cast<uint4 *>(dst + at) = make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
                        *reinterpret_cast<uint4 *>(dst + T::kPlaneBytes + at) =
                            make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
                    }
                    give_stage();
                }
            }
            if (is_v) {   // this tile's factors of K and V are there
                if (lane == 0) mbar_arrive(factors + 8 * (t & 1));
            }
        }
    } else if (warp < 8 && n > 0) {
        // ------------------------------------------------------------ softmax
        const int r = tid & 127, half = tid >> 7;
        const unsigned lane_at = tmem + ((unsigned)((warp & 3) * 32) << 16);
        const float row_factor = reinterpret_cast<const float *>(smem + kOffRowFac)[r];
        const bool live = r < rows, whole = it.runs == 1;
        float *const dst = (whole ? p.out + head_row(min(r, rows - 1)) * kD
                                  : p.part_acc + ((size_t)blockIdx.x * kRows + r) * kD);
        float m = -INFINITY, l = 0.0f, m_out = -INFINITY;   // m_out: the reference of what is in memory already
        // the other half's value of the row (the warps w and w + 4 meet)
        auto meet = [&](int x, float mine) {
            float *const buf = reinterpret_cast<float *>(smem + kOffMeet) + (x & 1) * 256;
            buf[128 * half + r] = mine;
            named_sync(2 + (warp & 3), 64);
            return buf[128 * (half ^ 1) + r];
        };
        // dims of column group j (32 columns) of this thread's half of O
        auto dims_of = [&](int j) { return kType == 0 ? 128 * half + 32 * j : 32 * T::block(half, j); };
        for (int i = 0; i < n; i++) {
            const unsigned s_at = lane_at + kTmemS + 64 * (i & 1) + T::kHalf * half;
            wait(s_ready + 8 * (i & 1), (i >> 1) & 1, 57);
            wait(factors + 8 * (i & 1), (i >> 1) & 1, 58);
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
            const float4 *const kf = reinterpret_cast<const float4 *>(smem + kOffKey) + 16 * (i % 3) + T::kHalf / 4 * half;
            const float4 *const vp = reinterpret_cast<const float4 *>(smem + kOffPow) + 16 * (i & 1) + T::kHalf / 4 * half;
            const float4 *const vi = reinterpret_cast<const float4 *>(smem + kOffInv) + 16 * (i & 1) + T::kHalf / 4 * half;
#pragma unroll
            for (int e = 0; e < T::kHalf; e += 4) {
                const float4 f = kf[e / 4], g = vp[e / 4];
                u[e] = fmaf(u[e] * f.x, row_factor, g.x);
                u[e + 1] = fmaf(u[e + 1] * f.y, row_factor, g.y);
                u[e + 2] = fmaf(u[e + 2] * f.z, row_factor, g.z);
                u[e + 3] = fmaf(u[e + 3] * f.w, row_factor, g.w);
            }
            const int key0 = lo_key + i * T::kKeys + T::kHalf * half;
            unsigned sees = 0xffffffffu;
            if (lo_key + (i + 1) * T::kKeys > it.base) {   // drafted rows, and none past the last
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
            float big[4] = {u[0], u[1], u[2], u[3]};
#pragma unroll
            for (int e = 4; e < T::kHalf; e += 4)
#pragma unroll
                for (int k = 0; k < 4; k++) big[k] = fmaxf(big[k], u[e + k]);
            float m_new = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
            m_new = fmaxf(m, fmaxf(m_new, meet(i, m_new)));
            const bool fresh = (i * T::kKeys) % kFlushKeys == 0;   // O starts afresh with this tile
            const bool flush = fresh && i > 0;
            const bool move = !fresh && (m_new > m + kThreshold || (m == -INFINITY && m_new > -INFINITY));
            if (flush || __any_sync(0xffffffffu, move)) {
                wait(o_done + 8 * ((i - 1) & 1), ((i - 1) >> 1) & 1, 59);
                __syncwarp();
                tc_fence_after();
            }
            if (flush) {
                // O, relative to m, is added to what is in memory (or takes its place, where that is nothing beside it)
                const bool over = m_out == -INFINITY || m > m_out + 60.0f;
                const float g = over ? 1.0f : exp2f(m - m_out);
#pragma unroll 1
                for (int j = 0; j < 4; j++) {
                    unsigned v[32];
                    tmem_ld32(lane_at + kTmemO + 128 * half + 32 * j, v);
                    if (!live || *wait.abort) continue;
                    float *const to = dst + dims_of(j);
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 w = make_float4(__uint_as_float(v[e]) * g, __uint_as_float(v[e + 1]) * g,
                                                     __uint_as_float(v[e + 2]) * g, __uint_as_float(v[e + 3]) * g);
                        if (over)
                            *reinterpret_cast<float4 *>(to + e) = w;
                        else
                            asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to + e), "f"(w.x), "f"(w.y),
                                         "f"(w.z), "f"(w.w)
                                         : "memory");
                    }
                }
                tc_fence_before();
                if (over) m_out = m;
            }
            if (fresh) {
                l *= m == -INFINITY ? 0.0f : exp2f(m - m_new);
                m = m_new;
            } else if (__any_sync(0xffffffffu, move)) {
                const float corr = m == -INFINITY ? 0.0f : exp2f(m - m_new);
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
            const float ref = (m == -INFINITY ? 0.0f : m) - kLift;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            unsigned o[T::kHalf];
#pragma unroll
            for (int e = 0; e < T::kHalf; e += 4) {
                const float4 g = vi[e / 4];
                const float w0 = ex2(u[e] - ref), w1 = ex2(u[e + 1] - ref), w2 = ex2(u[e + 2] - ref), w3 = ex2(u[e + 3] - ref);
                // (a hidden row's inverse may be not a number)
                sum[0] = sees >> e & 1 ? fmaf(w0, g.x, sum[0]) : sum[0];
                sum[1] = sees >> (e + 1) & 1 ? fmaf(w1, g.y, sum[1]) : sum[1];
                sum[2] = sees >> (e + 2) & 1 ? fmaf(w2, g.z, sum[2]) : sum[2];
                sum[3] = sees >> (e + 3) & 1 ? fmaf(w3, g.w, sum[3]) : sum[3];
                const int at = (e >> 4) * 16 + ((e & 15) >> 1);   // per 16 keys: eight words of hi, eight of lo
                split_pair(w0, w1, o[at], o[at + 8]);
                split_pair(w2, w3, o[at + 1], o[at + 9]);
            }
            if constexpr (T::kHalf == 32) {
                tmem_st32(s_at, o);
            } else {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; e++) v[e] = __uint_as_float(o[e]);
                tmem_st16(s_at, v);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(w_ready + 8 * (i & 1));
        }
        // ------------------------------------------------------------ epilogue
        l += meet(n, l);
        wait(o_done + 8 * ((n - 1) & 1), ((n - 1) >> 1) & 1, 59);
        __syncwarp();
        tc_fence_after();
        // O leaves through shared memory: whole rows of 1 KB by bulk copies (the planes and Q are dead: every MMA is done)
        float *const staged = reinterpret_cast<float *>(smem);
        const bool apart = m_out != -INFINITY;   // part of the row is in memory
        const float g = apart ? exp2f(m - m_out) : 1.0f;
        const float inv = whole ? 1.0f / l : 1.0f;
        // (where the last part outweighs what is in memory past all bounds, that is dropped)
        const bool drop = apart && m > m_out + 60.0f;
#pragma unroll 1
        for (int j = 0; j < 4; j++) {
            unsigned v[32];
            tmem_ld32(lane_at + kTmemO + 128 * half + 32 * j, v);
            float *const at = staged + r * kOutPitch + dims_of(j);
            if (live && !*wait.abort) {
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    float4 w = make_float4(__uint_as_float(v[e]), __uint_as_float(v[e + 1]), __uint_as_float(v[e + 2]),
                                           __uint_as_float(v[e + 3]));
                    if (apart && !drop) {
                        // (this thread's own stores and additions)
                        const float4 old = __ldcg(reinterpret_cast<const float4 *>(dst + dims_of(j) + e));
                        w.x = fmaf(w.x, g, old.x);
                        w.y = fmaf(w.y, g, old.y);
                        w.z = fmaf(w.z, g, old.z);
                        w.w = fmaf(w.w, g, old.w);
                    }
                    const float s = apart && !drop ? inv / g : inv;
                    *reinterpret_cast<float4 *>(at + e) = make_float4(w.x * s, w.y * s, w.z * s, w.w * s);
                }
            }
        }
        if (live && half == 0 && !whole && !*wait.abort) {
            const size_t at = 2 * ((size_t)blockIdx.x * kRows + r);
            p.part_ml[at] = m;
            p.part_ml[at + 1] = l;
        }
        fence_async_shared();
        named_sync(1, 256);
        if (!*wait.abort && lane == 0) {
            for (int rr = warp; rr < rows; rr += 8)
                bulk_store(whole ? p.out + head_row(rr) * kD : p.part_acc + ((size_t)blockIdx.x * kRows + rr) * kD,
                           smem_u32(staged + rr * kOutPitch), kD * 4);
            bulk_store_commit_wait_read();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
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
