// Products in 8-bit integers with a scale for each row and each channel, for one matrix or for the
// matrix of each expert over its segment of sorted rows:
//
//   out[r, c] = float(sum_i q[r, i] w[c, i]) * q_scale[r] * w_scale[c] + bias[c]
//
// The sum is exact: 32-bit integers hold it for up to 131,071 terms.  The tensor cores (tcgen05
// kind::i8) take 128 channels as the rows of a tile and kRows of the product's rows as its columns,
// so that one row costs a tile 16 wide, and a warp of the epilogue, whose 32 lanes hold 32
// neighbouring channels, writes 32 neighbouring elements of a row.
//
// What bounds it on B200 (2 x the measured bfloat16 rate is 3.37 POP/s, memory 6.54 TB/s):
//   16,384 x 4,096 x 4,096    165 us, 3.33 POP/s: the tensor cores (78 % busy in a capture, at 1.6 GHz: power)
//   4,096 x 65,536 x 128      168 us, 6.4 TB/s: writing 32-bit results
//   1 x 4,096 x 4,096         6.5 us: the latency of a launch and of a cluster's sum (2.6 us of weights, which stay in
//   the L2 cache when calls repeat)
//   8 tokens x 8 of 128 experts, 1,024 x 2,048 each: 23 us, 4.7 TB/s of weights; three rounds of 2.76 tiles an SM cost 8 %
//   of it, the segments are found before the first load, the rest is not accounted for
//   32,768 rows over 64 experts, 2,048 x 2,048 each: 122 to 127 us (82 by the tensor cores, 72 by memory).  Neither is
//   busy throughout: in a capture of half the size the tensor cores work 57 % of the time and memory moves at 48 % of
//   its rate; the last round of tiles costs 5 %, and tiles of 256 rows cover 23 % more rows than there are
//   131,072 rows of 64 experts, 2,048 x 4,096 each: 809 us, and 1,371 when half of them have no expert: their zeros take a
//   64-bit division an element, after the tiles
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "provider.h"
#include "tc_ptx.cuh"

namespace {

using stlq_b200::Aligned;
using stlq_b200::Bad;
using stlq_b200::Ck;
using stlq_b200::DeviceScope;
using stlq_b200::Guard;
using stlq_b200::LetLaterStart;
using stlq_b200::SetError;
using stlq_b200::WaitForEarlier;
namespace tc = stlq_b200::tc;

constexpr int kChannels = 128;                       // channels of a CTA's tile (its share of the MMA's M)
constexpr int kTileK = 128;                          // bytes of a 128-byte swizzle row
constexpr uint32_t kWBytes = kChannels * kTileK;
constexpr int kBoxRows = 32;                         // rows come in boxes of these where a tile has fewer than its height
constexpr int kWriters = 8;                          // warps of the epilogue
constexpr int kShare = kWriters / 4;                 // of them, those of a quarter of the TMEM lanes
constexpr int kThreads = 64 + 32 * kWriters;         // warp 0 loads, warp 1 multiplies, the others write
constexpr uint64_t kWaitNs = 2000000000ull;          // 2 s per barrier wait

// kOne: a CTA computes tiles of its own, one after the other.  kPair: two CTAs share a tile of 256
// channels (tcgen05 cta_group::2): each holds its channels and half of the rows, so that an operand
// byte in shared memory is used twice as often.  kSplit: the CTAs of a cluster each sum a part of kdim
// for one tile and add up over distributed shared memory, for products with few tiles.
enum Mode { kOne, kPair, kSplit };

template <int kRows, Mode kMode, typename T>
struct Shape {
    static constexpr int kXRows = kMode == kPair ? kRows / 2 : kRows;  // rows that a CTA holds of a full tile
    static constexpr uint32_t kXBytes = kXRows * kTileK;
    static constexpr uint32_t kStageBytes = kWBytes + kXBytes;
    // A writing warp takes this many rows of its 32 channels at a time, and lays them out for a TMA store, twice.
    static constexpr int kChunk = kMode != kSplit && kRows >= 128 ? 32 : 16;
    static constexpr uint32_t kOutBytes = kChunk * 32 * sizeof(T);
    static constexpr uint32_t kAllOut = kMode == kSplit ? 0 : 2 * kWriters * kOutBytes;
    static constexpr int kStages = std::min<int>(10, (209 * 1024 - kAllOut) / kStageBytes);
    static constexpr int kColumns = kRows < 32 ? 32 : kRows;        // TMEM columns of one accumulator
    static constexpr uint32_t kTmem = (kMode == kSplit ? 1 : 2) * kColumns;  // two: one is written out while the next is made
    static constexpr int kTileChannels = kMode == kPair ? 2 * kChannels : kChannels;
    static constexpr int kOwnRows = std::max(kChunk, kRows / kShare);   // rows of the tile that a writing warp takes
    static constexpr int kGranule = kMode == kPair ? 32 : 16;       // rows of an MMA come in multiples of this
};

// A wait that ran out raises *err, which stays raised until stlq_b200_kernels_sync reports it.  No wait gives up because it is
// raised: it may be from an earlier call, and what that one lost would then cost later calls their results.  A block whose wait
// ran out ends its loops, and whoever waits for it runs out in turn.
__device__ __forceinline__ bool Wait(uint64_t* bar, uint32_t parity, unsigned int* err) {
    return tc::MbarWait(bar, parity, err, kWaitNs, false);
}

struct MatmulArgs {
    const float* q_scale;
    const float* w_scale;
    const float* bias;
    const int* offsets;  // null: one matrix, all rows
    int experts, rows, n, kdim;
    int tma_n;           // channels that TMA may write: see Matmul
    int evict_first;     // the output is larger than the L2 cache's share for it
    int band;            // row tiles that run side by side over the channels
    void* out;
    int64_t ldo;
    unsigned int* err;
};

template <typename T>
__device__ __forceinline__ T Out(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
    else return __float2half_rn(v);
}

// Tile `id`: its expert, first row, end of its expert's rows, first channel.
struct Tile {
    int expert, row0, end, channel0;
};

// The segments of the experts, in shared memory: first[e] is the number of tiles before expert e's,
// begin[e] / end[e] its rows, within the product's.  Rows before begin[0] and from the last end on have no expert.
struct Segments {
    int* first;
    int* begin;
    int* end;
};

// Fills sg from the offsets, by the kThreads threads of a block; `ct` tiles for every kRows rows or part of them.  The block
// synchronises before it reads them.
template <int kRows, int kThreads>
__device__ __forceinline__ void FindSegments(const MatmulArgs& a, const Segments& sg, int ct) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int e = threadIdx.x; e < a.experts; e += kThreads) sg.end[e] = min(max(a.offsets[e + 1], 0), a.rows);
    __syncthreads();
    if (warp != 0) return;
    int before = 0, top = min(max(a.offsets[0], 0), a.rows);
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
        const int e = e0 + lane;
        // A segment begins where the one before it ended: a running maximum, so that offsets
        // in any order give segments that do not overlap.
        int end = e < a.experts ? sg.end[e] : 0;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end = max(end, y);
        }
        end = max(end, top);
        int begin = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) begin = top;
        top = __shfl_sync(0xffffffffu, end, 31);
        int s = e < a.experts ? (end - begin + kRows - 1) / kRows * ct : 0;
        const int mine = s;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        if (e < a.experts) {
            sg.begin[e] = begin;
            sg.end[e] = end;
            sg.first[e] = before + s - mine;
        }
        before += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) sg.first[a.experts] = before;
}

template <int kRows, int kTileChannels>
__device__ __forceinline__ Tile FindTile(const MatmulArgs& a, const Segments& sg, int id) {
    Tile t;
    const int ct = (a.n + kTileChannels - 1) / kTileChannels;
    int local = id;
    if (a.offsets) {
        int lo = 0, hi = a.experts;  // the last expert whose tiles begin at or before id
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sg.first[mid] <= id) lo = mid;
            else hi = mid;
        }
        t.expert = lo;
        t.row0 = sg.begin[lo];
        t.end = sg.end[lo];
        local = id - sg.first[lo];
    } else {
        t.expert = 0;
        t.row0 = 0;
        t.end = a.rows;
    }
    // Bands of row tiles, the band's row tiles running fastest.
    const int rt = (t.end - t.row0 + kRows - 1) / kRows;
    const int band = local / (a.band * ct), in = local - band * a.band * ct;
    const int height = min(a.band, rt - band * a.band);
    t.channel0 = in / height * kTileChannels;
    t.row0 += (band * a.band + in % height) * kRows;
    return t;
}

template <int kRows, Mode kMode, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    MatmulI8Kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                   const __grid_constant__ CUtensorMap tx_part, const __grid_constant__ CUtensorMap to, const MatmulArgs a,
                   int cluster) {
    using S = Shape<kRows, kMode, T>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = smem_raw + ((1024 - (tc::SmemAddr(smem_raw) & 1023)) & 1023);
    unsigned char* outs = base + S::kStages * S::kStageBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(outs + S::kAllOut);
    uint64_t* empty = full + S::kStages;
    uint64_t* made = empty + S::kStages;  // an accumulator is complete
    uint64_t* taken = made + 2;           // an accumulator has been read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(taken + 2);
    float* row_scales = reinterpret_cast<float*>(tmem_slot + 4);  // [kWriters][kOwnRows]
    Segments sg;
    sg.first = reinterpret_cast<int*>(row_scales + kWriters * S::kOwnRows);
    sg.begin = sg.first + (a.experts + 1);
    sg.end = sg.begin + a.experts;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = kMode == kOne ? 0 : static_cast<int>(tc::ClusterRank());
    const int ct = (a.n + S::kTileChannels - 1) / S::kTileChannels;
    const int nk = (a.kdim + kTileK - 1) / kTileK;
    // The steps of kdim that this CTA sums (all, but for kSplit).
    const int k_first = kMode == kSplit ? static_cast<int>(static_cast<int64_t>(nk) * rank / cluster) : 0;
    const int k_last = kMode == kSplit ? static_cast<int>(static_cast<int64_t>(nk) * (rank + 1) / cluster) : nk;
    const int first_tile = kMode == kOne ? blockIdx.x : blockIdx.x / cluster;
    const int tile_step = kMode == kOne ? gridDim.x : gridDim.x / cluster;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            tc::MbarInit(&full[s], 1);
            tc::MbarInit(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::MbarInit(&made[b], 1);
            tc::MbarInit(&taken[b], kMode == kPair ? 2 * kWriters : kWriters);
        }
        tc::FenceBarrierInit();
    }
    if (warp == 1) {
        if constexpr (kMode == kPair) tc::TmemAllocPair(tmem_slot, S::kTmem);
        else tc::TmemAlloc(tmem_slot, S::kTmem);
    }
    LetLaterStart();
    WaitForEarlier();
    if (a.offsets) FindSegments<kRows, kThreads>(a, sg, ct);
    tc::FenceBeforeSync();
    if constexpr (kMode == kPair) {
        __syncthreads();
        tc::ClusterSync();  // the pair's barriers exist before either arrives on them
    } else {
        __syncthreads();
    }
    tc::FenceAfterSync();
    const uint32_t tmem = *tmem_slot;
    const int tiles = a.offsets ? sg.first[a.experts] : (a.rows + kRows - 1) / kRows * ct;
    // Rows of a tile's MMA: what is left of the segment, rounded up.
    auto columns = [](const Tile& t) { return min(kRows, (t.end - t.row0 + S::kGranule - 1) / S::kGranule * S::kGranule); };

    // The two warps that load and multiply run converged, with one lane issuing: addresses and
    // descriptors then stay in uniform registers, and a step costs the issuing thread few instructions
    // (with a loop of lane 0's own, a step of four MMAs took 285 ns whatever the tile).
    if (warp == 0) {
        const bool one = tc::ElectOne();
        int s = 0, used = 0;         // the stage, and how many have been filled
        uint32_t parity = 1;         // of the wait for its last use
        bool ok = true;
        for (int id = first_tile; id < tiles && ok; id += tile_step) {
            const Tile t = FindTile<kRows, S::kTileChannels>(a, sg, id);
            const int wrow = t.expert * a.n + t.channel0 + (kMode == kPair ? rank * kChannels : 0);
            const int xrow = t.row0 + (kMode == kPair ? rank * (columns(t) / 2) : 0);
            // The last tile of a segment loads the rows that it has: it would take as long as a full one otherwise.
            const int boxes = S::kXRows <= kBoxRows ? 1 : (columns(t) * S::kXRows / kRows + kBoxRows - 1) / kBoxRows;
            const bool whole = S::kXRows <= kBoxRows || boxes * kBoxRows == S::kXRows;
            const uint32_t bytes = kWBytes + (whole ? S::kXBytes : boxes * kBoxRows * kTileK);
            for (int kb = k_first; kb < k_last; ++kb) {
                if (used >= S::kStages && !(ok = __all_sync(0xffffffffu, Wait(&empty[s], parity, a.err)))) break;
                unsigned char* st = base + s * S::kStageBytes;
                if (one) {
                    if constexpr (kMode == kPair) {
                        // The even CTA's barrier counts the bytes of both.
                        if (rank == 0) tc::MbarArriveExpectTx(&full[s], 2 * bytes);
                        const uint32_t bar = tc::ClusterAddr(&full[s], 0);
                        tc::TmaLoad2dPair(st, &tw, bar, kb * kTileK, wrow);
                        if (whole) tc::TmaLoad2dPair(st + kWBytes, &tx, bar, kb * kTileK, xrow);
                        else
                            for (int i = 0; i < boxes; ++i)
                                tc::TmaLoad2dPair(st + kWBytes + i * kBoxRows * kTileK, &tx_part, bar, kb * kTileK, xrow + i * kBoxRows);
                    } else {
                        tc::MbarArriveExpectTx(&full[s], bytes);
                        tc::TmaLoad2d(st, &tw, &full[s], kb * kTileK, wrow);
                        if (whole) tc::TmaLoad2d(st + kWBytes, &tx, &full[s], kb * kTileK, xrow);
                        else
                            for (int i = 0; i < boxes; ++i)
                                tc::TmaLoad2d(st + kWBytes + i * kBoxRows * kTileK, &tx_part, &full[s], kb * kTileK, xrow + i * kBoxRows);
                    }
                }
                __syncwarp();
                used = min(used + 1, 2 * S::kStages);
                if (++s == S::kStages) {
                    s = 0;
                    parity ^= 1;
                }
            }
        }
        // Copies still in flight land before the block may exit: the last use of each stage.
        if (kMode != kPair || rank == 0)
            for (int i = 0; i < min(used, S::kStages); ++i) {
                if (--s < 0) {
                    s = S::kStages - 1;
                    parity ^= 1;
                }
                Wait(&full[s], parity ^ 1, a.err);
            }
        if (kMode == kPair && !ok) {  // the other CTA's barrier says no more: leave them 10 ms
            const uint64_t t0 = tc::GlobalTimerNs();
            while (tc::GlobalTimerNs() - t0 < 10000000ull) {
            }
        }
    } else if (warp == 1 && (kMode != kPair || rank == 0)) {
        const bool one = tc::ElectOne();
        const uint64_t dw0 = tc::SmemDescSw128(tc::SmemAddr(base)), dx0 = tc::SmemDescSw128(tc::SmemAddr(base) + kWBytes);
        int s = 0, done = 0;
        uint32_t parity = 0;
        bool ok = true;
        for (int id = first_tile; id < tiles && ok; id += tile_step, ++done) {
            const Tile t = FindTile<kRows, S::kTileChannels>(a, sg, id);
            const uint32_t idesc = tc::InstrDescI8(S::kTileChannels, columns(t));
            const int b = kMode == kSplit ? 0 : done & 1, use = done >> 1;
            if (use > 0 && !(ok = __all_sync(0xffffffffu, Wait(&taken[b], (use - 1) & 1, a.err)))) break;
            tc::FenceAfterSync();
            const uint32_t acc = tmem + b * S::kColumns;
            uint32_t more = 0;
            for (int kb = k_first; kb < k_last; ++kb) {
                if (!(ok = __all_sync(0xffffffffu, Wait(&full[s], parity, a.err)))) break;
                tc::FenceAfterSync();
                // Addresses in a descriptor count 16-byte units: a step of 32 bytes of kdim is 2.
                const uint64_t dw = dw0 + s * (S::kStageBytes >> 4), dx = dx0 + s * (S::kStageBytes >> 4);
                if (one) {
#pragma unroll
                    for (int k = 0; k < kTileK / 32; ++k) {
                        if constexpr (kMode == kPair) tc::UmmaI8Pair(acc, dw + 2 * k, dx + 2 * k, idesc, k ? 1u : more);
                        else tc::UmmaI8(acc, dw + 2 * k, dx + 2 * k, idesc, k ? 1u : more);
                    }
                    if constexpr (kMode == kPair) tc::UmmaCommitPair(&empty[s]);
                    else tc::UmmaCommit(&empty[s]);
                }
                __syncwarp();
                more = 1;
                if (++s == S::kStages) {
                    s = 0;
                    parity ^= 1;
                }
            }
            if (ok && one) {
                if constexpr (kMode == kPair) tc::UmmaCommitPair(&made[b]);
                else tc::UmmaCommit(&made[b]);
            }
            __syncwarp();
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3;  // the TMEM lanes this warp may read
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        // Of every kChunk * kShare rows, this warp takes kChunk.
        constexpr int kChunk = S::kChunk, kStep = kChunk * kShare;
        const int share = (warp - 2) >> 2;
        float* scales = row_scales + (warp - 2) * S::kOwnRows;
        int* parts = reinterpret_cast<int*>(base);  // kSplit: [kRows][kChannels] over the stages, once they are read
        T* out = static_cast<T*>(a.out);
        int done = 0, slot = 0;
        bool ok = true;
        const bool one = tc::ElectOne();
        const uint64_t policy = tc::CachePolicy(a.evict_first);
        // What a tile needs beside its sums.  The next tile's is on its way while this one is written:
        // with few steps of kdim a tile would otherwise wait for it every time.
        constexpr int kOwn = (S::kOwnRows + 31) / 32;
        struct Side {
            Tile t;
            float ws, bias, qs[kOwn];
        };
        auto fetch = [&](int id) {
            Side x;
            x.t = FindTile<kRows, S::kTileChannels>(a, sg, id);
            const int c = x.t.channel0 + (kMode == kPair ? rank * kChannels : 0) + quarter * 32 + lane;
            const int64_t wc = static_cast<int64_t>(x.t.expert) * a.n + c;
            x.ws = c < a.n ? a.w_scale[wc] : 0.0f;
            x.bias = c < a.n && a.bias ? a.bias[wc] : 0.0f;
            const int count = min(kRows, x.t.end - x.t.row0);
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                const int r = i * 32 + lane, row = r / kChunk * kStep + share * kChunk + r % kChunk;
                x.qs[i] = r < S::kOwnRows && row < count ? a.q_scale[x.t.row0 + row] : 0.0f;
            }
            return x;
        };
        Side next{};
        if (first_tile < tiles) next = fetch(first_tile);
        for (int id = first_tile; id < tiles && ok; id += tile_step, ++done) {
            const Side now = next;
            const Tile t = now.t;
            const float ws = now.ws, bias = now.bias;
            if (kMode != kSplit && id + tile_step < tiles) next = fetch(id + tile_step);
            const int b = kMode == kSplit ? 0 : done & 1;
            const int c = t.channel0 + (kMode == kPair ? rank * kChannels : 0) + quarter * 32 + lane;
            const bool real = c < a.n;
            const int count = min(kRows, t.end - t.row0);
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                if (i * 32 + lane < S::kOwnRows) scales[i * 32 + lane] = now.qs[i];
            __syncwarp();
            T* direct = out + (static_cast<int64_t>(t.row0) + share * kChunk) * a.ldo + c;
            ok = __all_sync(0xffffffffu, Wait(&made[b], (done >> 1) & 1, a.err));
            if (ok) {
                tc::FenceAfterSync();
                const uint32_t from = tmem + lanes + b * S::kColumns;
                auto write = [&](const int (&v)[kChunk], int c0) {
                    if constexpr (kMode == kSplit) {
#pragma unroll
                        for (int j = 0; j < kChunk; ++j) parts[(c0 + j) * kChannels + quarter * 32 + lane] = v[j];
                    } else {
                        float y[kChunk];
                        const float4* own = reinterpret_cast<const float4*>(scales + c0 / kStep * kChunk);
#pragma unroll
                        for (int j = 0; j < kChunk; j += 4) {
                            const float4 sc = own[j / 4];
                            y[j] = fmaf(__int2float_rn(v[j]) * sc.x, ws, bias);
                            y[j + 1] = fmaf(__int2float_rn(v[j + 1]) * sc.y, ws, bias);
                            y[j + 2] = fmaf(__int2float_rn(v[j + 2]) * sc.z, ws, bias);
                            y[j + 3] = fmaf(__int2float_rn(v[j + 3]) * sc.w, ws, bias);
                        }
                        // A chunk of this segment at once by TMA, which also leaves out rows past the output's
                        // end; rows that belong to the next segment are left out here.
                        if (c - lane < a.tma_n && (c0 + kChunk <= count || !a.offsets)) {
                            T* lay = reinterpret_cast<T*>(outs + (2 * (warp - 2) + slot) * S::kOutBytes);
                            if (one) tc::BulkWaitRead<1>();
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < kChunk; ++j) lay[j * 32 + lane] = Out<T>(y[j]);
                            tc::FenceAsyncShared();
                            __syncwarp();
                            // Every chunk that takes a slot makes a group: the wait above counts groups.
                            if (one) {
                                tc::TmaStore2d(&to, lay, c - lane, t.row0 + c0, policy);
                                tc::BulkCommit();
                            }
                            slot ^= 1;
                        } else {
                            const int left = real ? count - c0 : 0;
                            T* row = direct;
                            if (left >= kChunk) {
#pragma unroll
                                for (int j = 0; j < kChunk; ++j, row += a.ldo) *row = Out<T>(y[j]);
                            } else {
#pragma unroll
                                for (int j = 0; j < kChunk; ++j, row += a.ldo)
                                    if (j < left) *row = Out<T>(y[j]);
                            }
                        }
                        direct += kStep * a.ldo;
                    }
                };
                // The next columns are on their way while these are written.
                int va[kChunk], vb[kChunk];
                int c0 = share * kChunk;
                if (c0 < count) tc::TmemLoad(from + c0, va);
#pragma unroll 1
                for (; c0 < count; c0 += 2 * kStep) {
                    tc::TmemLoadWait(va);
                    if (c0 + kStep < count) tc::TmemLoad(from + c0 + kStep, vb);
                    write(va, c0);
                    if (c0 + kStep >= count) break;
                    tc::TmemLoadWait(vb);
                    if (c0 + 2 * kStep < count) tc::TmemLoad(from + c0 + 2 * kStep, va);
                    write(vb, c0 + kStep);
                }
                tc::FenceBeforeSync();
            }
            __syncwarp();
            if constexpr (kMode == kSplit) break;  // one tile each; its rows are finished below
            if (ok && lane == 0) {
                if (kMode == kPair && rank != 0) tc::MbarArriveCluster(tc::ClusterAddr(&taken[b], 0));
                else tc::MbarArrive(&taken[b]);
            }
        }
        if (kMode != kSplit && one) tc::BulkWaitAll();  // before the memory that they read goes
    }
    if constexpr (kMode == kSplit) {
        // Row j of the tile is finished by CTA j % cluster: the parts in order of kdim.  A quarter's
        // warps take these rows in turn.
        tc::FenceBeforeSync();
        __syncwarp();
        tc::ClusterSync();
        if (warp >= 2 && first_tile < tiles) {
            const Tile t = FindTile<kRows, S::kTileChannels>(a, sg, first_tile);
            const int at = (warp & 3) * 32 + lane, c = t.channel0 + at;
            const int64_t wc = static_cast<int64_t>(t.expert) * a.n + c;
            const int count = min(kRows, t.end - t.row0);
            if (c < a.n) {
                const float ws = a.w_scale[wc], bias = a.bias ? a.bias[wc] : 0.0f;
                for (int j = rank + cluster * ((warp - 2) >> 2); j < count; j += kShare * cluster) {
                    const float scale = a.q_scale[t.row0 + j];
                    int sum = 0;
#pragma unroll 8
                    for (int r = 0; r < cluster; ++r) sum += tc::LoadCluster(tc::ClusterAddr(base, r) + (j * kChannels + at) * 4);
                    static_cast<T*>(a.out)[(static_cast<int64_t>(t.row0) + j) * a.ldo + c] =
                        Out<T>(fmaf(__int2float_rn(sum) * scale, ws, bias));
                }
            }
        }
    }
    if (a.offsets && warp >= 2) {  // rows without an expert (after the last segment: dropped choices) hold zeros
        T* out = static_cast<T*>(a.out);
        auto zeros = [&](int64_t from, int64_t to) {
            const int64_t left = (to - from) * a.n;
            for (int64_t i = static_cast<int64_t>(blockIdx.x) * (32 * kWriters) + threadIdx.x - 64; i < left; i += gridDim.x * (32 * kWriters))
                out[(from + i / a.n) * a.ldo + i % a.n] = Out<T>(0.0f);
        };
        zeros(0, sg.begin[0]);
        zeros(sg.end[a.experts - 1], a.rows);
    }
    tc::FenceBeforeSync();
    __syncwarp();
    if constexpr (kMode == kOne) __syncthreads();
    else tc::ClusterSync();  // no CTA leaves while another reads its memory or arrives on its barriers
    if (warp == 1) {
        if constexpr (kMode == kPair) tc::TmemDeallocPair(tmem, S::kTmem);
        else tc::TmemDealloc(tmem, S::kTmem);
    }
}

// Without a term to sum (kdim 0): the bias, and zeros in rows without an expert.
constexpr int kBiasBlock = 256;
template <typename T>
__global__ void __launch_bounds__(kBiasBlock) BiasRowsKernel(const MatmulArgs a) {
    extern __shared__ int segments[];
    Segments sg;
    sg.first = segments;
    sg.begin = sg.first + (a.experts + 1);
    sg.end = sg.begin + a.experts;
    LetLaterStart();
    WaitForEarlier();
    if (a.offsets) FindSegments<1, kBiasBlock>(a, sg, 0);
    __syncthreads();
    const int64_t total = static_cast<int64_t>(a.rows) * a.n;
    const int head = a.offsets ? sg.begin[0] : 0, kept = a.offsets ? sg.end[a.experts - 1] : a.rows;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBiasBlock + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * kBiasBlock) {
        const int r = static_cast<int>(i / a.n), c = static_cast<int>(i % a.n);
        float y = 0.0f;
        if (a.bias && r >= head && r < kept) {
            int e = 0;
            if (a.offsets) {
                int hi = a.experts - 1;  // the first expert whose segment ends after r
                while (e < hi) {
                    const int mid = (e + hi) >> 1;
                    if (sg.end[mid] > r) hi = mid;
                    else e = mid + 1;
                }
            }
            y = a.bias[static_cast<int64_t>(e) * a.n + c];
        }
        static_cast<T*>(a.out)[r * a.ldo + c] = Out<T>(y);
    }
}

PFN_cuTensorMapEncodeTiled_v12000 EncodeFn() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// Row-major rows x cols elements, row_bytes apart, in boxes of box_rows x box_cols; zeros out of bounds.
// The 8-bit operands come with the 128-byte swizzle, the output without one.
bool MakeMap(CUtensorMap* map, CUtensorMapDataType type, const void* p, int64_t rows, int cols, int64_t row_bytes, int box_rows,
             int box_cols) {
    const auto fn = EncodeFn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estride[2] = {1, 1};
    return fn(map, type, 2, const_cast<void*>(p), dims, strides, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
              type == CU_TENSOR_MAP_DATA_TYPE_UINT8 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Operands {
    const int8_t* q;
    int64_t ldq;
    const int8_t* w;
    int64_t ldw;
    int sms, device;
    cudaStream_t stream;
};

// The most row tiles that `rows` rows in `experts` segments can make.
int64_t MostRowTiles(const MatmulArgs& a, int height) {
    const int64_t full = (static_cast<int64_t>(a.rows) + height - 1) / height;
    return a.offsets ? std::min<int64_t>(a.rows, full + a.experts) : full;
}

// And how many are likely: every expert that can have a row ends in a part of a tile.
int64_t LikelyRowTiles(const MatmulArgs& a, int height) {
    if (!a.offsets) return MostRowTiles(a, height);
    const int64_t used = std::min(a.rows, a.experts);
    return std::max<int64_t>(used, a.rows / height + used / 2);
}

template <int kRows, Mode kMode, typename T>
cudaError_t LaunchTiles(const Operands& o, const MatmulArgs& a, int cluster) {
    using S = Shape<kRows, kMode, T>;
    CUtensorMap tw, tx, tx_part{}, to{};
    if (!MakeMap(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, o.w, static_cast<int64_t>(a.experts) * a.n, a.kdim, o.ldw, kChannels, kTileK) ||
        !MakeMap(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, o.q, a.rows, a.kdim, o.ldq, S::kXRows, kTileK))
        return cudaErrorInvalidValue;
    if (S::kXRows > kBoxRows && !MakeMap(&tx_part, CU_TENSOR_MAP_DATA_TYPE_UINT8, o.q, a.rows, a.kdim, o.ldq, kBoxRows, kTileK))
        return cudaErrorInvalidValue;
    constexpr auto kOutType = sizeof(T) == 4                       ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                              : std::is_same_v<T, __nv_bfloat16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (kMode != kSplit && a.tma_n > 0 &&
        !MakeMap(&to, kOutType, a.out, a.rows, a.n, a.ldo * static_cast<int64_t>(sizeof(T)), S::kChunk, 32))
        return cudaErrorInvalidValue;
    const size_t smem = 1024 + static_cast<size_t>(S::kStages) * S::kStageBytes + S::kAllOut + (2 * S::kStages + 4) * 8 + 16 +
                        4 * kWriters * S::kOwnRows + (a.offsets ? (3 * static_cast<size_t>(a.experts) + 1) * 4 : 0);
    const auto kernel = MatmulI8Kernel<kRows, kMode, T>;
    // Once for each device, as the call takes longer than the rest of the host's work.
    static thread_local uint64_t set_on = 0;
    const uint64_t bit = o.device < 64 ? uint64_t{1} << o.device : 0;
    if (!(set_on & bit)) {
        if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024); e != cudaSuccess) return e;
        set_on |= bit;
    }
    const int64_t tiles = MostRowTiles(a, kRows) * ((a.n + S::kTileChannels - 1) / S::kTileChannels);
    const int64_t clusters = kMode == kSplit ? tiles : std::min<int64_t>(o.sms / cluster, tiles);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    config.stream = o.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    config.attrs = attr;
    config.numAttrs = kMode == kOne ? 1 : 2;
    return cudaLaunchKernelEx(&config, kernel, tw, tx, tx_part, to, a, cluster);
}

template <typename T>
cudaError_t LaunchAs(const Operands& o, const MatmulArgs& a, Mode mode, int height, int parts) {
    if (mode == kPair) return LaunchTiles<256, kPair, T>(o, a, 2);
    if (mode == kOne) {
        if (height == 16) return LaunchTiles<16, kOne, T>(o, a, 1);
        if (height == 32) return LaunchTiles<32, kOne, T>(o, a, 1);
        if (height == 64) return LaunchTiles<64, kOne, T>(o, a, 1);
        return LaunchTiles<128, kOne, T>(o, a, 1);
    }
    if (height == 16) return LaunchTiles<16, kSplit, T>(o, a, parts);
    if (height == 32) return LaunchTiles<32, kSplit, T>(o, a, parts);
    return LaunchTiles<64, kSplit, T>(o, a, parts);
}

// Which tile, and whether CTAs share one: the least of the times that a call is expected to take, in
// microseconds, fitted to what was measured on B200.  A wave of tiles h rows high takes
// 0.22 us + 0.4 ns h for every 128 terms (issuing the loads and MMAs bounds it, hence so little of the
// height) and 0.5 us + 8.6 ns h beside them; a wave of pairs 0.235 and 3.6 us.  A kernel without work takes
// 2.4 us, one of pairs 5; adding up the parts of a tile 3 us, 50 ns a row and 10 ns a row of its height.
// Measured at both sides of the borders (rows x n x kdim, 16-bit results, calls in a row): 16 x 4,096 x 4,096, four parts
// 6.9 us, one 9.1; 128 x 4,096 x 4,096, one 32 high 9.7, two parts 12.0; 777 x 1,000 x 960, one 64 high 5.1, 128 high 5.7;
// 512 x 4,096 x 4,096, one 128 high 11.5, pairs 14.8; 1,024 x 4,096 x 4,096, pairs 15.5, one 128 high 19.5;
// 4,096 x 1,024 x 1,024, 8.3 and 8.5; 8,000 x 8,000 x 1,000, pairs 68, one 128 high 104; 4,096 x 65,536 x 128 to 32 bits,
// one 128 high 162, pairs 204.  The fit is older than the present epilogue: of 26 sizes it takes the fastest form or one
// within 5 % in 25, and loses 10 % at 4,000 rows over 64 experts, 1,000 x 512 (13.7; one 128 high 12.4).
template <typename T>
cudaError_t Launch(const Operands& o, const MatmulArgs& a) {
    if (a.kdim == 0) {
        return stlq_b200::LaunchAfter(BiasRowsKernel<T>, o.sms * 4, kBiasBlock, a.offsets ? (3 * static_cast<size_t>(a.experts) + 1) * 4 : 0, o.stream, a);
    }
    const int64_t ct = (a.n + kChannels - 1) / kChannels;
    const int nk = (a.kdim + kTileK - 1) / kTileK;
    Mode mode = kOne;
    int best_height = 128, best_parts = 1;
    double best = 1e300;
    const auto take = [&](double us, Mode m, int height, int parts) {
        if (us < best) {
            best = us;
            mode = m;
            best_height = height;
            best_parts = parts;
        }
    };
    const auto waves = [](int64_t tiles, int64_t at_once) { return static_cast<double>((tiles + at_once - 1) / at_once); };
    for (int height = 128; height >= 16; height /= 2) {
        const double step = 0.22 + 0.0004 * height, write = 0.5 + 0.0086 * height;
        take(2.4 + waves(LikelyRowTiles(a, height) * ct, o.sms) * (step * nk + write), kOne, height, 1);
        if (height > 64) continue;
        const int64_t most = MostRowTiles(a, height) * ct;
        for (int parts = 2; parts <= 8 && nk >= 2 * parts; parts *= 2) {
            // Clusters of eight find room on fewer SMs: 16 of them did not run at once, 12 did.
            if (most * parts > (parts == 8 ? o.sms * 2 / 3 : o.sms * 7 / 8)) break;
            take(2.4 + step * ((nk + parts - 1) / parts) + 3.0 + 0.05 * std::min(a.rows, height) + 0.01 * height, kSplit, height, parts);
        }
    }
    take(5.0 + waves(LikelyRowTiles(a, 256) * ((a.n + 255) / 256), o.sms / 2) * (0.235 * nk + 3.6), kPair, 256, 2);
    return LaunchAs<T>(o, a, mode, best_height, best_parts);
}


int Matmul(stlq_b200_kernels* k, const int8_t* q, int64_t ldq, const float* q_scale, const int8_t* w, int64_t ldw,
           const float* w_scale, const float* bias, const int32_t* offsets, int experts, int64_t rows, int n, int kdim,
           void* out, int out_dtype, int64_t ldo, void* stream) {
    if (!k) return Bad("kernel-provider handle is null");
    if (out_dtype != STLQ_B200_F32 && out_dtype != STLQ_B200_BF16 && out_dtype != STLQ_B200_F16)
        return Bad("out_dtype must be F32, BF16 or F16");
    if (rows < 0 || n < 0 || kdim < 0) return Bad("rows, n and kdim must be >= 0");
    if (kdim > STLQ_B200_MAX_I8_K) return Bad("kdim above 131071: a 32-bit sum could overflow");
    if (ldq < kdim || ldw < kdim || ldo < n) return Bad("ldq, ldw or ldo below the row's length");
    if (rows == 0 || n == 0) return 0;
    if (!out || !q_scale || !w_scale || (kdim > 0 && (!q || !w))) return Bad("null pointer");
    if (rows > 0x7fffff00 || static_cast<int64_t>(experts) * n > 0x7fffff00) return Bad("rows and experts * n must be below 2^31 - 256");
    if (((rows + 15) / 16 + experts) * ((static_cast<int64_t>(n) + kChannels - 1) / kChannels) > 0x7fffff00)
        return Bad("rows * n too large for one call");
    if (ldq >= (int64_t{1} << 40) || ldw >= (int64_t{1} << 40)) return Bad("ldq and ldw must be below 2^40");
    if (kdim > 0 && (!Aligned(q, 16) || !Aligned(w, 16) || ldq % 16 || ldw % 16))
        return Bad("q and w must be 16-byte aligned with ldq and ldw multiples of 16");
    if (!Aligned(q_scale, 4) || !Aligned(w_scale, 4) || !Aligned(bias, 4) || !Aligned(offsets, 4) ||
        !Aligned(out, out_dtype == STLQ_B200_F32 ? 4 : 2))
        return Bad("a scale, bias, offsets or out pointer is not aligned to its element");
    DeviceScope scope(k->device);
    if (!scope.ok()) return SetError(STLQ_B200_ECUDA, "cudaSetDevice failed");
    const int64_t out_bytes = out_dtype == STLQ_B200_F32 ? 4 : 2;
    // TMA's rows begin on 16-byte boundaries, less than 2^40 bytes apart.  It leaves out what is past a row's end in steps of 16
    // bytes: an output whose rows end inside such a step, as one that is part of a wider matrix may, has the channels of
    // its last, partial chunk written by the threads.
    const bool tma = Aligned(out, 16) && ldo * out_bytes % 16 == 0 && ldo < (int64_t{1} << 37);
    const int tma_n = !tma ? 0 : n * out_bytes % 16 == 0 ? n : n / 32 * 32;
    // A large output is written in rows as long as possible, and leaves the cache in that order: tiles run along
    // the channels and its lines are marked to go first (4,096 x 65,536 x 128 to 32 bits: 220 us without the two,
    // 205 with the mark, 166 with both, 6.5 TB/s).  A matrix that does not stay in the cache from one row of
    // tiles to the next is read for eight at a time instead.
    const int evict_first = static_cast<int64_t>(rows) * n * out_bytes > (int64_t{48} << 20);
    const int band = static_cast<int64_t>(n) * kdim <= (int64_t{32} << 20) ? 1 : 8;
    const MatmulArgs a{q_scale, w_scale, bias, offsets, experts, static_cast<int>(rows), n, kdim, tma_n, evict_first, band, out, ldo,
                       static_cast<unsigned int*>(k->err.p)};
    const Operands o{q, ldq, w, ldw, k->num_sms, k->device, static_cast<cudaStream_t>(stream)};
    if (out_dtype == STLQ_B200_F32) return Ck(Launch<float>(o, a), "matmul_i8");
    if (out_dtype == STLQ_B200_BF16) return Ck(Launch<__nv_bfloat16>(o, a), "matmul_i8");
    return Ck(Launch<__half>(o, a), "matmul_i8");
}

}  // namespace

extern "C" {

int stlq_b200_matmul_i8(stlq_b200_kernels* k, const int8_t* q, int64_t ldq, const float* q_scale, const int8_t* w,
                        int64_t ldw, const float* w_scale, const float* bias, int64_t rows, int n, int kdim, void* out,
                        int out_dtype, int64_t ldo, void* stream) {
    return Guard([&] { return Matmul(k, q, ldq, q_scale, w, ldw, w_scale, bias, nullptr, 1, rows, n, kdim, out, out_dtype, ldo, stream); });
}

int stlq_b200_matmul_i8_grouped(stlq_b200_kernels* k, const int8_t* q, int64_t ldq, const float* q_scale, const int8_t* w,
                                int64_t ldw, const float* w_scale, const float* bias, const int32_t* offsets, int experts,
                                int64_t rows, int n, int kdim, void* out, int out_dtype, int64_t ldo, void* stream) {
    return Guard([&] {
        if (experts < 1 || experts > STLQ_B200_MAX_EXPERTS) return Bad("1 <= experts <= 1024 required");
        if (!offsets) return Bad("null offsets");
        return Matmul(k, q, ldq, q_scale, w, ldw, w_scale, bias, offsets, experts, rows, n, kdim, out, out_dtype, ldo, stream);
    });
}

}  // extern "C"
