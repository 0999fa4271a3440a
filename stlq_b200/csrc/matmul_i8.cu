// Products in 8-bit integers with a scale for each row and each channel, for one matrix or for the
// matrix of each expert over its segment of sorted rows:
//
//   out[r, c] = float(sum_i q[r, i] w[c, i]) * q_scale[r] * w_scale[c] + bias[c]
//
// The sum is exact: 32-bit integers hold it for up to 131,071 terms.  The tensor cores (tcgen05
// kind::i8) take 128 channels as the rows of a tile and kRows of the product's rows as its columns,
// so that one row costs a tile 16 wide, and a warp of the epilogue, whose 32 lanes hold 32
// neighbouring channels, writes 32 neighbouring elements of a row.
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

using stlq_b200::Ck;
using stlq_b200::DeviceScope;
using stlq_b200::SetError;
namespace tc = stlq_b200::tc;

constexpr int kChannels = 128;                       // channels of a tile (the MMA's M)
constexpr int kTileK = 128;                          // bytes of a 128-byte swizzle row
constexpr uint32_t kWBytes = kChannels * kTileK;
constexpr int kThreads = 192;                        // warp 0 loads, warp 1 multiplies, 2..5 write
constexpr uint64_t kWaitNs = 2000000000ull;          // 2 s per barrier wait
constexpr int kBand = 8;                             // row tiles that run side by side over the channels

template <int kRows>
struct Shape {
    static constexpr uint32_t kXBytes = kRows * kTileK;
    static constexpr uint32_t kStageBytes = kWBytes + kXBytes;
    static constexpr int kStages = std::min<int>(10, 200 * 1024 / kStageBytes);
    static constexpr int kColumns = kRows < 32 ? 32 : kRows;  // TMEM columns of one accumulator
    static constexpr uint32_t kTmem = 2 * kColumns;           // two: one is written out while the next is made
};

struct MatmulArgs {
    const float* q_scale;
    const float* w_scale;
    const float* bias;
    const int* offsets;  // null: one matrix, all rows
    int experts, rows, n, kdim;
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
// begin[e] / end[e] its rows, within the
// product's.
struct Segments {
    int* first;
    int* begin;
    int* end;
};

template <int kRows>
__device__ __forceinline__ Tile FindTile(const MatmulArgs& a, const Segments& sg, int id) {
    Tile t;
    const int ct = (a.n + kChannels - 1) / kChannels;
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
    // Bands of kBand row tiles, the band's row tiles running fastest: the tiles in flight share few
    // rows and few channels, which stay in L2.
    const int rt = (t.end - t.row0 + kRows - 1) / kRows;
    const int band = local / (kBand * ct), in = local - band * kBand * ct;
    const int height = min(kBand, rt - band * kBand);
    t.channel0 = in / height * kChannels;
    t.row0 += (band * kBand + in % height) * kRows;
    return t;
}

template <int kRows, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    MatmulI8Kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx, const MatmulArgs a) {
    using S = Shape<kRows>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = smem_raw + ((1024 - (tc::SmemAddr(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(base + S::kStages * S::kStageBytes);
    uint64_t* empty = full + S::kStages;
    uint64_t* made = empty + S::kStages;  // an accumulator is complete
    uint64_t* taken = made + 2;           // an accumulator has been read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(taken + 2);
    Segments sg;
    sg.first = reinterpret_cast<int*>(tmem_slot + 4);
    sg.begin = sg.first + (a.experts + 1);
    sg.end = sg.begin + a.experts;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ct = (a.n + kChannels - 1) / kChannels;
    const int nk = (a.kdim + kTileK - 1) / kTileK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            tc::MbarInit(&full[s], 1);
            tc::MbarInit(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::MbarInit(&made[b], 1);
            tc::MbarInit(&taken[b], 4);
        }
        tc::FenceBarrierInit();
    }
    if (warp == 1) tc::TmemAlloc(tmem_slot, S::kTmem);
    if (a.offsets) {
        for (int e = threadIdx.x; e < a.experts; e += kThreads) sg.end[e] = min(max(a.offsets[e + 1], 0), a.rows);
        __syncthreads();
        if (warp == 0) {
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
    }
    tc::FenceBeforeSync();
    __syncthreads();
    tc::FenceAfterSync();
    const uint32_t tmem = *tmem_slot;
    const int tiles = a.offsets ? sg.first[a.experts] : (a.rows + kRows - 1) / kRows * ct;

    if (warp == 0 && lane == 0) {
        int64_t step = 0;
        bool ok = true;
        for (int id = blockIdx.x; id < tiles && ok; id += gridDim.x) {
            const Tile t = FindTile<kRows>(a, sg, id);
            const int wrow = t.expert * a.n + t.channel0;
            for (int kb = 0; kb < nk; ++kb, ++step) {
                const int s = static_cast<int>(step % S::kStages);
                const int64_t round = step / S::kStages;
                if (round > 0 && !(ok = tc::MbarWait(&empty[s], (round - 1) & 1, a.err, kWaitNs))) break;
                unsigned char* st = base + s * S::kStageBytes;
                tc::MbarArriveExpectTx(&full[s], S::kStageBytes);
                tc::TmaLoad2d(st, &tw, &full[s], kb * kTileK, wrow);
                tc::TmaLoad2d(st + kWBytes, &tx, &full[s], kb * kTileK, t.row0);
            }
        }
        // Copies still in flight land before the block may exit.
        for (int64_t i = step - 1; i >= 0 && i >= step - S::kStages; --i)
            tc::MbarWait(&full[i % S::kStages], (i / S::kStages) & 1, a.err, kWaitNs, false);
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = tc::InstrDescI8(kChannels, kRows);
        int64_t step = 0;
        int done = 0;
        bool ok = true;
        for (int id = blockIdx.x; id < tiles && ok; id += gridDim.x, ++done) {
            const int b = done & 1, use = done >> 1;
            if (use > 0 && !(ok = tc::MbarWait(&taken[b], (use - 1) & 1, a.err, kWaitNs))) break;
            tc::FenceAfterSync();
            for (int kb = 0; kb < nk; ++kb, ++step) {
                const int s = static_cast<int>(step % S::kStages);
                if (!(ok = tc::MbarWait(&full[s], (step / S::kStages) & 1, a.err, kWaitNs))) break;
                tc::FenceAfterSync();
                const uint32_t w = tc::SmemAddr(base + s * S::kStageBytes), x = w + kWBytes;
#pragma unroll
                for (int k = 0; k < kTileK / 32; ++k)
                    tc::UmmaI8(tmem + b * S::kColumns, tc::SmemDescSw128(w + k * 32), tc::SmemDescSw128(x + k * 32), idesc,
                               (kb > 0 || k > 0) ? 1u : 0u);
                tc::UmmaCommit(&empty[s]);
            }
            if (ok) tc::UmmaCommit(&made[b]);
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3;  // the TMEM lanes this warp may read
        T* out = static_cast<T*>(a.out);
        int done = 0;
        bool ok = true;
        for (int id = blockIdx.x; id < tiles && ok; id += gridDim.x, ++done) {
            const Tile t = FindTile<kRows>(a, sg, id);
            const int b = done & 1;
            const int c = t.channel0 + quarter * 32 + lane;
            const bool real = c < a.n;
            const int64_t wc = static_cast<int64_t>(t.expert) * a.n + c;
            const float ws = real ? a.w_scale[wc] : 0.0f;
            const float bias = real && a.bias ? a.bias[wc] : 0.0f;
            ok = __all_sync(0xffffffffu, tc::MbarWait(&made[b], (done >> 1) & 1, a.err, kWaitNs));
            if (!ok) break;
            tc::FenceAfterSync();
#pragma unroll 1
            for (int c0 = 0; c0 < kRows; c0 += 16) {
                const int r0 = t.row0 + c0;
                if (r0 >= t.end) break;
                int v[16];
                tc::TmemLoad16(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + b * S::kColumns + c0, v);
                const float qs = r0 + (lane & 15) < t.end ? a.q_scale[r0 + (lane & 15)] : 0.0f;
                tc::TmemLoadWait();
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float s = __shfl_sync(0xffffffffu, qs, j);
                    const float y = fmaf(__int2float_rn(v[j]) * s, ws, bias);
                    if (real && r0 + j < t.end) out[(static_cast<int64_t>(r0) + j) * a.ldo + c] = Out<T>(y);
                }
            }
            tc::FenceBeforeSync();
            __syncwarp();
            if (lane == 0) tc::MbarArrive(&taken[b]);
        }
        // Rows after the last segment (dropped choices) hold zeros.
        if (a.offsets) {
            const int64_t kept = sg.end[a.experts - 1];
            const int64_t left = (a.rows - kept) * a.n;
            for (int64_t i = blockIdx.x * 128 + threadIdx.x - 64; i < left; i += gridDim.x * 128)
                out[(kept + i / a.n) * a.ldo + i % a.n] = Out<T>(0.0f);
        }
    }
    tc::FenceBeforeSync();
    __syncthreads();
    if (warp == 1) tc::TmemDealloc(tmem, S::kTmem);
}

// Without a term to sum (kdim 0): the bias, and zeros after the last segment.
template <typename T>
__global__ void BiasRowsKernel(const MatmulArgs a) {
    const int64_t total = static_cast<int64_t>(a.rows) * a.n;
    const int kept = a.offsets ? min(max(a.offsets[a.experts], 0), a.rows) : a.rows;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int r = static_cast<int>(i / a.n), c = static_cast<int>(i % a.n);
        float y = 0.0f;
        if (a.bias && r < kept) {
            int e = 0;
            if (a.offsets) {
                int lo = 0, hi = a.experts;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (a.offsets[mid] <= r) lo = mid;
                    else hi = mid;
                }
                e = lo;
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

// Row-major rows x kdim bytes, boxes of box_rows x 128 bytes, 128-byte swizzle, zeros out of bounds.
bool MakeMap(CUtensorMap* map, const int8_t* p, int64_t rows, int kdim, int64_t ld, int box_rows) {
    const auto fn = EncodeFn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(kdim), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2] = {kTileK, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estride[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dims, strides, box, estride,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kRows, typename T>
cudaError_t LaunchRows(const CUtensorMap& tw, const int8_t* q, int64_t ldq, const MatmulArgs& a, int sms, cudaStream_t s) {
    using S = Shape<kRows>;
    CUtensorMap tx;
    if (!MakeMap(&tx, q, a.rows, a.kdim, ldq, kRows)) return cudaErrorInvalidValue;
    const size_t smem = 1024 + static_cast<size_t>(S::kStages) * S::kStageBytes + (2 * S::kStages + 4) * 8 + 16 +
                        (a.offsets ? (3 * static_cast<size_t>(a.experts) + 1) * 4 : 0);
    const auto kernel = MatmulI8Kernel<kRows, T>;
    if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024); e != cudaSuccess) return e;
    const int64_t ct = (a.n + kChannels - 1) / kChannels;
    const int64_t most = (static_cast<int64_t>(a.rows) + kRows - 1) / kRows + (a.offsets ? a.experts : 0);
    const int grid = static_cast<int>(std::min<int64_t>(sms, ct * most));
    kernel<<<grid, kThreads, smem, s>>>(tw, tx, a);
    return cudaGetLastError();
}

// The tile's width in rows: the least that holds a segment (their mean, for experts), so that few
// rows cost few columns; wider tiles read a weight fewer times.
template <typename T>
cudaError_t Launch(const int8_t* q, int64_t ldq, const int8_t* w, int64_t ldw, const MatmulArgs& a, int sms, cudaStream_t s) {
    if (a.kdim == 0) {
        BiasRowsKernel<T><<<sms * 4, 256, 0, s>>>(a);
        return cudaGetLastError();
    }
    CUtensorMap tw;
    if (!MakeMap(&tw, w, static_cast<int64_t>(a.experts) * a.n, a.kdim, ldw, kChannels)) return cudaErrorInvalidValue;
    const int64_t mean = (a.rows + a.experts - 1) / a.experts;
    if (mean <= 16) return LaunchRows<16, T>(tw, q, ldq, a, sms, s);
    if (mean <= 32) return LaunchRows<32, T>(tw, q, ldq, a, sms, s);
    if (mean <= 64) return LaunchRows<64, T>(tw, q, ldq, a, sms, s);
    if (mean <= 128) return LaunchRows<128, T>(tw, q, ldq, a, sms, s);
    return LaunchRows<256, T>(tw, q, ldq, a, sms, s);
}

int Bad(const char* msg) { return SetError(STLQ_B200_EINVAL, msg); }
bool Aligned(const void* p, int64_t to) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(to) == 0; }

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
    if (kdim > 0 && (!Aligned(q, 16) || !Aligned(w, 16) || ldq % 16 || ldw % 16))
        return Bad("q and w must be 16-byte aligned with ldq and ldw multiples of 16");
    if (!Aligned(q_scale, 4) || !Aligned(w_scale, 4) || !Aligned(bias, 4) || !Aligned(offsets, 4) ||
        !Aligned(out, out_dtype == STLQ_B200_F32 ? 4 : 2))
        return Bad("a scale, bias, offsets or out pointer is not aligned to its element");
    DeviceScope scope(k->device);
    if (!scope.ok()) return SetError(STLQ_B200_ECUDA, "cudaSetDevice failed");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const MatmulArgs a{q_scale, w_scale, bias, offsets, experts, static_cast<int>(rows), n, kdim, out, ldo,
                       static_cast<unsigned int*>(k->err.p)};
    if (out_dtype == STLQ_B200_F32) return Ck(Launch<float>(q, ldq, w, ldw, a, k->num_sms, s), "matmul_i8");
    if (out_dtype == STLQ_B200_BF16) return Ck(Launch<__nv_bfloat16>(q, ldq, w, ldw, a, k->num_sms, s), "matmul_i8");
    return Ck(Launch<__half>(q, ldq, w, ldw, a, k->num_sms, s), "matmul_i8");
}

template <typename F>
int Guard(F&& f) {
    try {
        return f();
    } catch (...) {
        return STLQ_B200_ENOMEM;  // the only thing that throws here is a message's memory
    }
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
