// Rows quantised to 8 bits, rows sorted by the expert (or root codeword) they were assigned to and
// back, with weights applied, and the gradient of that exchange.
//
// T tokens (rows) with k choices of E experts make P = T k pairs; pair p = t k + j.  A choice outside
// [0, E) is dropped.  order is the stable sort of the pairs by expert, dropped pairs last; position
// its inverse; offsets[e] the first sorted row of expert e, offsets[E] the rows kept.  Every kernel
// compares a position with offsets[E] and with P before it uses it, so arrays that no sort made
// cannot lead outside a buffer.  Nothing here accumulates through atomics in an order that matters:
// results do not change from call to call.
#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "provider.h"

namespace {

using stlq_b200::Aligned;
using stlq_b200::Bad;
using stlq_b200::Ck;
using stlq_b200::DeviceScope;
using stlq_b200::Guard;
using stlq_b200::LaunchAfter;
using stlq_b200::LetLaterStart;
using stlq_b200::SetError;
using stlq_b200::WaitForEarlier;

constexpr int kBlock = 256;
constexpr int64_t kMostPairs = 0x7ffffc00;  // so that a block's worth past the last pair is still an int
// Likewise for columns: a thread counts up to a row's packs, at most 8 of a block's worth ahead and one past the end.
constexpr int kMostCols = STLQ_B200_MAX_COLS;
static_assert(int64_t{kMostCols} + 8 * kBlock + 2 * kBlock <= 0x7fffffff, "a column counter past a row's end would overflow");

template <typename T>
__device__ __forceinline__ float ToFloat(T v) {
    if constexpr (std::is_same_v<T, float>) return v;
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
    else return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T FromFloat(float v) {
    if constexpr (std::is_same_v<T, float>) return v;
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
    else return __float2half_rn(v);
}

// N consecutive elements moved as one access (N * sizeof(T) bytes, aligned to as many).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// Accesses whose lines leave the cache first, for what is read or written once and is larger than it: combine's
// y (16,384 x 8 x 2,048 bfloat16: 98 us without, 92 with) and its gradient's dy (199 and 191).  The gradient's y is
// read the ordinary way (184; 187 otherwise).
template <typename P>
__device__ __forceinline__ void StoreStreaming(void* to, const P& v) {
    if constexpr (sizeof(P) == 16) __stcs(static_cast<uint4*>(to), *reinterpret_cast<const uint4*>(&v));
    else *static_cast<P*>(to) = v;
}

template <bool kStreaming, typename P>
__device__ __forceinline__ void Load(P& v, const void* from) {
    if constexpr (sizeof(P) == 16 && kStreaming) {
        // Volatile, so that it stays behind WaitForEarlier.
        uint4 u;
        asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(from));
        *reinterpret_cast<uint4*>(&v) = u;
    } else if constexpr (sizeof(P) == 16) *reinterpret_cast<uint4*>(&v) = *static_cast<const uint4*>(from);
    else v = *static_cast<const P*>(from);
}

__device__ __forceinline__ float LoadAs(const void* p, int64_t i, int dtype) {
    if (dtype == STLQ_B200_F32) return static_cast<const float*>(p)[i];
    if (dtype == STLQ_B200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void StoreAs(void* p, int64_t i, int dtype, float v) {
    if (dtype == STLQ_B200_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == STLQ_B200_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// offsets[E] as the kernels use it: rows kept, within [0, P].
__device__ __forceinline__ int Kept(const int* offsets, int experts, int pairs) {
    return min(max(offsets[experts], 0), pairs);
}

// ---- quantisation of rows ----------------------------------------------------------------------

// 127 x / amax in 32 bits (two roundings), to the nearest integer, ties to even.  `down` keeps 127 x
// finite for the largest rows: both are multiplied by 2^-8, which changes no bit of the quotient.
__device__ __noinline__ int Quantise(float x, float amax, float down) {
    return __float2int_rn(__fdiv_rn(__fmul_rn(__fmul_rn(x, down), 127.0f), __fmul_rn(amax, down)));
}

// What a row's quantisation needs beside its largest |x|.
struct RowScale {
    float amax, down, r;
    bool finite;
    bool some;   // the row has numbers other than zeros, and nothing else
    bool quick;  // and products decide its values
};

// The same for N values without the division, which bound the kernel (16,384 x 4,096 bfloat16: 90 us with
// one for each value).  Adding 1.5 * 2^23 rounds to an integer and leaves it in the low bits.
//
// 16-bit rows.  Write x = m 2^a and amax = M 2^b with integers below 2^11.  The quotient is exactly n + 1/2 only if
// 254 m 2^s = (2n + 1) M for some s, and as 127 is prime, then 127 divides M or 2n + 1 = 127: but for the rows whose
// M it divides (1 in 128, divided), the one tie is 63.5, which goes to 64.  Any other quotient v is at least
// v / (254 m) > v 2^-19 from a tie.  So x r with r = (1 + 2^-20) 127 / amax, whose reciprocal and
// product are off by less than 2^-21.4, is above v by 2^-20.8 to 2^-19.5 of it and rounds as the quotient does.
//
// 32-bit rows.  x r with r = 127 / amax differs from the rounded quotient by less than 4 roundings of a number up to
// 127 (4 * 127 * 2^-24 < 3.1e-5), so it rounds to the same integer unless it is nearer than that to the middle
// between two; a pack with such a value is divided.
template <typename T, int N>
__device__ __noinline__ Pack<int8_t, N> DividePack(Pack<T, N> x, float amax, float down) {
    Pack<int8_t, N> q;
#pragma unroll
    for (int i = 0; i < N; ++i) q.v[i] = static_cast<int8_t>(Quantise(ToFloat(x.v[i]), amax, down));
    return q;
}

template <typename T, int N>
__device__ __forceinline__ Pack<int8_t, N> QuantisePack(const Pack<T, N>& x, const RowScale& s) {
    constexpr float kMagic = 12582912.0f;
    unsigned low[N];
    bool sure = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float v = ToFloat(x.v[i]);
        const float t = fmaf(v, s.r, kMagic);
        if (sizeof(T) != 2) sure = sure && fabsf(fmaf(v, s.r, kMagic - t)) < 0.5f - 4e-5f;
        low[i] = __float_as_uint(t);
    }
    if (sizeof(T) != 2 && !sure) return DividePack(x, s.amax, s.down);
    Pack<int8_t, N> q;
    if constexpr (N % 4 == 0) {
        unsigned* w = reinterpret_cast<unsigned*>(&q);
#pragma unroll
        for (int i = 0; i < N; i += 4)
            w[i / 4] = __byte_perm(__byte_perm(low[i], low[i + 1], 0x0040), __byte_perm(low[i + 2], low[i + 3], 0x0040), 0x5410);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) q.v[i] = static_cast<int8_t>(low[i]);
    }
    return q;
}

// From the bits of the largest |x| of a row.
template <typename T>
__device__ __forceinline__ RowScale ScaleOf(unsigned int top) {
    RowScale s;
    s.amax = __uint_as_float(top);
    s.finite = top < 0x7f800000u;
    s.some = s.finite && top != 0;
    s.down = s.amax > 1e36f ? 0.00390625f : 1.0f;
    // Where 127 / amax and its products are ordinary numbers.
    s.quick = s.some && s.amax >= 1e-30f && s.amax <= 1e30f;
    if constexpr (sizeof(T) == 2) {
        s.r = 127.0f * (1.0f + 9.5367431640625e-7f) * __fdividef(1.0f, s.amax);  // 1 + 2^-20
        s.quick = s.quick && ((top & 0x7fffffu) | 0x800000u) % 127u != 0;
    } else {
        s.r = __fdiv_rn(127.0f, s.amax);
    }
    return s;
}

// The larger of `top` and the |x|, by bits: unsigned order puts every NaN above infinity above the numbers.
template <typename T, int N>
__device__ __forceinline__ unsigned int LargestBits(const Pack<T, N>& x, unsigned int top) {
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
        using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
        const T2* p = reinterpret_cast<const T2*>(&x);
        T2 m = __habs2(p[0]);
#pragma unroll
        for (int i = 1; i < N / 2; ++i) m = __hmax2_nan(m, __habs2(p[i]));
        return max(top, max(__float_as_uint(fabsf(ToFloat(m.x))), __float_as_uint(fabsf(ToFloat(m.y)))));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(ToFloat(x.v[i])) & 0x7fffffffu);
        return top;
    }
}

// One group of L threads quantises one row and writes it once, or (kSpread) to the rows of its choices.  The row
// is read once: a thread keeps its first kHold packs in registers between the maximum and the rounding, and
// re-reads the rest.  What a thread does once a row (addresses, the maximum over the group, the scale) costs as
// much as quantising some five packs, and instructions bound the kernel; so a thread takes four packs, from four
// threads a row for 128 bfloat16 to 256 for 8,192.  Sixteen packs a thread cost too many registers (66 us), two leave
// too much beside them (48 us).  16,384 x 4,096 bfloat16 take 36 us, 5.6 TB/s, float32 63 us, 5.4 TB/s, 300,000 x 128 22
// and 36 us, one row of 4,096 1.6 us (with 256 threads and two packs each, as its latency counts).
template <typename T, int N, int L, int kHold, bool kSpread>
__global__ void __launch_bounds__(kBlock, sizeof(T) == 2 ? 6 : 4)
    QuantizeRowsKernel(const T* x, int64_t ldx, int64_t rows, int cols, int topk,
                       const int* position, const int* offsets, int experts, int pairs,
                       int8_t* q, int64_t ldq, float* scale) {
    constexpr int kGroups = kBlock / L;
    using In = Pack<T, N>;
    using Out = Pack<int8_t, N>;
    __shared__ unsigned int part[kBlock / 32];
    const int group = threadIdx.x / L, at = threadIdx.x % L;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
    const bool real = row < rows;
    const int full = cols / N;
    LetLaterStart();
    WaitForEarlier();
    const T* xr = x + (real ? row : 0) * ldx;
    const In* packs = reinterpret_cast<const In*>(xr) + at;
    In hold[kHold];
    unsigned int top = 0;
    if (real) {
        // The group's packs of the row, but for its last ones, without a test for each.
        if (kHold * L <= full) {
#pragma unroll
            for (int h = 0; h < kHold; ++h) hold[h] = packs[h * L];
        } else {
#pragma unroll
            for (int h = 0; h < kHold; ++h) hold[h] = at + h * L < full ? packs[h * L] : In{};
        }
#pragma unroll
        for (int h = 0; h < kHold; ++h) top = LargestBits(hold[h], top);
        for (int c = kHold * L; c + at < full; c += L) top = LargestBits(packs[c], top);
        if (full * N < cols)
            for (int c = full * N + at; c < cols; c += L) top = max(top, __float_as_uint(ToFloat(xr[c])) & 0x7fffffffu);
    }
    if constexpr (L < 32) {
        for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    } else {
        top = __reduce_max_sync(0xffffffffu, top);
    }
    if constexpr (L > 32) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < L / 32; ++w) top = max(top, part[group * (L / 32) + w]);
    }
    if (!real) return;
    const RowScale rs = ScaleOf<T>(top);
    const int kept = kSpread ? Kept(offsets, experts, pairs) : 0;
    // One row, or one for each choice: zeros (and scale 0) where it was dropped.
    auto spread = [&](auto&& write) {
        if constexpr (!kSpread) {
            write(row, true);
        } else {
            for (int j0 = 0; j0 < topk; j0 += 4) {  // four positions in flight
                int p[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = j0 + j < topk ? position[row * topk + j0 + j] : -1;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (static_cast<unsigned>(p[j]) < static_cast<unsigned>(pairs)) write(static_cast<int64_t>(p[j]), p[j] < kept);
            }
        }
    };
    // The packs in registers, where products decide them; a row that is divided reads its packs again, in the loop
    // below (a test inside for each pack, with the division beside it, cost 16,384 x 4,096 bfloat16 6 us of 44).
    int from = 0;
    if (rs.quick) {
        Out held[kHold];
#pragma unroll
        for (int h = 0; h < kHold; ++h) held[h] = QuantisePack(hold[h], rs);
        spread([&](int64_t to, bool real_row) {
            Out* qr = reinterpret_cast<Out*>(q + to * ldq) + at;
            if (real_row && kHold * L <= full) {
#pragma unroll
                for (int h = 0; h < kHold; ++h) qr[h * L] = held[h];
            } else {
#pragma unroll
                for (int h = 0; h < kHold; ++h)
                    if (at + h * L < full) qr[h * L] = real_row ? held[h] : Out{};
            }
        });
        from = kHold * L;
    }
    for (int c = from; c + at < full; c += L) {
        const Out r = rs.quick ? QuantisePack(packs[c], rs) : rs.some ? DividePack(packs[c], rs.amax, rs.down) : Out{};
        spread([&](int64_t to, bool real_row) { (reinterpret_cast<Out*>(q + to * ldq) + at)[c] = real_row ? r : Out{}; });
    }
    if (full * N < cols)
        for (int c = full * N + at; c < cols; c += L) {
            const int8_t r = rs.some ? static_cast<int8_t>(Quantise(ToFloat(xr[c]), rs.amax, rs.down)) : static_cast<int8_t>(0);
            spread([&](int64_t to, bool real_row) { q[to * ldq + c] = real_row ? r : static_cast<int8_t>(0); });
        }
    if (at == 0) {
        const float s = rs.finite ? __fdiv_rn(rs.amax, 127.0f) : __int_as_float(0x7fc00000);
        spread([&](int64_t to, bool real_row) { scale[to] = real_row ? s : 0.0f; });
    }
}

// ---- sort by expert ----------------------------------------------------------------------------

// A counting sort over `bins` digits, stable: a tile of keys per block, each of its warps ranking a
// contiguous piece 32 keys at a time (a ballot for each bit of the digit gives the lanes that share it).  Up to
// kOneBins - 1 experts it is one pass; above that two passes of half the key's bits each, from the low
// digit to the high one.  A sort of few pairs is one launch of one block; others take three a pass: count, scan
// each digit over the tiles, scatter.  12 bytes a pair are all that must move (2 us for a million): latency
// bounds it, that of a launch (3.0 us for 512 pairs) or of seven with their barriers and, in the last, a scattered
// write of each position (39 us for a million pairs over 16,384 experts; 9.4 us in three for 131,072 over 128).
constexpr int kSortBlock = 512;
constexpr int kSortWarps = kSortBlock / 32;
// Keys of a warp: more make longer runs of a digit to write, fewer use more SMs (32,768 pairs over 64 experts took
// 11 us in 8 tiles of the longer ones).
constexpr int kFewPerWarp = 64, kManyPerWarp = 256;
constexpr int64_t kFewPairs = 148 * kSortWarps * 2 * kFewPerWarp;
constexpr int kOneBins = 1025;
constexpr int kAloneBlock = 1024;
// The most pairs that one block sorts as fast as three launches (8,192 of 256 take it 14.1 us, three 10.5; 4,096 8.4), or over
// two digits as seven (2,048 of 16,384 25 us, seven 20.9; 1,024 15.0): as many keys of a lane.
constexpr int kAloneRounds = 4;
constexpr int kAlone = kAloneBlock * kAloneRounds;
constexpr int kWideRounds = 1;
constexpr int kWide = kAloneBlock * kWideRounds;

struct SortPass {
    const void* ids;   // first pass: the caller's ids
    int wide;          // ids are int64
    const int2* records;  // second pass: the keys and pairs that the first pass left
    int n, experts, shift, mask, bins, tiles;
};

__device__ __forceinline__ int KeyOf(const SortPass& a, int i) {
    if (a.records) return a.records[i].x;
    const int64_t id = a.wide ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int*>(a.ids)[i];
    return id >= 0 && id < a.experts ? static_cast<int>(id) : a.experts;
}

// One round of a warp: each lane's digit (bins: no key; below 2^kBits) counted into count[]; the lane's rank among the
// warp's keys of its digit so far.
template <int kBits>
__device__ __forceinline__ int CountRound(int d, const SortPass& a, unsigned short* count) {
    const int lane = threadIdx.x & 31;
    unsigned same = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kBits; ++i) {
        const bool set = (d >> i) & 1;
        const unsigned with = __ballot_sync(0xffffffffu, set);
        same &= set ? with : ~with;
    }
    const int before = d < a.bins ? count[d] : 0;
    const int mine = __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (mine == 0 && d < a.bins) count[d] = static_cast<unsigned short>(before + __popc(same));
    __syncwarp();
    return before + mine;
}

// The sum of x over the threads before this one in its block; `all`: over all.
__device__ __forceinline__ int ScanThreads(int x, int* part, int* all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int s = x;
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    if (lane == 31) part[warp] = s;
    __syncthreads();
    if (warp == 0) {
        int t = lane < warps ? part[lane] : 0;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += y;
        }
        part[lane] = t;
    }
    __syncthreads();
    *all = part[warps - 1];
    const int before = (warp ? part[warp - 1] : 0) + s - x;
    __syncthreads();
    return before;
}

// counts [warps][bins] to the sums over the warps before; base[b] = the keys of the digits before b.
__device__ __forceinline__ void ScanDigits(unsigned short* counts, int warps, int bins, int* base) {
    __shared__ int part[32];
    int carry = 0;
    for (int b0 = 0; b0 < bins; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        int own = 0;
        if (b < bins)
#pragma unroll 8
            for (int w = 0; w < warps; ++w) {
                const int c = counts[w * bins + b];
                counts[w * bins + b] = static_cast<unsigned short>(own);
                own += c;
            }
        int all;
        const int before = ScanThreads(own, part, &all);
        if (b < bins) base[b] = carry + before;
        carry += all;
    }
    __syncthreads();
}

// The whole sort in one block.
template <int kBits>
__global__ void __launch_bounds__(kAloneBlock)
    SortAloneKernel(SortPass a, int rounds, int* order, int* position, int* offsets) {
    extern __shared__ int base[];  // [bins], then the counts [warps][bins]
    unsigned short* counts = reinterpret_cast<unsigned short*>(base + a.bins);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    LetLaterStart();
    for (int i = threadIdx.x; i < warps * a.bins; i += blockDim.x) counts[i] = 0;
    __syncthreads();
    WaitForEarlier();
    const int first = warp * rounds * 32 + lane;
    int key[kAloneRounds];
    unsigned short rank[kAloneRounds];
#pragma unroll
    for (int r = 0; r < kAloneRounds; ++r)
        if (r < rounds) key[r] = first + r * 32 < a.n ? KeyOf(a, first + r * 32) : a.bins;
#pragma unroll
    for (int r = 0; r < kAloneRounds; ++r)
        if (r < rounds) rank[r] = static_cast<unsigned short>(CountRound<kBits>(key[r], a, counts + warp * a.bins));
    __syncthreads();
    ScanDigits(counts, warps, a.bins, base);
    for (int b = threadIdx.x; b < a.bins; b += blockDim.x) offsets[b] = base[b];
#pragma unroll
    for (int r = 0; r < kAloneRounds; ++r) {
        const int i = first + r * 32;
        if (r < rounds && i < a.n) {
            const int to = base[key[r]] + counts[warp * a.bins + key[r]] + rank[r];
            order[to] = i;
            position[i] = to;
        }
    }
}

// A warp's part of the offsets of a two-pass sort: r is the first row of every expert after `after`, the key of row
// r - 1, up to `to`, row r's.  The warp fills such a stretch together, as it may be as long as there are experts.
__device__ __forceinline__ void FillOffsets(int r, int after, int to, int* offsets) {
    const int lane = threadIdx.x & 31;
    for (unsigned left = __ballot_sync(0xffffffffu, after < to); left; left &= left - 1) {
        const int from = __ffs(left) - 1;
        const int a = __shfl_sync(0xffffffffu, after, from), b = __shfl_sync(0xffffffffu, to, from);
        for (int e = a + 1 + lane; e <= b; e += 32) offsets[e] = r - lane + from;
    }
}

// Both passes of a sort over more than kOneBins - 1 experts in one block, the records between them in shared memory
// (the seven launches of the general form take the host 20 us; this 10 to 15).
template <int kBits>
__global__ void __launch_bounds__(kAloneBlock)
    SortWideKernel(SortPass a, SortPass b, int rounds, int* order, int* position, int* offsets) {
    extern __shared__ int2 records[];  // [n], later the sorted keys; then base [bins] and the counts [warps][bins]
    const int bins = max(a.bins, b.bins);
    int* base = reinterpret_cast<int*>(records + a.n);
    unsigned short* counts = reinterpret_cast<unsigned short*>(base + bins);
    int* sorted = reinterpret_cast<int*>(records);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    LetLaterStart();
    for (int i = threadIdx.x; i < warps * a.bins; i += blockDim.x) counts[i] = 0;
    __syncthreads();
    WaitForEarlier();
    const int first = warp * rounds * 32 + lane;
    int2 rec[kWideRounds];
    unsigned short rank[kWideRounds];
    // Each lane's place in the order of one digit.
    auto pass = [&](const SortPass& p) {
#pragma unroll
        for (int r = 0; r < kWideRounds; ++r)
            if (r < rounds)
                rank[r] = static_cast<unsigned short>(CountRound<kBits>(
                    first + r * 32 < a.n ? (rec[r].x >> p.shift) & p.mask : p.bins, p, counts + warp * p.bins));
        __syncthreads();
        ScanDigits(counts, warps, p.bins, base);
    };
    auto place = [&](const SortPass& p, int r) {
        const int d = (rec[r].x >> p.shift) & p.mask;
        return base[d] + counts[warp * p.bins + d] + rank[r];
    };
#pragma unroll
    for (int r = 0; r < kWideRounds; ++r)
        rec[r] = r < rounds && first + r * 32 < a.n ? make_int2(KeyOf(a, first + r * 32), first + r * 32) : make_int2(0, 0);
    pass(a);
#pragma unroll
    for (int r = 0; r < kWideRounds; ++r)
        if (r < rounds && first + r * 32 < a.n) records[place(a, r)] = rec[r];
    __syncthreads();
    for (int i = threadIdx.x; i < warps * b.bins; i += blockDim.x) counts[i] = 0;
#pragma unroll
    for (int r = 0; r < kWideRounds; ++r)
        if (r < rounds && first + r * 32 < a.n) rec[r] = records[first + r * 32];
    __syncthreads();
    pass(b);
#pragma unroll
    for (int r = 0; r < kWideRounds; ++r)
        if (r < rounds && first + r * 32 < a.n) {
            const int to = place(b, r);
            order[to] = rec[r].y;
            position[rec[r].y] = to;
            sorted[to] = rec[r].x;  // every record is in registers by now
        }
    __syncthreads();
    for (int r0 = warp * 32; r0 <= a.n; r0 += blockDim.x) {
        const int r = r0 + lane;
        FillOffsets(r, r <= a.n ? (r > 0 ? sorted[r - 1] : -1) : 0, r < a.n ? sorted[r] : r == a.n ? a.experts : -1, offsets);
    }
}

// hist[b * tiles + tile] = keys of digit b in the tile.
template <int kPerWarp>
__global__ void __launch_bounds__(kSortBlock) SortCountKernel(SortPass a, int* hist) {
    constexpr int kTile = kSortWarps * kPerWarp;
    extern __shared__ int base[];  // [bins]
    LetLaterStart();
    for (int b = threadIdx.x; b < a.bins; b += kSortBlock) base[b] = 0;
    __syncthreads();
    WaitForEarlier();
    const int first = blockIdx.x * kTile + threadIdx.x;
    int key[kTile / kSortBlock];
#pragma unroll
    for (int r = 0; r < kTile / kSortBlock; ++r) key[r] = first + r * kSortBlock < a.n ? KeyOf(a, first + r * kSortBlock) : -1;
#pragma unroll
    for (int r = 0; r < kTile / kSortBlock; ++r)
        if (key[r] >= 0) atomicAdd(base + ((key[r] >> a.shift) & a.mask), 1);  // whole numbers: in any order
    __syncthreads();
    for (int b = threadIdx.x; b < a.bins; b += kSortBlock) hist[static_cast<int64_t>(b) * a.tiles + blockIdx.x] = base[b];
}

// One warp per digit: its counts to the sums over the tiles before, its total to sums[].
constexpr int kScanBlock = 256;
__global__ void __launch_bounds__(kScanBlock) SortScanKernel(int* hist, int bins, int tiles, int* sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    LetLaterStart();
    WaitForEarlier();
    const int b = blockIdx.x * (kScanBlock / 32) + warp;
    if (b >= bins) return;
    int* own = hist + static_cast<int64_t>(b) * tiles;
    int carry = 0;
    for (int t0 = 0; t0 < tiles; t0 += 128) {
        int v[4], s = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = t0 + lane * 4 + i < tiles ? own[t0 + lane * 4 + i] : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) s += v[i];
        const int mine = s;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        int before = carry + s - mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (t0 + lane * 4 + i < tiles) own[t0 + lane * 4 + i] = before;
            before += v[i];
        }
        carry += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) sums[b] = carry;
}

// offsets of a two-pass sort from its sorted keys.
__global__ void SortOffsetsKernel(const int* sorted, int n, int experts, int* offsets) {
    LetLaterStart();
    WaitForEarlier();
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    FillOffsets(r, r <= n ? (r > 0 ? sorted[r - 1] : -1) : 0, r < n ? sorted[r] : r == n ? experts : -1, offsets);
}

// Each key to its place: the first of two passes writes records, the last one the order, the positions and
// (two passes) the sorted keys.  offsets (one pass): where each digit begins.  The tile is put in order in shared
// memory first, so that neighbouring threads write neighbouring elements of a digit (written from where the keys
// lay, a pass of a million took 27 us, most of them for partly filled sectors).
template <int kBits, int kPerWarp>
__global__ void __launch_bounds__(kSortBlock)
    SortScatterKernel(SortPass a, const int* hist, const int* sums, int2* records,
                      int* sorted, int* order, int* position, int* offsets) {
    constexpr int kTile = kSortWarps * kPerWarp;
    extern __shared__ int2 tile[];  // [kTile], then the digits' places [2][bins] and the counts [kSortWarps][bins]
    __shared__ int part[32];
    int* local = reinterpret_cast<int*>(tile + kTile);  // of the digit's first key in the tile
    int* shift = local + a.bins;                        // from there to its place in the result
    unsigned short* counts = reinterpret_cast<unsigned short*>(shift + a.bins);
    LetLaterStart();
    for (int i = threadIdx.x; i < kSortWarps * a.bins; i += kSortBlock) counts[i] = 0;
    __syncthreads();
    WaitForEarlier();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = blockIdx.x * kTile + warp * kPerWarp + lane;
    int2 rec[kPerWarp / 32];
    unsigned short rank[kPerWarp / 32];
#pragma unroll
    for (int r = 0; r < kPerWarp / 32; ++r) {
        const int i = first + r * 32;
        rec[r] = i >= a.n ? make_int2(-1, 0) : a.records ? a.records[i] : make_int2(KeyOf(a, i), i);
    }
#pragma unroll
    for (int r = 0; r < kPerWarp / 32; ++r)
        rank[r] = static_cast<unsigned short>(
            CountRound<kBits>(rec[r].x < 0 ? a.bins : (rec[r].x >> a.shift) & a.mask, a, counts + warp * a.bins));
    __syncthreads();
    int before_all = 0, before_own = 0;
    for (int b0 = 0; b0 < a.bins; b0 += kSortBlock) {
        const int b = b0 + threadIdx.x;
        int own = 0;
        if (b < a.bins)
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                const int c = counts[w * a.bins + b];
                counts[w * a.bins + b] = static_cast<unsigned short>(own);
                own += c;
            }
        int all, all_own;
        const int start = before_all + ScanThreads(b < a.bins ? sums[b] : 0, part, &all);
        const int mine = before_own + ScanThreads(own, part, &all_own);
        if (b < a.bins) {
            local[b] = mine;
            shift[b] = start + hist[static_cast<int64_t>(b) * a.tiles + blockIdx.x] - mine;
            if (offsets && blockIdx.x == 0) offsets[b] = start;
        }
        before_all += all;
        before_own += all_own;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kPerWarp / 32; ++r) {
        if (rec[r].x < 0) continue;
        const int d = (rec[r].x >> a.shift) & a.mask;
        tile[local[d] + counts[warp * a.bins + d] + rank[r]] = rec[r];
    }
    __syncthreads();
    const int n = min(kTile, a.n - static_cast<int>(blockIdx.x) * kTile);
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kSortBlock) {
        const int2 v = tile[i];
        const int to = shift[(v.x >> a.shift) & a.mask] + i;
        if (records) {
            records[to] = v;
        } else {
            order[to] = v.y;
            position[v.y] = to;
            if (sorted) sorted[to] = v.x;
        }
    }
}

__global__ void ZeroKernel(int* p, int n) {
    LetLaterStart();
    WaitForEarlier();
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) p[i] = 0;
}

struct SortPlan {
    int bins[2], shift[2], passes, tile, tiles;
    size_t sums, records, sorted, bytes;  // places in the workspace, which begins with the counts of each tile
};

bool Alone(int64_t n, int experts) { return n <= (experts + 1 <= kOneBins ? kAlone : kWide); }

SortPlan PlanSort(int64_t n, int experts) {
    SortPlan p{};
    p.tile = kSortWarps * (n <= kFewPairs ? kFewPerWarp : kManyPerWarp);
    p.tiles = static_cast<int>((n + p.tile - 1) / p.tile);
    if (experts + 1 <= kOneBins) {
        p.passes = 1;
        p.bins[0] = experts + 1;
    } else {
        int bits = 1;
        while ((experts >> bits) != 0) ++bits;
        p.passes = 2;
        p.shift[1] = (bits + 1) / 2;
        p.bins[0] = 1 << p.shift[1];
        p.bins[1] = (experts >> p.shift[1]) + 1;
    }
    if (Alone(n, experts)) return p;  // no workspace
    const auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
    const size_t most = std::max(p.bins[0], p.bins[1]);
    p.sums = up(most * p.tiles * sizeof(int));
    p.records = p.sums + up(most * sizeof(int));
    p.sorted = p.bytes = p.records;
    if (p.passes == 2) {
        p.sorted = p.records + up(static_cast<size_t>(n) * sizeof(int2));
        p.bytes = p.sorted + up(static_cast<size_t>(n) * sizeof(int));
    }
    return p;
}

size_t SortSmem(int warps, int bins) { return static_cast<size_t>(bins) * 4 + static_cast<size_t>(warps) * bins * 2; }

// ---- exchange ----------------------------------------------------------------------------------

// Rows of `bytes` bytes as packs of V: dispatch copies whatever the element type is.  L threads per
// token, which read a piece of its row once and write it to every choice, so that a token's row crosses
// memory once in and topk times out.  Bound by the writes: 16,384 x 8 x 2,048 bfloat16 in 100 us, 6.0 TB/s
// (the copy rate measured is 6.54); 64 x 8 x 256 in 1.8 us.
template <typename V, int L>
__global__ void __launch_bounds__(kBlock)
    DispatchKernel(const unsigned char* x, int64_t ldx, int64_t tokens, int packs, int topk,
                   const int* position, const int* offsets, int experts, int pairs,
                   unsigned char* out, int64_t ldo) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kBlock / L) + threadIdx.x / L;
    LetLaterStart();
    WaitForEarlier();
    if (t >= tokens) return;
    const int kept = Kept(offsets, experts, pairs);
    const V* row = reinterpret_cast<const V*>(x + t * ldx);
    for (int c = threadIdx.x % L; c < packs; c += L) {
        const V v = row[c];
        for (int j0 = 0; j0 < topk; j0 += 4) {  // four positions in flight
            int p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = j0 + j < topk ? position[t * topk + j0 + j] : -1;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (static_cast<unsigned>(p[j]) < static_cast<unsigned>(pairs))
                    reinterpret_cast<V*>(out + p[j] * ldo)[c] = p[j] < kept ? v : V{};
        }
    }
}

// out[t] = sum over the kept choices of w[t, j] y[position[t, j]], j ascending, in 32 bits, rounded once.  Rows of
// dropped choices are never read.  Null weights are ones (the gradient of dispatch).  By token rather than by
// sorted row, so that nothing is added through memory and the sum has one order.  Bound by reading y:
// 16,384 x 8 x 2,048 bfloat16 in 92 us, 6.5 TB/s; 64 x 8 x 256 in 2.4 us.
template <typename T, int N, int L>
__global__ void __launch_bounds__(kBlock)
    CombineKernel(const T* y, int64_t ldy, int64_t tokens, int cols, int topk,
                  const void* weights, int wtype, const int* position,
                  const int* offsets, int experts, int pairs, T* out, int64_t ldo) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kBlock / L) + threadIdx.x / L;
    LetLaterStart();
    WaitForEarlier();
    if (t >= tokens) return;
    const unsigned kept = static_cast<unsigned>(Kept(offsets, experts, pairs));
    const int full = cols / N;
    for (int c = threadIdx.x % L; c < full; c += L) {
        float acc[N];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.0f;
        // Four choices' rows in flight; a dropped one adds nothing (its row may hold anything, so it is not a
        // product with 0).
        for (int j0 = 0; j0 < topk; j0 += 4) {
            unsigned p[4];
            Pack<T, N> v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = j0 + j < topk ? static_cast<unsigned>(position[t * topk + j0 + j]) : kept;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p[j] < kept) Load<true>(v[j], y + p[j] * ldy + static_cast<int64_t>(c) * N);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p[j] < kept) {
                    const float w = weights ? LoadAs(weights, t * topk + j0 + j, wtype) : 1.0f;
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[i] = fmaf(w, ToFloat(v[j].v[i]), acc[i]);
                }
        }
        Pack<T, N> r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = FromFloat<T>(acc[i]);
        *reinterpret_cast<Pack<T, N>*>(out + t * ldo + static_cast<int64_t>(c) * N) = r;
    }
    for (int c = full * N + threadIdx.x % L; c < cols; c += L) {
        float acc = 0.0f;
        for (int j = 0; j < topk; ++j) {
            const unsigned p = static_cast<unsigned>(position[t * topk + j]);
            if (p >= kept) continue;
            acc = fmaf(weights ? LoadAs(weights, t * topk + j, wtype) : 1.0f, ToFloat(y[p * ldy + c]), acc);
        }
        out[t * ldo + c] = FromFloat<T>(acc);
    }
}

// The gradient of combine: dy[position[t, j]] = w[t, j] dout[t], dw[t, j] = <dout[t], y[position[t, j]]>,
// zeros where the choice was dropped.  By token, so that dout is read once; dw's sum over the row goes through
// registers, then the group's warps in order.  Bound by reading y and writing dy: 16,384 x 4 x 4,096 bfloat16 in
// 187 us, 6.5 TB/s; 64 x 8 x 256 in 4.0 us.
template <typename T, int N, int L>
__global__ void __launch_bounds__(kBlock, 4)
    CombineBackwardKernel(const T* dout, int64_t ldd, const T* y, int64_t ldy, int64_t tokens,
                          int cols, int topk, const void* weights, int wtype,
                          const int* position, const int* offsets, int experts, int pairs,
                          T* dy, int64_t lddy, void* dweights) {
    extern __shared__ float part[];  // [kBlock / 32][topk]
    const int group = threadIdx.x / L, at = threadIdx.x % L, warp = threadIdx.x >> 5;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kBlock / L) + group;
    const bool real = t < tokens;
    LetLaterStart();
    WaitForEarlier();
    const int kept = Kept(offsets, experts, pairs);
    const int full = cols / N;
    const T* d = dout + (real ? t : 0) * ldd;
    // Four choices at a time, their rows of y in flight together; dout comes from the cache after the first four.
    for (int j0 = 0; j0 < topk; j0 += 4) {
        int p[4];
        float w[4], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[j] = real && j0 + j < topk ? position[t * topk + j0 + j] : -1;
            if (p[j] >= pairs) p[j] = -1;
            w[j] = p[j] >= 0 && p[j] < kept ? LoadAs(weights, t * topk + j0 + j, wtype) : 0.0f;
        }
        for (int c = at; c < full; c += L) {
            const int64_t e = static_cast<int64_t>(c) * N;
            Pack<T, N> v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p[j] >= 0 && p[j] < kept) Load<false>(v[j], y + p[j] * ldy + e);
            const Pack<T, N> g = real ? *reinterpret_cast<const Pack<T, N>*>(d + e) : Pack<T, N>{};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (p[j] < 0) continue;
                Pack<T, N> r{};  // zeros for a dropped choice, whose row of y is not read
                if (p[j] < kept) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        sum[j] = fmaf(ToFloat(g.v[i]), ToFloat(v[j].v[i]), sum[j]);
                        r.v[i] = FromFloat<T>(__fmul_rn(w[j], ToFloat(g.v[i])));
                    }
                }
                StoreStreaming(dy + p[j] * lddy + e, r);
            }
        }
        if (full * N < cols)
            for (int c = full * N + at; c < cols; c += L) {
                const float g = real ? ToFloat(d[c]) : 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (p[j] < 0) continue;
                    if (p[j] < kept) sum[j] = fmaf(g, ToFloat(y[p[j] * ldy + c]), sum[j]);
                    dy[p[j] * lddy + c] = FromFloat<T>(p[j] < kept ? __fmul_rn(w[j], g) : 0.0f);
                }
            }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            for (int o = 16; o > 0; o >>= 1) sum[j] += __shfl_down_sync(0xffffffffu, sum[j], o);
            if ((threadIdx.x & 31) == 0 && j0 + j < topk) part[warp * topk + j0 + j] = sum[j];
        }
    }
    __syncthreads();
    if (!real) return;
    for (int j = at; j < topk; j += L) {
        float sum = 0.0f;
        for (int w = 0; w < L / 32; ++w) sum += part[(group * (L / 32) + w) * topk + j];
        StoreAs(dweights, t * topk + j, wtype, sum);
    }
}

// ---- host --------------------------------------------------------------------------------------

bool IsFloat(int dtype) { return dtype == STLQ_B200_F32 || dtype == STLQ_B200_BF16 || dtype == STLQ_B200_F16; }
int64_t SizeOf(int dtype) { return dtype == STLQ_B200_F32 ? 4 : 2; }

// Sets a kernel's dynamic shared memory limit, once for each device.
template <typename K>
cudaError_t MostSmem(K kernel, size_t bytes) {
    struct Seen {
        const void* kernel;
        int device;
    };
    static thread_local Seen seen[8];
    static thread_local int used = 0;
    int device = 0;
    if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return e;
    for (int i = 0; i < used; ++i)
        if (seen[i].kernel == reinterpret_cast<const void*>(kernel) && seen[i].device == device) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == cudaSuccess && used < 8) seen[used++] = {reinterpret_cast<const void*>(kernel), device};
    return e;
}

template <typename F>
void ForType(int dtype, F&& f) {
    if (dtype == STLQ_B200_F32) f(float{});
    else if (dtype == STLQ_B200_BF16) f(__nv_bfloat16{});
    else f(__half{});
}

// The widest pack of T that the bases and row strides allow: 16 bytes, 8, 4, or one element.  An odd number of 16-bit
// columns leaves one element a pack, which takes longer than 16 bytes do: 16,384 x 4 x 2,047 against 2,048, dispatch 2.0
// times (109 us), combine 2.4 (128), its gradient 2.4 (237).
template <typename T, typename F>
void ForWidth(std::initializer_list<const void*> bases, std::initializer_list<int64_t> strides, F&& f) {
    uint64_t all = 16;
    for (const void* p : bases) all |= reinterpret_cast<uintptr_t>(p);
    for (const int64_t v : strides) all |= static_cast<uint64_t>(v) * sizeof(T);
    if (all % 16 == 0) f(std::integral_constant<int, 16 / sizeof(T)>{});
    else if (all % 8 == 0) f(std::integral_constant<int, 8 / sizeof(T)>{});
    else if (sizeof(T) == 2 && all % 4 == 0) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 1>{});
}

// Threads per row: a warp for short rows, otherwise enough that a thread has at most `each` packs of it; more where
// there are few rows, up to one pack a thread, as the time that one row takes is then the call's.
// Rows shorter than a warp's packs leave lanes idle: a million rows of 128 bfloat16 to 16,384 experts take combine 299 us,
// 1.7 TB/s, and its gradient 522 us; dispatch 135 us, 3.8 TB/s.
template <typename F>
void ForLanes(int64_t packs, int each, int64_t rows, int sms, F&& f) {
    int lanes = packs <= 32 * each ? 32 : packs <= 128 * each ? 128 : 256;
    if (rows * lanes < 1024 * static_cast<int64_t>(sms)) lanes = packs <= 32 ? 32 : packs <= 128 ? 128 : 256;
    if (lanes == 32) f(std::integral_constant<int, 32>{});
    else if (lanes == 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 256>{});
}

// Blocks for `rows` rows at L threads each; 0 if they do not fit a grid.
unsigned Blocks(int64_t rows, int L) {
    const int64_t b = (rows + kBlock / L - 1) / (kBlock / L);
    return b > 0x7fffffff ? 0u : static_cast<unsigned>(b);
}

int CheckRouting(int64_t tokens, int topk, int experts, const void* position, const void* offsets) {
    if (tokens < 0 || topk < 1 || topk > STLQ_B200_MAX_TOPK) return Bad("tokens >= 0 and 1 <= topk <= 64 required");
    if (experts < 1 || experts > STLQ_B200_MAX_ROOT) return Bad("1 <= experts <= 65536 required");
    if (tokens > kMostPairs / topk) return Bad("tokens * topk must be at most 2^31 - 1024");
    if (tokens > 0 && (!position || !offsets)) return Bad("null position or offsets");
    if (!Aligned(position, 4) || !Aligned(offsets, 4)) return Bad("position and offsets must be 4-byte aligned");
    return 0;
}

int CheckCols(int64_t cols) {
    if (cols < 0) return Bad("cols must be >= 0");
    if (cols > kMostCols) return Bad("cols must be at most 2^31 - 4096");
    return 0;
}

int Quantize(stlq_b200_kernels* k, const void* x, int x_dtype, int64_t ldx, int64_t rows, int cols, int topk,
             const int* position, const int* offsets, int experts, int8_t* q, int64_t ldq, float* scale, void* stream) {
    if (!IsFloat(x_dtype)) return Bad("x_dtype must be F32, BF16 or F16");
    if (rows < 0) return Bad("rows must be >= 0");
    if (int rc = CheckCols(cols)) return rc;
    if (ldx < cols || ldq < cols) return Bad("ldx or ldq below cols");
    if (rows == 0) return 0;
    if (!scale || (cols > 0 && (!x || !q))) return Bad("null pointer");
    if (!Aligned(x, SizeOf(x_dtype)) || !Aligned(scale, 4)) return Bad("x or scale not aligned to its element");
    DeviceScope scope(k->device);
    if (!scope.ok()) return SetError(STLQ_B200_ECUDA, "cudaSetDevice failed");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int pairs = position ? static_cast<int>(rows * topk) : 0;
    bool fits = true;
    cudaError_t error = cudaSuccess;
    ForType(x_dtype, [&](auto one) {
        using T = decltype(one);
        const T* xp = static_cast<const T*>(x);
        // A pack of N values is N bytes of q, so q's alignment counts as x's does.
        ForWidth<T>({x, reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(q) * sizeof(T))}, {ldx, ldq}, [&](auto width) {
            constexpr int N = decltype(width)::value;
            using std::integral_constant;
            const auto lay = [&](auto lanes, auto held) {
                constexpr int L = decltype(lanes)::value, H = decltype(held)::value;
                const unsigned grid = Blocks(rows, L);
                fits = grid != 0;
                const auto launch = [&](auto kernel) {
                    error = LaunchAfter(kernel, grid, kBlock, 0, s, xp, ldx, rows, cols, topk, position, offsets, experts, pairs, q, ldq, scale);
                };
                if (!fits) return;
                if (position) launch(QuantizeRowsKernel<T, N, L, H, true>);
                else launch(QuantizeRowsKernel<T, N, L, H, false>);
            };
            const int packs = cols / N;
            if constexpr (N * sizeof(T) != 16) {
                const integral_constant<int, 4> four;
                const integral_constant<int, N == 1 ? 8 : 4> most;  // single elements cost few registers
                if (packs <= 128) lay(integral_constant<int, 32>{}, four);
                else if (packs <= 256 && N == 1) lay(integral_constant<int, 32>{}, most);
                else if (packs <= 512) lay(integral_constant<int, 128>{}, four);
                else if (packs <= 1024) lay(integral_constant<int, 256>{}, four);
                else lay(integral_constant<int, 256>{}, most);
            } else if (packs > 16 && rows * ((packs + 3) / 4) < 1024 * static_cast<int64_t>(k->num_sms)) {
                // Few rows: the time of one counts.
                const integral_constant<int, 2> two;
                if (packs <= 64) lay(integral_constant<int, 32>{}, two);
                else if (packs <= 128) lay(integral_constant<int, 64>{}, two);
                else lay(integral_constant<int, 256>{}, two);
            } else {
                const integral_constant<int, 4> four;
                if (packs <= 16) lay(integral_constant<int, 4>{}, four);
                else if (packs <= 32) lay(integral_constant<int, 8>{}, four);
                else if (packs <= 64) lay(integral_constant<int, 16>{}, four);
                else if (packs <= 128) lay(integral_constant<int, 32>{}, four);
                else if (packs <= 256) lay(integral_constant<int, 64>{}, four);
                else if (packs <= 512) lay(integral_constant<int, 128>{}, four);
                else lay(integral_constant<int, 256>{}, four);
            }
        });
    });
    if (!fits) return Bad("too many rows");
    return Ck(error, "quantize_rows");
}

}  // namespace

extern "C" {

int stlq_b200_quantize_rows(stlq_b200_kernels* k, const void* x, int x_dtype, int64_t ldx, int64_t rows, int cols,
                            int8_t* q, int64_t ldq, float* scale, void* stream) {
    return Guard([&] {
        if (!k) return Bad("kernel-provider handle is null");
        return Quantize(k, x, x_dtype, ldx, rows, cols, 1, nullptr, nullptr, 0, q, ldq, scale, stream);
    });
}

int stlq_b200_dispatch_i8(stlq_b200_kernels* k, const void* x, int x_dtype, int64_t ldx, int64_t tokens, int cols, int topk,
                          const int32_t* position, const int32_t* offsets, int experts, int8_t* q, int64_t ldq,
                          float* scale, void* stream) {
    return Guard([&] {
        if (!k) return Bad("kernel-provider handle is null");
        if (int rc = CheckRouting(tokens, topk, experts, position, offsets)) return rc;
        return Quantize(k, x, x_dtype, ldx, tokens, cols, topk, position, offsets, experts, q, ldq, scale, stream);
    });
}

int stlq_b200_sort_by_expert_workspace(int64_t tokens, int topk, int experts, size_t* bytes) {
    return Guard([&] {
        if (!bytes) return Bad("bytes is null");
        *bytes = 0;
        if (int rc = CheckRouting(tokens, topk, experts, bytes, bytes)) return rc;
        *bytes = PlanSort(tokens * topk, experts).bytes;
        return 0;
    });
}

int stlq_b200_sort_by_expert(stlq_b200_kernels* k, const void* ids, int ids_dtype, int64_t tokens, int topk, int experts,
                             int32_t* order, int32_t* position, int32_t* offsets, void* workspace, size_t workspace_bytes,
                             void* stream) {
    return Guard([&] {
        if (!k) return Bad("kernel-provider handle is null");
        if (ids_dtype != STLQ_B200_I32 && ids_dtype != STLQ_B200_I64) return Bad("ids_dtype must be I32 or I64");
        if (int rc = CheckRouting(tokens, topk, experts, position, offsets)) return rc;
        if (!offsets) return Bad("null offsets");
        const int n = static_cast<int>(tokens * topk);
        if (n > 0 && (!ids || !order)) return Bad("null ids or order");
        if (!Aligned(ids, ids_dtype == STLQ_B200_I64 ? 8 : 4) || !Aligned(order, 4)) return Bad("ids or order not aligned to its element");
        const SortPlan p = PlanSort(n, experts);
        if (workspace_bytes < p.bytes || (p.bytes && (!workspace || !Aligned(workspace, 16))))
            return Bad("workspace below stlq_b200_sort_by_expert_workspace's bytes, or not 16-byte aligned");
        DeviceScope scope(k->device);
        if (!scope.ok()) return SetError(STLQ_B200_ECUDA, "cudaSetDevice failed");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (n == 0) return Ck(LaunchAfter(ZeroKernel, std::min(experts / 256 + 1, 64), 256, 0, s, offsets, experts + 1), "sort_by_expert");
        SortPass a{ids, ids_dtype == STLQ_B200_I64, nullptr, n, experts, 0, 0x7fffffff, experts + 1, p.tiles};
        const size_t most = 76 << 10;
        if (Alone(n, experts)) {
            // As many warps as there are rounds for, so that few pairs take one round, and not too few for the digits.
            const int digits = std::max(p.bins[0], p.bins[1]);
            const int warps = std::min(kAloneBlock / 32, std::max((n + 31) / 32, (digits + 127) / 128));
            const int rounds = (n + warps * 32 - 1) / (warps * 32);
            if (p.passes == 2) {
                a.bins = p.bins[0];
                a.mask = p.bins[0] - 1;
                const SortPass b{nullptr, 0, nullptr, n, experts, p.shift[1], 0x7fffffff, p.bins[1], 0};
                const auto kernel = digits < 256 ? SortWideKernel<8> : SortWideKernel<11>;
                if (int rc = Ck(MostSmem(kernel, 112 << 10), "sort_by_expert")) return rc;
                return Ck(LaunchAfter(kernel, 1, warps * 32, n * sizeof(int2) + SortSmem(warps, digits), s, a, b, rounds, order, position, offsets), "sort_by_expert");
            }
            const auto kernel = a.bins < 256 ? SortAloneKernel<8> : SortAloneKernel<11>;
            if (int rc = Ck(MostSmem(kernel, most), "sort_by_expert")) return rc;
            return Ck(LaunchAfter(kernel, 1, warps * 32, SortSmem(warps, a.bins), s, a, rounds, order, position, offsets), "sort_by_expert");
        }
        char* ws = static_cast<char*>(workspace);
        int* hist = reinterpret_cast<int*>(ws);
        int* sums = reinterpret_cast<int*>(ws + p.sums);
        int2* records = reinterpret_cast<int2*>(ws + p.records);
        int* sorted = reinterpret_cast<int*>(ws + p.sorted);
        const auto pass = [&](const SortPass& x, int2* records_out, int* sorted_out, int* offsets_out) {
            const int blocks = (x.bins + kScanBlock / 32 - 1) / (kScanBlock / 32);
            const bool few = p.tile == kSortWarps * kFewPerWarp;
            const auto count = few ? SortCountKernel<kFewPerWarp> : SortCountKernel<kManyPerWarp>;
            const auto scatter = x.bins < 256 ? (few ? SortScatterKernel<8, kFewPerWarp> : SortScatterKernel<8, kManyPerWarp>)
                                              : (few ? SortScatterKernel<11, kFewPerWarp> : SortScatterKernel<11, kManyPerWarp>);
            if (int rc = Ck(MostSmem(scatter, most), "sort_by_expert")) return rc;
            if (int rc = Ck(LaunchAfter(count, p.tiles, kSortBlock, x.bins * sizeof(int), s, x, hist), "sort_by_expert")) return rc;
            if (int rc = Ck(LaunchAfter(SortScanKernel, blocks, kScanBlock, 0, s, hist, x.bins, p.tiles, sums), "sort_by_expert")) return rc;
            return Ck(LaunchAfter(scatter, p.tiles, kSortBlock, p.tile * sizeof(int2) + x.bins * sizeof(int) + SortSmem(kSortWarps, x.bins), s, x, hist, sums, records_out, sorted_out, order, position, offsets_out), "sort_by_expert");
        };
        if (p.passes == 1) return pass(a, nullptr, nullptr, offsets);
        a.mask = p.bins[0] - 1;
        a.bins = p.bins[0];
        if (int rc = pass(a, records, nullptr, nullptr)) return rc;
        const SortPass b{nullptr, 0, records, n, experts, p.shift[1], 0x7fffffff, p.bins[1], p.tiles};
        if (int rc = pass(b, nullptr, sorted, nullptr)) return rc;
        return Ck(LaunchAfter(SortOffsetsKernel, n / 256 + 1, 256, 0, s, sorted, n, experts, offsets), "sort_by_expert");
    });
}

int stlq_b200_dispatch(stlq_b200_kernels* k, const void* x, int elem_bytes, int64_t ldx, int64_t tokens, int cols, int topk,
                       const int32_t* position, const int32_t* offsets, int experts, void* out, int64_t ldo, void* stream) {
    return Guard([&] {
        if (!k) return Bad("kernel-provider handle is null");
        if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) return Bad("elem_bytes must be 1, 2 or 4");
        if (int rc = CheckRouting(tokens, topk, experts, position, offsets)) return rc;
        if (int rc = CheckCols(cols)) return rc;
        if (ldx < cols || ldo < cols) return Bad("ldx and ldo must be at least cols");
        if (tokens == 0 || cols == 0) return 0;
        if (!x || !out) return Bad("null x or out");
        if (!Aligned(x, elem_bytes) || !Aligned(out, elem_bytes)) return Bad("x or out not aligned to its element");
        if (cols > 0x7fffffff / elem_bytes) return Bad("rows of 2^31 bytes or more");
        DeviceScope scope(k->device);
        if (!scope.ok()) return SetError(STLQ_B200_ECUDA, "cudaSetDevice failed");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const int pairs = static_cast<int>(tokens * topk);
        const int bytes = cols * elem_bytes;
        const int64_t bx = ldx * elem_bytes, bo = ldo * elem_bytes;
        bool fits = true;
        cudaError_t error = cudaSuccess;
        auto launch = [&](auto pack) {
            using V = decltype(pack);
            const int packs = bytes / static_cast<int>(sizeof(V));
            ForLanes(packs, 4, tokens, k->num_sms, [&](auto lanes) {
                constexpr int L = decltype(lanes)::value;
                const unsigned grid = Blocks(tokens, L);
                fits = grid != 0;
                if (!fits) return;
                error = LaunchAfter(DispatchKernel<V, L>, grid, kBlock, 0, s, static_cast<const unsigned char*>(x), bx, tokens, packs, topk,
                                                             position, offsets, experts, pairs,
                                                             static_cast<unsigned char*>(out), bo);
            });
        };
        // The widest access that the rows, their strides and both bases allow.
        auto fit = [&](int v) { return bytes % v == 0 && bx % v == 0 && bo % v == 0 && Aligned(x, v) && Aligned(out, v); };
        if (fit(16)) launch(uint4{});
        else if (fit(8)) launch(uint2{});
        else if (fit(4)) launch(uint32_t{});
        else if (fit(2)) launch(uint16_t{});
        else launch(uint8_t{});
        if (!fits) return Bad("too many tokens");
        return Ck(error, "dispatch");
    });
}

int stlq_b200_combine(stlq_b200_kernels* k, const void* y, int dtype, int64_t ldy, int64_t tokens, int cols, int topk,
                      const void* weights, int weights_dtype, const int32_t* position, const int32_t* offsets, int experts,
                      void* out, int64_t ldo, void* stream) {
    return Guard([&] {
        if (!k) return Bad("kernel-provider handle is null");
        if (!IsFloat(dtype) || (weights && !IsFloat(weights_dtype))) return Bad("dtypes must be F32, BF16 or F16");
        if (int rc = CheckRouting(tokens, topk, experts, position, offsets)) return rc;
        if (int rc = CheckCols(cols)) return rc;
        if (ldy < cols || ldo < cols) return Bad("ldy and ldo must be at least cols");
        if (tokens == 0 || cols == 0) return 0;
        if (!y || !out) return Bad("null y or out");
        if (!Aligned(y, SizeOf(dtype)) || !Aligned(out, SizeOf(dtype)) || (weights && !Aligned(weights, SizeOf(weights_dtype))))
            return Bad("y, weights or out not aligned to its element");
        DeviceScope scope(k->device);
        if (!scope.ok()) return SetError(STLQ_B200_ECUDA, "cudaSetDevice failed");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const int pairs = static_cast<int>(tokens * topk);
        bool fits = true;
        cudaError_t error = cudaSuccess;
        ForType(dtype, [&](auto one) {
            using T = decltype(one);
            ForWidth<T>({y, out}, {ldy, ldo}, [&](auto width) {
                constexpr int N = decltype(width)::value;
                ForLanes(cols / N, N * sizeof(T) == 16 ? 4 : 8, tokens, k->num_sms, [&](auto lanes) {
                    constexpr int L = decltype(lanes)::value;
                    const unsigned grid = Blocks(tokens, L);
                    fits = grid != 0;
                    if (fits)
                        error = LaunchAfter(CombineKernel<T, N, L>, grid, kBlock, 0, s, static_cast<const T*>(y), ldy, tokens, cols, topk,
                                            weights, weights_dtype, position, offsets, experts, pairs, static_cast<T*>(out), ldo);
                });
            });
        });
        if (!fits) return Bad("too many tokens");
        return Ck(error, "combine");
    });
}

int stlq_b200_combine_backward(stlq_b200_kernels* k, const void* dout, int dtype, int64_t ldd, const void* y, int64_t ldy,
                               int64_t tokens, int cols, int topk, const void* weights, int weights_dtype,
                               const int32_t* position, const int32_t* offsets, int experts, void* dy, int64_t lddy,
                               void* dweights, void* stream) {
    return Guard([&] {
        if (!k) return Bad("kernel-provider handle is null");
        if (!IsFloat(dtype) || !IsFloat(weights_dtype)) return Bad("dtypes must be F32, BF16 or F16");
        if (int rc = CheckRouting(tokens, topk, experts, position, offsets)) return rc;
        if (int rc = CheckCols(cols)) return rc;
        if (ldd < cols || ldy < cols || lddy < cols) return Bad("leading dimensions must be at least cols");
        if (tokens == 0) return 0;
        if (!weights || !dweights || (cols > 0 && (!dout || !y || !dy))) return Bad("null pointer");
        if (!Aligned(dout, SizeOf(dtype)) || !Aligned(y, SizeOf(dtype)) || !Aligned(dy, SizeOf(dtype)) ||
            !Aligned(weights, SizeOf(weights_dtype)) || !Aligned(dweights, SizeOf(weights_dtype)))
            return Bad("a pointer is not aligned to its element");
        DeviceScope scope(k->device);
        if (!scope.ok()) return SetError(STLQ_B200_ECUDA, "cudaSetDevice failed");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const int pairs = static_cast<int>(tokens * topk);
        const size_t smem = sizeof(float) * (kBlock / 32) * topk;
        bool fits = true;
        cudaError_t error = cudaSuccess;
        ForType(dtype, [&](auto one) {
            using T = decltype(one);
            ForWidth<T>({dout, y, dy}, {ldd, ldy, lddy}, [&](auto width) {
                constexpr int N = decltype(width)::value;
                ForLanes(cols / N, N * sizeof(T) == 16 ? 4 : 8, tokens, k->num_sms, [&](auto lanes) {
                    constexpr int L = decltype(lanes)::value;
                    const unsigned grid = Blocks(tokens, L);
                    fits = grid != 0;
                    if (fits)
                        error = LaunchAfter(CombineBackwardKernel<T, N, L>, grid, kBlock, smem, s, static_cast<const T*>(dout), ldd,
                                            static_cast<const T*>(y), ldy, tokens, cols, topk, weights, weights_dtype, position, offsets,
                                            experts, pairs, static_cast<T*>(dy), lddy, dweights);
                });
            });
        });
        if (!fits) return Bad("too many tokens");
        return Ck(error, "combine_backward");
    });
}

}  // extern "C"
