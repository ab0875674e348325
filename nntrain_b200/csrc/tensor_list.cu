// Global L2 norm over a list of separately allocated gradient tensors, and the
// clip that follows from it (ABI minor 36).
//
// The reference walks the leaves: one sum-of-squares launch and one scale
// launch per tensor with a host read between them (NNtrain.Core/Tensors/
// Tensor.CudaKernels.cs:119-854, NNtrain.Core/Torch/nn.cs:32-81).  Here a table
// of the tensors lies on the device and two or three launches serve all of
// them:
//
//   squares   one CTA per chunk of a tensor -> one binary64 partial per chunk
//   finish    partials -> tensor norms, norm and coefficient (short lists: in
//             the clip)
//   clip      one CTA per chunk again: destination = value * coefficient
//
//   n_t = sqrt(sum of v^2),  n = (float)sqrt(sum of n_t^2),
//   c   = n > max_norm ? max_norm / (n + 1e-6f) : 1
//
// Every sum is binary64 in a fixed order (no atomics), so the same list gives
// the same bits every time.  Squares of BFP8 values are summed as integers:
// sum over blocks of scale^2 * (sum of code^2), the inner sum exact, which
// keeps the fp32 -> fp64 conversions (16 per clock and SM) off the path.
// A norm that is not finite in binary32 raises the flag and gives c = 1, so a
// list that holds a NaN or an Inf comes out as it went in.
//
// Bound: HBM.  The norm has to be known before the first value is written, so
// values are read twice; the clip walks the chunks from the back, where the
// values that the squares pass read last are still in L2 (126 MB).
#include "operator_launch.cuh"

#include "nntrain_grad_abi.h"

#include <algorithm>
#include <vector>

namespace ngb {
namespace {

enum TensorKind : int { kKindF32 = 0, kKindBf16 = 1, kKindBfp8 = 2 };

constexpr int kUnroll = 4;              // 128-bit loads in flight per thread
constexpr int kShiftedUnroll = 2;       // of two loads each
constexpr int kFinishThreads = 1024;

// A chunk is the same number of bytes for every kind: chunk_values fp32 values,
// twice as many bf16 and four times as many BFP8 ones.  It grows with the list
// (a 2048th of it) from 16 KB, one trip of a CTA, where a short list still
// covers the SMs, to 96 KB.  Measured on the 41.6 M-value bf16 list: 54 us with
// 16 KB chunks, 45 us with 48 KB, 49 us with 96 KB; on 1.54 G fp32 values 2.93 ms
// with 16 KB, 2.68 ms with 48 or 96 KB and 2.73 ms with 256 KB.
constexpr long long kChunkLeast = 4096, kChunkMost = 24576;

// Lists of at most this many chunks are finished by every CTA of the clip on
// its own, which saves a launch and its latency.
constexpr long long kFusedFinishChunks = 1024;

struct alignas(8) Chunk {
    int tensor;
    unsigned index;                     // the tensor's values [index, index + 1) * kind_values()
};

__host__ __device__ __forceinline__ long long kind_values(int chunk_values, int kind) {
    return static_cast<long long>(chunk_values) << kind;
}

__device__ __forceinline__ double square_of(float v) {
    const double d = static_cast<double>(v);
    return d * d;
}

// The unaligned head of a range that starts at `p`: values before the first
// 16-byte boundary (values are at least as aligned as their type).
__device__ __forceinline__ int head_values(const void* p, int value_bytes, int n) {
    const int head = static_cast<int>((16u - (static_cast<unsigned>(reinterpret_cast<std::uintptr_t>(p)) & 15u)) & 15u) / value_bytes;
    return head < n ? head : n;
}

__device__ double chunk_squares_f32(const float* p, int n) {
    const int head = head_values(p, 4, n), vectors = (n - head) >> 2, tail = head + vectors * 4;
    double a = 0.0, b = 0.0;
    if (static_cast<int>(threadIdx.x) < head) a += square_of(p[threadIdx.x]);
    if (tail + static_cast<int>(threadIdx.x) < n) b += square_of(p[tail + threadIdx.x]);
    const float4* body = reinterpret_cast<const float4*>(p + head);
    int i = threadIdx.x;
    for (; i + (kUnroll - 1) * kThreads < vectors; i += kUnroll * kThreads) {
        float4 x[kUnroll];
        #pragma unroll
        for (int j = 0; j < kUnroll; ++j) x[j] = __ldg(body + i + j * kThreads);
        #pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            a += square_of(x[j].x); b += square_of(x[j].y);
            a += square_of(x[j].z); b += square_of(x[j].w);
        }
    }
    for (; i < vectors; i += kThreads) {
        const float4 x = __ldg(body + i);
        a += square_of(x.x); b += square_of(x.y);
        a += square_of(x.z); b += square_of(x.w);
    }
    return a + b;
}

__device__ double chunk_squares_bf16(const unsigned short* p, int n) {
    const int head = head_values(p, 2, n), vectors = (n - head) >> 3, tail = head + vectors * 8;
    double a = 0.0, b = 0.0;
    if (static_cast<int>(threadIdx.x) < head) a += square_of(bf16_value(p[threadIdx.x]));
    if (tail + static_cast<int>(threadIdx.x) < n) b += square_of(bf16_value(p[tail + threadIdx.x]));
    const uint4* body = reinterpret_cast<const uint4*>(p + head);
    int i = threadIdx.x;
    for (; i + (kUnroll - 1) * kThreads < vectors; i += kUnroll * kThreads) {
        uint4 x[kUnroll];
        #pragma unroll
        for (int j = 0; j < kUnroll; ++j) x[j] = __ldg(body + i + j * kThreads);
        #pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            a += square_of(bf16_low(x[j].x)); b += square_of(bf16_high(x[j].x));
            a += square_of(bf16_low(x[j].y)); b += square_of(bf16_high(x[j].y));
            a += square_of(bf16_low(x[j].z)); b += square_of(bf16_high(x[j].z));
            a += square_of(bf16_low(x[j].w)); b += square_of(bf16_high(x[j].w));
        }
    }
    for (; i < vectors; i += kThreads) {
        const uint4 x = __ldg(body + i);
        a += square_of(bf16_low(x.x)); b += square_of(bf16_high(x.x));
        a += square_of(bf16_low(x.y)); b += square_of(bf16_high(x.y));
        a += square_of(bf16_low(x.z)); b += square_of(bf16_high(x.z));
        a += square_of(bf16_low(x.w)); b += square_of(bf16_high(x.w));
    }
    return a + b;
}

// scale^2, or NaN for a scale that no encoding has (NaN, Inf, zero, negative):
// such a tensor makes the norm NaN, which raises the flag.
__device__ __forceinline__ double scale_square(float scale) {
    if (!(scale > 0.0f) || is_non_finite(scale)) return __longlong_as_double(0x7ff8000000000000ll);
    return square_of(scale);
}

// Number of the block that value `start + i` is in, for i of a chunk: one 64-bit
// division a chunk, and a shift or a 32-bit one a value.
struct BlockIndex {
    long long first;                    // block of value `start`
    unsigned offset, block;             // start's place in it, block size (0: one block)
    int shift;                          // block = 1 << shift, or < 0

    __device__ __forceinline__ BlockIndex(long long start, int block_size, bool one_block) {
        block = one_block ? 0u : static_cast<unsigned>(block_size);
        first = one_block ? 0 : start / block_size;
        offset = one_block ? 0u : static_cast<unsigned>(start - first * block_size);
        shift = one_block || (block & (block - 1u)) != 0 ? -1 : 31 - __clz(static_cast<int>(block));
    }
    __device__ __forceinline__ long long at(int i) const {
        if (block == 0) return 0;
        const unsigned place = offset + static_cast<unsigned>(i);
        return first + (shift >= 0 ? place >> shift : place / block);
    }
};

__device__ __forceinline__ int word_squares(const uint4& w) {
    int sum = __dp4a(static_cast<int>(w.x), static_cast<int>(w.x), 0);
    sum = __dp4a(static_cast<int>(w.y), static_cast<int>(w.y), sum);
    sum = __dp4a(static_cast<int>(w.z), static_cast<int>(w.z), sum);
    return __dp4a(static_cast<int>(w.w), static_cast<int>(w.w), sum);
}

// Codes [start, start + n) of a payload whose blocks of `block` values begin at
// its first value.  A 16-byte word lies inside one block when block % 16 == 0
// (or there is one block only) and the payload is 16-byte aligned; chunks start
// at multiples of 4096 values.  Other layouts go value by value.
__device__ double chunk_squares_bfp8(const signed char* payload, const float* scales, long long start, int n,
                                     int block_size, bool one_block) {
    const BlockIndex index(start, block_size, one_block);
    const bool vector_ok = (reinterpret_cast<std::uintptr_t>(payload) & 15u) == 0 && (one_block || block_size % 16 == 0);
    const int vectors = vector_ok ? n >> 4 : 0;
    const uint4* body = reinterpret_cast<const uint4*>(payload + start);
    double a = 0.0;
    for (int i = threadIdx.x; i < vectors; i += kUnroll * kThreads) {
        uint4 w[kUnroll];
        float scale[kUnroll];
        #pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int at = i + j * kThreads;
            w[j] = at < vectors ? __ldg(body + at) : make_uint4(0, 0, 0, 0);
            scale[j] = at < vectors ? __ldg(scales + index.at(at * 16)) : 1.0f;
        }
        #pragma unroll
        for (int j = 0; j < kUnroll; ++j) a += scale_square(scale[j]) * static_cast<double>(word_squares(w[j]));
    }
    for (int i = vectors * 16 + threadIdx.x; i < n; i += kThreads) {
        const int code = payload[start + i];
        a += scale_square(__ldg(scales + index.at(i))) * static_cast<double>(code * code);
    }
    return a;
}

__global__ void __launch_bounds__(kThreads)
tensor_list_squares_kernel(const nntrain_gradient_tensor* __restrict__ tensors, const Chunk* __restrict__ chunks,
                           int chunk_values, double* __restrict__ partials) {
    let_next_start();
    const Chunk chunk = chunks[blockIdx.x];
    const nntrain_gradient_tensor t = tensors[chunk.tensor];
    const long long values = kind_values(chunk_values, t.kind), start = chunk.index * values;
    const int n = static_cast<int>(t.length - start < values ? t.length - start : values);
    double squares;
    if (t.kind == kKindF32) {
        squares = chunk_squares_f32(static_cast<const float*>(t.values) + start, n);
    } else if (t.kind == kKindBf16) {
        squares = chunk_squares_bf16(static_cast<const unsigned short*>(t.values) + start, n);
    } else {
        const bool one_block = t.block_size == 0 || t.block_size >= t.length;
        squares = chunk_squares_bfp8(static_cast<const signed char*>(t.values), t.scales, start, n,
                                     t.block_size, one_block);
    }
    cta_store_partial(squares, partials);
}

// Sum of values[first, end): thread `at` of `step` takes every step-th one.
__device__ __forceinline__ double strided_sum(const double* values, long long first, long long end, int at, int step) {
    double sums[4] = {};
    long long i = first + at;
    for (; i + 3 * step < end; i += 4 * step) {
        #pragma unroll
        for (int j = 0; j < 4; ++j) sums[j] += values[i + j * step];
    }
    for (; i < end; i += step) sums[0] += values[i];
    return (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

constexpr int kSumLanes = 1024;         // lanes of the fixed summation order, whatever the CTA's size

// The sum of all partials, the same bits for every CTA size: virtual lane v of
// 1024 takes every 1024th, the lanes are summed by warps, the warps in order.
// To be called by all threads of a CTA of kCtaThreads; the result is valid in
// its first warp.
template <int kCtaThreads>
__device__ double sum_of_partials(const double* partials, long long chunks, double (&totals)[kSumLanes / 32]) {
    const int lane = threadIdx.x & 31;
    #pragma unroll
    for (int v = threadIdx.x; v < kSumLanes; v += kCtaThreads) {
        const double sum = warp_sum(strided_sum(partials, 0, chunks, v, kSumLanes));
        if (lane == 0) totals[v >> 5] = sum;
    }
    __syncthreads();
    return threadIdx.x < 32 ? warp_sum(totals[lane]) : 0.0;
}

struct NormResult { float norm, coefficient; };

__device__ __forceinline__ NormResult norm_result(double squares, float max_norm) {
    const float norm = static_cast<float>(sqrt(squares));
    const bool clip = !is_non_finite(norm) && norm > max_norm;
    return {norm, clip ? __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f)) : 1.0f};
}

__device__ __forceinline__ void store_result(NormResult r, float* norm_and_coefficient, int* finite_status) {
    norm_and_coefficient[0] = r.norm;
    norm_and_coefficient[1] = r.coefficient;
    if (finite_status != nullptr && is_non_finite(r.norm)) *finite_status = 1;
}

// The norm of tensor t by one warp; t may be beyond the list.
__device__ void store_tensor_norm(const nntrain_gradient_tensor* tensors, int count, long long chunks, int t,
                                  const double* partials, float* tensor_norms) {
    long long first = 0, end = 0;
    if (t < count) {
        first = tensors[t].first_chunk;
        end = t + 1 < count ? tensors[t + 1].first_chunk : chunks;
    }
    wait_for_previous();
    let_next_start();
    const int lane = threadIdx.x & 31;
    const double squares = warp_sum(strided_sum(partials, first, end, lane, 32));
    if (t < count && lane == 0) tensor_norms[t] = static_cast<float>(sqrt(squares));
}

// CTA 0 sums all partials and leaves norm and coefficient; the others, there
// when tensor_norms is asked for, take a tensor per warp.
__global__ void __launch_bounds__(kFinishThreads)
tensor_list_finish_kernel(const nntrain_gradient_tensor* __restrict__ tensors, int count, long long chunks,
                          const double* partials, float max_norm, float* norm_and_coefficient, float* tensor_norms,
                          int* finite_status) {
    __shared__ double totals[kSumLanes / 32];
    if (blockIdx.x > 0) {
        const int t = (blockIdx.x - 1) * (kFinishThreads / 32) + (threadIdx.x >> 5);
        store_tensor_norm(tensors, count, chunks, t, partials, tensor_norms);
        return;
    }
    wait_for_previous();
    let_next_start();
    const double squares = sum_of_partials<kFinishThreads>(partials, chunks, totals);
    if (threadIdx.x == 0) store_result(norm_result(squares, max_norm), norm_and_coefficient, finite_status);
}

// ---- clip ---------------------------------------------------------------------

template <int kKind>
__device__ __forceinline__ uint4 scaled(uint4 v, float c) {
    if constexpr (kKind == kKindF32) {
        return make_uint4(__float_as_uint(__fmul_rn(__uint_as_float(v.x), c)), __float_as_uint(__fmul_rn(__uint_as_float(v.y), c)),
                          __float_as_uint(__fmul_rn(__uint_as_float(v.z), c)), __float_as_uint(__fmul_rn(__uint_as_float(v.w), c)));
    } else {
        return make_uint4(pack_bf16(__fmul_rn(bf16_low(v.x), c), __fmul_rn(bf16_high(v.x), c)),
                          pack_bf16(__fmul_rn(bf16_low(v.y), c), __fmul_rn(bf16_high(v.y), c)),
                          pack_bf16(__fmul_rn(bf16_low(v.z), c), __fmul_rn(bf16_high(v.z), c)),
                          pack_bf16(__fmul_rn(bf16_low(v.w), c), __fmul_rn(bf16_high(v.w), c)));
    }
}

// The 16 bytes that start `shift` bytes into the 32 bytes a, b.
__device__ __forceinline__ uint4 shifted(uint4 a, uint4 b, int shift) {
    const int words = shift >> 2, bits = (shift & 3) * 8;
    unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (words & 2) {
        #pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (words & 1) {
        #pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// destination[start, start + n) = source[start, start + n) * c; c == 1 copies
// the bits.  Stores are whole 16-byte words of the destination.  Where the
// source lies differently to the 16-byte grid (a leaf gathered to its
// running-sum offset in an arena), a word is put together from the two source
// words around it; the second is the neighbouring thread's first, so it comes
// from L1.  Words next to the ends of the tensor, whose source words would
// reach outside of it, go value by value.
template <int kKind, typename T>
__device__ void clip_chunk(const T* source, T* destination, long long length, long long start, int n, float c) {
    constexpr int kBytes = sizeof(T), kPerWord = 16 / kBytes;
    const T* from = source + start;
    T* to = destination + start;
    const int head = head_values(to, kBytes, n), words = (n - head) / kPerWord, tail = head + words * kPerWord;
    const bool copy = c == 1.0f;
    auto one = [&](int i) {
        if (copy) {
            to[i] = from[i];
        } else if constexpr (kKind == kKindF32) {
            to[i] = __fmul_rn(from[i], c);
        } else {
            to[i] = bf16_bits(__fmul_rn(bf16_value(from[i]), c));
        }
    };
    if (static_cast<int>(threadIdx.x) < head) one(threadIdx.x);
    if (tail + static_cast<int>(threadIdx.x) < n) one(tail + threadIdx.x);
    uint4* out = reinterpret_cast<uint4*>(to + head);
    const int shift = static_cast<int>(reinterpret_cast<std::uintptr_t>(from + head) & 15u);
    if (shift == 0) {
        const uint4* in = reinterpret_cast<const uint4*>(from + head);
        for (int i = threadIdx.x; i < words; i += kUnroll * kThreads) {
            uint4 v[kUnroll];
            #pragma unroll
            for (int j = 0; j < kUnroll; ++j)
                if (i + j * kThreads < words) v[j] = __ldcs(in + i + j * kThreads);
            #pragma unroll
            for (int j = 0; j < kUnroll; ++j)
                if (i + j * kThreads < words) __stcs(out + i + j * kThreads, copy ? v[j] : scaled<kKind>(v[j], c));
        }
        return;
    }
    const uint4* in = reinterpret_cast<const uint4*>(reinterpret_cast<std::uintptr_t>(from + head) - shift);
    const uint4* first = reinterpret_cast<const uint4*>(source);
    const uint4* last = reinterpret_cast<const uint4*>(source + length);
    auto inside = [&](int i) {
        return reinterpret_cast<std::uintptr_t>(in + i) >= reinterpret_cast<std::uintptr_t>(first) &&
               reinterpret_cast<std::uintptr_t>(in + i + 2) <= reinterpret_cast<std::uintptr_t>(last);
    };
    for (int i = threadIdx.x; i < words; i += kShiftedUnroll * kThreads) {
        uint4 a[kShiftedUnroll], b[kShiftedUnroll];
        #pragma unroll
        for (int j = 0; j < kShiftedUnroll; ++j) {
            const int w = i + j * kThreads;
            if (w < words && inside(w)) {
                a[j] = __ldg(in + w);
                b[j] = __ldg(in + w + 1);
            }
        }
        #pragma unroll
        for (int j = 0; j < kShiftedUnroll; ++j) {
            const int w = i + j * kThreads;
            if (w >= words) continue;
            if (inside(w)) {
                const uint4 v = shifted(a[j], b[j], shift);
                __stcs(out + w, copy ? v : scaled<kKind>(v, c));
            } else {
                for (int k = 0; k < kPerWord; ++k) one(head + w * kPerWord + k);
            }
        }
    }
}

struct ClipArguments {
    const nntrain_gradient_tensor* tensors;
    const Chunk* chunks;
    const double* partials;
    float* norm_and_coefficient;
    float* tensor_norms;
    int* finite_status;
    float max_norm;
    int count, chunk_count, chunk_values;
};

// kFinish: norm and coefficient are not there yet; every CTA forms them from
// the partials (the same bits in each), CTA 0 stores them, and CTAs behind the
// chunks store the tensor norms.
template <bool kFinish>
__global__ void __launch_bounds__(kThreads)
tensor_list_clip_kernel(ClipArguments a) {
    if (kFinish && static_cast<int>(blockIdx.x) >= a.chunk_count) {
        const int t = (blockIdx.x - a.chunk_count) * kWarpsPerCta + (threadIdx.x >> 5);
        store_tensor_norm(a.tensors, a.count, a.chunk_count, t, a.partials, a.tensor_norms);
        return;
    }
    // from the back: what the squares pass read last is read first
    const Chunk chunk = a.chunks[a.chunk_count - 1 - blockIdx.x];
    const nntrain_gradient_tensor t = a.tensors[chunk.tensor];
    const long long values = kind_values(a.chunk_values, t.kind), start = chunk.index * values;
    const int n = static_cast<int>(t.length - start < values ? t.length - start : values);
    wait_for_previous();
    float c;
    if constexpr (kFinish) {
        __shared__ double totals[kSumLanes / 32];
        __shared__ float coefficient;
        const double squares = sum_of_partials<kThreads>(a.partials, a.chunk_count, totals);
        if (threadIdx.x == 0) {
            const NormResult r = norm_result(squares, a.max_norm);
            coefficient = r.coefficient;
            if (blockIdx.x == 0) store_result(r, a.norm_and_coefficient, a.finite_status);
        }
        __syncthreads();
        c = coefficient;
    } else {
        c = a.norm_and_coefficient[1];
    }
    if (t.kind == kKindBfp8) {
        // scale' = max(scale * c, FLT_MIN), payload untouched: the blocks whose
        // first value is in this chunk
        float* out = t.destination != nullptr ? static_cast<float*>(t.destination) : t.scales;
        if (c == 1.0f && out == t.scales) return;
        const long long block = t.block_size == 0 || t.block_size >= t.length ? t.length : t.block_size;
        const long long first = (start + block - 1) / block, end = (start + n - 1) / block + 1;
        for (long long b = first + threadIdx.x; b < end; b += kThreads)
            out[b] = c == 1.0f ? t.scales[b] : fmaxf(__fmul_rn(t.scales[b], c), FLT_MIN);
        return;
    }
    void* out = t.destination != nullptr ? t.destination : const_cast<void*>(t.values);
    if (c == 1.0f && out == t.values) return;
    if (t.kind == kKindF32)
        clip_chunk<kKindF32>(static_cast<const float*>(t.values), static_cast<float*>(out), t.length, start, n, c);
    else
        clip_chunk<kKindBf16>(static_cast<const unsigned short*>(t.values), static_cast<unsigned short*>(out), t.length, start, n, c);
}

bool valid_tensor(const nntrain_gradient_tensor& t) {
    if (t.length < 0 || t.block_size < 0 || t.kind < kKindF32 || t.kind > kKindBfp8) return false;
    if (t.length == 0) return true;
    if (t.values == nullptr || (t.kind == kKindBfp8 && t.scales == nullptr)) return false;
    const std::uintptr_t bytes = t.kind == kKindF32 ? 4 : (t.kind == kKindBf16 ? 2 : 1);
    return aligned_for(t.values, bytes) && aligned_for(t.scales, 4) &&
           aligned_for(t.destination, t.kind == kKindBfp8 ? 4 : bytes);
}

struct Range {
    std::uintptr_t begin, end;
    int tensor;
    bool source;                        // read: what its own tensor's clip is made from
};

// Whether what the clip writes for one tensor is read or written for another
// one (the same tensor twice, a destination over a neighbour): chunks run in any
// order, so such a list has no defined result.  In place a tensor's values, or a
// payload's scales, are read and written at one place by one thread; scales are
// never written over a payload, which may be just as long.
bool overlapping(const nntrain_gradient_tensor* tensors, int count) {
    std::vector<Range> written, read;
    for (int i = 0; i < count; ++i) {
        const nntrain_gradient_tensor& t = tensors[i];
        if (t.length == 0) continue;
        const auto range = [&](const void* p, long long bytes, bool source) {
            const std::uintptr_t at = reinterpret_cast<std::uintptr_t>(p);
            return Range{at, at + static_cast<std::uintptr_t>(bytes), i, source};
        };
        if (t.kind == kKindBfp8) {
            const long long blocks = t.block_size == 0 || t.block_size >= t.length ? 1 : (t.length + t.block_size - 1) / t.block_size;
            read.push_back(range(t.values, t.length, false));
            read.push_back(range(t.scales, blocks * 4, true));
            written.push_back(range(t.destination != nullptr ? t.destination : t.scales, blocks * 4, false));
        } else {
            const long long bytes = t.length * (t.kind == kKindF32 ? 4 : 2);
            read.push_back(range(t.values, bytes, true));
            written.push_back(range(t.destination != nullptr ? t.destination : t.values, bytes, false));
        }
    }
    const auto by_begin = [](const Range& a, const Range& b) { return a.begin < b.begin; };
    std::sort(written.begin(), written.end(), by_begin);
    for (size_t i = 1; i < written.size(); ++i)
        if (written[i].begin < written[i - 1].end) return true;
    for (const Range& r : read) {
        // written ranges are apart: those that meet r are next to where it begins
        auto w = std::upper_bound(written.begin(), written.end(), r, by_begin);
        if (w != written.begin()) --w;
        for (; w != written.end() && w->begin < r.end; ++w) {
            const bool itself = r.source && w->tensor == r.tensor && w->begin == r.begin && w->end == r.end;
            if (w->end > r.begin && !itself) return true;
        }
    }
    return false;
}

int plan_list(nntrain_gradient_tensor* tensors, int count, int* chunk_map, long long capacity,
              long long* chunk_count, int* chunk_values) {
    if (!tensors || count <= 0 || !chunk_count || !chunk_values || capacity < 0)
        return static_cast<int>(cudaErrorInvalidValue);
    long long total = 0;                // in fp32 values
    for (int i = 0; i < count; ++i) {
        if (!valid_tensor(tensors[i]) || tensors[i].length > (1ll << 46) - total) return static_cast<int>(cudaErrorInvalidValue);
        total += tensors[i].length >> tensors[i].kind;
    }
    if (chunk_map == nullptr && overlapping(tensors, count)) return static_cast<int>(cudaErrorInvalidValue);
    long long size = (total / 2048 + kChunkLeast - 1) / kChunkLeast * kChunkLeast;
    size = size < kChunkLeast ? kChunkLeast : (size > kChunkMost ? kChunkMost : size);
    long long chunks = 0;
    for (int i = 0; i < count; ++i) {
        tensors[i].first_chunk = chunks;
        const long long values = kind_values(static_cast<int>(size), tensors[i].kind);
        const long long here = (tensors[i].length + values - 1) / values;
        if (chunk_map != nullptr) {
            if (chunks + here > capacity) return static_cast<int>(cudaErrorInvalidValue);
            for (long long k = 0; k < here; ++k) {
                chunk_map[2 * (chunks + k)] = i;
                chunk_map[2 * (chunks + k) + 1] = static_cast<int>(k);
            }
        }
        chunks += here;
    }
    if (chunks > 2147483647ll) return static_cast<int>(cudaErrorInvalidValue);
    *chunk_count = chunks;
    *chunk_values = static_cast<int>(size);
    return static_cast<int>(cudaSuccess);
}

int clip_list(int device, const nntrain_gradient_tensor* tensors, int count, const int* chunk_map,
              long long chunk_count, int chunk_values, double* workspace, float max_norm, int apply,
              float* norm_and_coefficient, float* tensor_norms, int* finite_status, cudaStream_t stream) {
    if (!tensors || count <= 0 || chunk_count < 0 || chunk_count > 2147483647ll || chunk_values < kChunkLeast ||
        chunk_values > kChunkMost || chunk_values % kChunkLeast != 0 || !norm_and_coefficient || !(max_norm > 0.0f) ||
        (chunk_count > 0 && (!chunk_map || !workspace)) || !aligned_for(chunk_map, 8) || !aligned_for(workspace, 8))
        return static_cast<int>(cudaErrorInvalidValue);
    const DeviceScope scope(device);
    if (scope.status() != cudaSuccess) return scope.status();
    const Chunk* chunks = reinterpret_cast<const Chunk*>(chunk_map);
    const int grid = static_cast<int>(chunk_count);
    cudaError_t e = cudaSuccess;
    if (grid > 0) e = launch(tensor_list_squares_kernel, dim3(grid), kThreads, 0, stream, tensors, chunks, chunk_values, workspace);
    if (e != cudaSuccess) return static_cast<int>(e);
    const ClipArguments a{tensors, chunks, workspace, norm_and_coefficient, tensor_norms, finite_status, max_norm, count,
                          grid, chunk_values};
    if (apply && grid > 0 && grid <= kFusedFinishChunks)
        return static_cast<int>(launch_dependent(tensor_list_clip_kernel<true>,
                                                 grid + (tensor_norms ? (count + kWarpsPerCta - 1) / kWarpsPerCta : 0),
                                                 kThreads, 0, stream, a));
    constexpr int kFinishWarps = kFinishThreads / 32;
    e = launch_dependent(tensor_list_finish_kernel, 1 + (tensor_norms ? (count + kFinishWarps - 1) / kFinishWarps : 0),
                         kFinishThreads, 0, stream, tensors, count, chunk_count, workspace, max_norm,
                         norm_and_coefficient, tensor_norms, finite_status);
    if (e == cudaSuccess && apply && grid > 0)
        e = launch_dependent(tensor_list_clip_kernel<false>, grid, kThreads, 0, stream, a);
    return static_cast<int>(e);
}

}  // namespace
}  // namespace ngb

using namespace ngb;

NNTRAIN_EXPORT int nntrain_gradient_list_plan(nntrain_gradient_tensor* tensors, int count, int* chunk_map,
                                              long long capacity, long long* chunk_count, int* chunk_values) {
    int status;
    try {
        status = plan_list(tensors, count, chunk_map, capacity, chunk_count, chunk_values);
    } catch (...) {                      // the ranges are sorted in host memory
        status = static_cast<int>(cudaErrorMemoryAllocation);
    }
    return complete(kOpTensorList, -1, status);
}

NNTRAIN_EXPORT int nntrain_gradient_list_clip(int device, const nntrain_gradient_tensor* tensors, int count,
                                              const int* chunk_map, long long chunk_count, int chunk_values,
                                              double* workspace, float max_norm, int apply,
                                              float* norm_and_coefficient, float* tensor_norms, int* finite_status,
                                              nntrain_stream_t stream) {
    return complete(kOpTensorList, device,
                    clip_list(device, tensors, count, chunk_map, chunk_count, chunk_values, workspace, max_norm, apply,
                              norm_and_coefficient, tensor_norms, finite_status, static_cast<cudaStream_t>(stream)));
}
