// Root-mean-square norm of x + residual with its output in the codec's 8 bits,
// and its gradient (ABI minor 36).
//
//   h = x + residual,  i = 1 / sqrt(mean(h^2) + epsilon),  y = h * i * w
//   scale = max|y| / 127 over a block (1 for a block of zeros),
//   code  = clamp(rne(y / scale), +-127)
//
//   g = dy * w,  n = h * i,  dx = i * (g - n * mean(g * n)) + dh,  dw = sum over rows of dy * n
//
// The encode is the codec's (NNtrain.Core/Tensors/Bfp8Quantization.cs:188-274,
// NNtrain.Cuda/native/cuda_runtime_bridge.cu:138-232) applied to y in
// registers: y is not written in 16 or 32 bits to be read again by an encode
// launch.  All arithmetic is fp32; h, y and dx are rounded once, when they are
// stored.  The sum of squares uses the unrounded h.
//
// Layout: the threads of a CTA hold one row in registers, groups of 8
// consecutive values (one 128-bit load of bf16, two of fp32) or single values
// where the row does not lie on 16-byte boundaries (odd widths); the grid is
// one resident wave and a CTA walks rows, so the weight is loaded once and the
// weight's gradient stays in registers until the end.  Rows too long for
// registers are read again for each pass (they are in L1 / L2 then).
//
// Bound.  Backward: HBM, 8 bytes a value of bf16 with residual; 32768 x 1536 in
// 65 us, 59 of them at 6.8 TB/s and the rest the join of the weight gradient.
// Forward: 7.1 bytes a value (x, residual, h, payload, scales; 2 more for a
// decoded copy), but before that the instructions of the encode: 16384 x 1536
// with the copy in 41 us, 75 % of the issue slots used, 86 % of HBM's rate;
// y alone, without an encode, in 38 us.  Narrow rows, one warp to a row, wait for
// their two reductions instead: 2^20 x 128 bf16 without a residual 198 us forward
// (2.7 TB/s) and 719 us backward, and half as wide ones take as long.
#include "bfp8_kernels.cuh"
#include "operator_launch.cuh"

#include "nntrain_grad_abi.h"

#include <atomic>

namespace ngb {
namespace {

constexpr int kRowThreads = 512;              // most threads on a row held in registers
constexpr int kStagedThreads = 256;           // and on one that is staged in shared memory
constexpr int kLoopThreads = 256;             // threads on a row that is not
constexpr int kMostPartials = 1184;           // most CTAs that leave a partial weight gradient: 8 on each of 148 SMs
constexpr int kJoinColumns = 8, kJoinRows = 64;   // 32 bytes of a partial, a sector

struct RowSum {
    float (*slots)[kRowThreads / 32];
    int turn;
};

template <bool kMaximum>
__device__ __forceinline__ float combine(float a, float b) {
    return kMaximum ? fmaxf(a, b) : __fadd_rn(a, b);
}

// Sum / maximum of values that are not negative (or any sum) over the CTA, the
// same value in every thread.  Two sets of slots take turns, so one barrier per
// reduction is enough: a set is written again only behind the barrier of the
// other one.
template <bool kMaximum>
__device__ __forceinline__ float over_cta(float v, RowSum& s) {
    #pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) v = combine<kMaximum>(v, __shfl_xor_sync(0xffffffffu, v, offset));
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    float* slots = s.slots[s.turn];
    s.turn ^= 1;
    const int lane = threadIdx.x & 31;
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    // every warp adds the (at most 16) warps' values: a load and four shuffles
    v = (lane & 15) < warps ? slots[lane & 15] : 0.0f;
    #pragma unroll
    for (int offset = 8; offset > 0; offset >>= 1) v = combine<kMaximum>(v, __shfl_xor_sync(0xffffffffu, v, offset));
    return v;
}

// ---- loads and stores of a group -------------------------------------------------

// A group as it lies in memory, so that the next row's can be on its way while
// this row is worked on.
template <typename T, int kVec>
struct Raw {
    T value;
};
template <typename T>
struct Raw<T, 8> {
    uint4 words[sizeof(T) / 2];
};

template <typename T, int kVec>
__device__ __forceinline__ void load_raw(const T* p, Raw<T, kVec>& raw) {
    if constexpr (kVec == 1) {
        raw.value = *p;
    } else {
        #pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) raw.words[i] = reinterpret_cast<const uint4*>(p)[i];
    }
}

template <typename T, int kVec>
__device__ __forceinline__ void unpack(const Raw<T, kVec>& raw, float (&v)[kVec]) {
    if constexpr (kVec == 1) {
        if constexpr (sizeof(T) == 4) v[0] = raw.value;
        else v[0] = bf16_value(raw.value);
    } else {
        #pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
            const uint4 w = raw.words[i];
            if constexpr (sizeof(T) == 4) {
                v[4 * i] = __uint_as_float(w.x); v[4 * i + 1] = __uint_as_float(w.y);
                v[4 * i + 2] = __uint_as_float(w.z); v[4 * i + 3] = __uint_as_float(w.w);
            } else {
                v[0] = bf16_low(w.x); v[1] = bf16_high(w.x); v[2] = bf16_low(w.y); v[3] = bf16_high(w.y);
                v[4] = bf16_low(w.z); v[5] = bf16_high(w.z); v[6] = bf16_low(w.w); v[7] = bf16_high(w.w);
            }
        }
    }
}

// First column of the thread's group g: a warp has 32 * kGroups neighbouring
// groups, so the groups of a thread are a constant distance apart.
template <int kVec, int kGroups>
__device__ __forceinline__ int column_of(int g) {
    return ((static_cast<int>(threadIdx.x) & ~31) * kGroups + g * 32 + (static_cast<int>(threadIdx.x) & 31)) * kVec;
}

// A row's groups of this thread; columns beyond the width are left alone.
template <typename T, int kVec, int kGroups>
__device__ __forceinline__ void load_row(const void* base, long long row, long long stride, int width, Raw<T, kVec> (&raw)[kGroups]) {
    const T* p = static_cast<const T*>(base) + row * stride;
    #pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        if (column_of<kVec, kGroups>(g) < width) load_raw<T, kVec>(p + column_of<kVec, kGroups>(0) + g * 32 * kVec, raw[g]);
    }
}

// Rows on their way, in shared memory: every thread copies the groups that it
// will read itself (cp.async, 16 bytes each) kStages - 1 rows ahead, so loads
// cost no registers and a thread waits for its own copies only.  No stages for
// rows with more than two 16-byte words a thread and input: those have enough
// loads in flight by themselves.
template <typename T, int kVec, int kGroups>
__host__ __device__ constexpr int row_stages() {
    constexpr int kWords = kGroups * static_cast<int>(sizeof(T)) / 2;
    return kVec == 1 || kWords > 2 ? 0 : (kWords == 1 ? 3 : 2);
}

__device__ __forceinline__ void copy_async16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void close_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kOpen>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(kOpen) : "memory"); }

template <typename T, int kVec, int kGroups, int kInputs>
struct RowRing {
    static constexpr int kStages = row_stages<T, kVec, kGroups>();
    static constexpr int kWords = static_cast<int>(sizeof(T)) / 2;      // 16-byte words of a group
    static constexpr int kThreadBytes = kStages * kInputs * kGroups * kWords * 16;

    uint4* words;                      // [stage][input][group][word][thread]

    __device__ __forceinline__ uint4* at(int stage, int input, int group, int word) const {
        return words + (((stage * kInputs + input) * kGroups + group) * kWords + word) * static_cast<int>(blockDim.x) + threadIdx.x;
    }
    __device__ __forceinline__ void copy(int stage, int input, const void* base, long long row, long long stride, int width) const {
        const T* p = static_cast<const T*>(base) + row * stride + column_of<kVec, kGroups>(0);
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (column_of<kVec, kGroups>(g) >= width) continue;
            #pragma unroll
            for (int w = 0; w < kWords; ++w) copy_async16(at(stage, input, g, w), reinterpret_cast<const uint4*>(p + g * 32 * kVec) + w);
        }
    }
    __device__ __forceinline__ void read(int stage, int input, Raw<T, kVec> (&raw)[kGroups]) const {
        if constexpr (kVec == 8) {
            #pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                #pragma unroll
                for (int w = 0; w < kWords; ++w) raw[g].words[w] = *at(stage, input, g, w);
            }
        }
    }
};

template <typename T>
__device__ __forceinline__ float load_value(const T* p) {
    if constexpr (sizeof(T) == 4) return *p;
    else return bf16_value(*p);
}

template <int kVec>
__device__ __forceinline__ void store_group(float* p, const float (&v)[kVec]) {
    if constexpr (kVec == 1) {
        *p = v[0];
    } else {
        store_f4(p, make_float4(v[0], v[1], v[2], v[3]));
        store_f4(p + 4, make_float4(v[4], v[5], v[6], v[7]));
    }
}
template <int kVec>
__device__ __forceinline__ void store_group(unsigned short* p, const float (&v)[kVec]) {
    if constexpr (kVec == 1) {
        *p = bf16_bits(v[0]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]),
                                                  pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
}
__device__ __forceinline__ float load_weight(const void* weight, int kind, long long i) {
    return kind == 0 ? static_cast<const float*>(weight)[i] : bf16_value(static_cast<const unsigned short*>(weight)[i]);
}

// The weight's group at `column`: 128-bit loads where the weight lies on 16 bytes
// (it is a view of a parameter arena and need not).
template <int kVec>
__device__ __forceinline__ void load_weights(const void* weight, int kind, bool aligned, int column, float (&w)[kVec]) {
    if constexpr (kVec == 8) {
        if (aligned) {
            if (kind == 0) {
                Raw<float, 8> raw;
                load_raw<float, 8>(static_cast<const float*>(weight) + column, raw);
                unpack<float, 8>(raw, w);
            } else {
                Raw<unsigned short, 8> raw;
                load_raw<unsigned short, 8>(static_cast<const unsigned short*>(weight) + column, raw);
                unpack<unsigned short, 8>(raw, w);
            }
            return;
        }
    }
    #pragma unroll
    for (int i = 0; i < kVec; ++i) w[i] = load_weight(weight, kind, column + i);
}

// Whether a thread keeps its weights in registers from row to row; with more of
// them they would spill, and come from L1 for each row instead.
template <int kVec, int kGroups>
__host__ __device__ constexpr bool keeps_weights() { return kVec * kGroups <= 16; }

// ---- forward ------------------------------------------------------------------

struct ForwardArguments {
    const void* x;
    const void* residual;              // null: h = x
    const void* weight;
    void* residual_out;                // null: h is not stored
    void* y;                           // null, or y (no payload) / the decode of the payload
    signed char* payload;              // null: not encoded
    float* scales;
    float* inverse_rms;                // null: not stored
    int* finite_status;                // null: not raised
    long long rows, x_stride, residual_stride;
    int width, block, weight_kind, y_kind;
    bool weight_aligned;
    float epsilon, reciprocal_width;
};

// 1 / sqrt(squares / width + epsilon).  The mean is a product with fl(1/width)
// and the root the hardware's estimate (relative error below 2^-22) after one
// Newton step, v + v/2 (1 - x v^2): three halves of a rounding off, and a few
// instructions where the correctly rounded operations take some thirty, in every
// warp of every row.
__device__ __forceinline__ float inverse_of(float squares, float reciprocal_width, float epsilon, bool& bad) {
    const float mean = __fmul_rn(squares, reciprocal_width);
    const float x = __fadd_rn(mean, epsilon);
    const float v = rsqrtf(x);
    // for x of 0 or infinity the estimate is the answer, and the step would make it NaN
    const float refined = __fmaf_rn(__fmul_rn(0.5f, v), __fmaf_rn(-__fmul_rn(x, v), v, 1.0f), v);
    const float inverse = x > 0.0f && !is_non_finite(x) ? refined : v;
    bad |= is_non_finite(mean) || is_non_finite(inverse);
    return inverse;
}

template <int kVec>
__device__ __forceinline__ void store_y(void* y, int kind, long long at, const float (&v)[kVec]) {
    if (kind == 0) store_group<kVec>(static_cast<float*>(y) + at, v);
    else store_group<kVec>(static_cast<unsigned short*>(y) + at, v);
}

// Codes of a group against its block's scale: payload, and the values that the
// codes stand for.
template <int kVec>
__device__ __forceinline__ void encode_group(float (&y)[kVec], float scale, signed char* payload) {
    const BlockScale divisor = block_scale(scale);
    if constexpr (kVec == 1) {
        const float t = biased_code_of(y[0], divisor);
        *payload = code_byte(t);
        y[0] = __fmul_rn(code_value(t), scale);
    } else {
        float t[8];
        biased_codes_of(make_float4(y[0], y[1], y[2], y[3]), divisor, t[0], t[1], t[2], t[3]);
        biased_codes_of(make_float4(y[4], y[5], y[6], y[7]), divisor, t[4], t[5], t[6], t[7]);
        *reinterpret_cast<uint2*>(payload) = make_uint2(pack_codes(t[0], t[1], t[2], t[3]), pack_codes(t[4], t[5], t[6], t[7]));
        #pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(code_value(t[i]), scale);
    }
}

// kBlock: -1 = no encode, 0 = one scale a row, else the block size; a block is
// kBlock / kVec neighbouring lanes of a warp.
template <typename T, int kVec, int kGroups, int kBlock>
__global__ void __launch_bounds__(kRowThreads)
rms_norm_forward_kernel(ForwardArguments a) {
    __shared__ float slots[2][kRowThreads / 32];
    RowSum sums{slots, 0};
    constexpr bool kKeep = keeps_weights<kVec, kGroups>();
    float kept[kKeep ? kGroups : 1][kVec] = {};
    if (kKeep) {
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int column = column_of<kVec, kGroups>(g);
            if (column < a.width) load_weights<kVec>(a.weight, a.weight_kind, a.weight_aligned, column, kept[kKeep ? g : 0]);
        }
    }
    extern __shared__ uint4 ring_words[];
    using Ring = RowRing<T, kVec, kGroups, 2>;
    const Ring ring{ring_words};
    constexpr int kStages = Ring::kStages;
    Raw<T, kVec> x[kGroups], r[kGroups];
    auto copy = [&](long long row, int stage) {
        if (row < a.rows) {
            ring.copy(stage, 0, a.x, row, a.x_stride, a.width);
            if (a.residual != nullptr) ring.copy(stage, 1, a.residual, row, a.residual_stride, a.width);
        }
        close_copies();                          // an empty one too: the waits count them
    };
    // A y that is not finite has an h that is not (the mean shows it), a weight
    // that is not (checked here, once) or overflows (its block's maximum shows
    // it); where there is no maximum every y is looked at: y * 0 is 0 or NaN.
    constexpr bool kCheckValues = kBlock < 0 || !kKeep;
    bool bad = false;
    float not_finite = 0.0f;
    if (kKeep) {
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            #pragma unroll
            for (int i = 0; i < kVec; ++i) bad |= is_non_finite(kept[kKeep ? g : 0][i]);
        }
    }
    int stage = 0;
    if constexpr (kStages > 0) {
        #pragma unroll
        for (int s = 0; s < kStages - 1; ++s) copy(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
    }
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long base = row * a.width;
        float h[kGroups][kVec];
        if constexpr (kStages > 0) {
            copy(row + static_cast<long long>(kStages - 1) * gridDim.x, stage == 0 ? kStages - 1 : stage - 1);
            wait_copies<kStages - 1>();
            ring.read(stage, 0, x);
            if (a.residual != nullptr) ring.read(stage, 1, r);
            stage = stage == kStages - 1 ? 0 : stage + 1;
        } else {
            load_row<T, kVec, kGroups>(a.x, row, a.x_stride, a.width, x);
            if (a.residual != nullptr) load_row<T, kVec, kGroups>(a.residual, row, a.residual_stride, a.width, r);
        }
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int column = column_of<kVec, kGroups>(g);
            #pragma unroll
            for (int i = 0; i < kVec; ++i) h[g][i] = 0.0f;
            if (column >= a.width) continue;
            unpack<T, kVec>(x[g], h[g]);
            if (a.residual != nullptr) {
                float v[kVec];
                unpack<T, kVec>(r[g], v);
                #pragma unroll
                for (int i = 0; i < kVec; ++i) h[g][i] = __fadd_rn(h[g][i], v[i]);
            }
        }
        float squares = 0.0f;
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int column = column_of<kVec, kGroups>(g);
            if (a.residual_out != nullptr && column < a.width)
                store_group<kVec>(static_cast<T*>(a.residual_out) + base + column, h[g]);
            #pragma unroll
            for (int i = 0; i < kVec; ++i) squares = __fmaf_rn(h[g][i], h[g][i], squares);
        }
        const float inverse = inverse_of(over_cta<false>(squares, sums), a.reciprocal_width, a.epsilon, bad);
        if (a.inverse_rms != nullptr && threadIdx.x == 0) a.inverse_rms[row] = inverse;
        float largest = 0.0f;
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int column = column_of<kVec, kGroups>(g);
            float w[kVec] = {};
            if (!kKeep && column < a.width) load_weights<kVec>(a.weight, a.weight_kind, a.weight_aligned, column, w);
            #pragma unroll
            for (int i = 0; i < kVec; ++i) {
                h[g][i] = __fmul_rn(__fmul_rn(h[g][i], inverse), kKeep ? kept[kKeep ? g : 0][i] : w[i]);
                if (kCheckValues) not_finite = __fmaf_rn(h[g][i], 0.0f, not_finite);
                if (kBlock == 0) largest = fmaxf(largest, fabsf(h[g][i]));
            }
        }
        float row_scale = 1.0f;
        if constexpr (kBlock == 0) {
            largest = over_cta<true>(largest, sums);
            bad |= is_non_finite(largest);
            row_scale = scale_from_maximum_fast(largest);
            if (threadIdx.x == 0) a.scales[row] = row_scale;
        }
        if constexpr (kVec == 1 && kBlock == 0) {
            // single values of one block: codes of four at a time, as of a group
            const BlockScale divisor = block_scale(row_scale);
            #pragma unroll
            for (int g = 0; g < kGroups; g += 4) {
                float t[4];
                biased_codes_of(make_float4(h[g][0], h[g + 1][0], h[g + 2][0], h[g + 3][0]), divisor, t[0], t[1], t[2], t[3]);
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int column = column_of<1, kGroups>(g + i);
                    if (column < a.width) a.payload[base + column] = code_byte(t[i]);
                    h[g + i][0] = __fmul_rn(code_value(t[i]), row_scale);
                }
            }
        }
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int column = column_of<kVec, kGroups>(g);
            if constexpr (kBlock > 0) {
                constexpr int kLanes = kBlock / kVec;
                float maximum = 0.0f;
                #pragma unroll
                for (int i = 0; i < kVec; ++i) maximum = fmaxf(maximum, fabsf(h[g][i]));
                maximum = group_max<kLanes>(maximum);
                bad |= is_non_finite(maximum);
                const float scale = scale_from_maximum_fast(maximum);
                if (column < a.width) {
                    if (threadIdx.x % kLanes == 0) a.scales[(base + column) / kBlock] = scale;
                    encode_group<kVec>(h[g], scale, a.payload + base + column);
                }
            } else if constexpr (kBlock == 0 && kVec == 8) {
                if (column < a.width) encode_group<kVec>(h[g], row_scale, a.payload + base + column);
            }
            if (a.y != nullptr && column < a.width) store_y<kVec>(a.y, a.y_kind, base + column, h[g]);
        }
    }
    bad |= !(not_finite == 0.0f);
    if (a.finite_status != nullptr && __any_sync(0xffffffffu, bad) && (threadIdx.x & 31) == 0)
        atomicExch(a.finite_status, 1);
}

// Any width, any block size that divides it, any alignment: the row is read
// once for its sum of squares, (one scale a row: once more for its maximum,)
// and then block by block, a warp to a block, for the maximum and the codes.
// h may be stored over x or the residual, so it is stored by the last pass,
// by the thread that reads the value there.
template <typename T>
__global__ void __launch_bounds__(kLoopThreads)
rms_norm_forward_loop_kernel(ForwardArguments a) {
    __shared__ float slots[2][kRowThreads / 32];
    RowSum sums{slots, 0};
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kLoopThreads / 32;
    bool bad = false;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* residual = a.residual == nullptr ? nullptr : static_cast<const T*>(a.residual) + row * a.residual_stride;
        const long long base = row * a.width;
        auto h_at = [&](int i) {
            const float v = load_value(x + i);
            return residual != nullptr ? __fadd_rn(v, load_value(residual + i)) : v;
        };
        float squares = 0.0f;
        for (int i = threadIdx.x; i < a.width; i += kLoopThreads) {
            const float h = h_at(i);
            squares = __fmaf_rn(h, h, squares);
        }
        const float inverse = inverse_of(over_cta<false>(squares, sums), a.reciprocal_width, a.epsilon, bad);
        if (a.inverse_rms != nullptr && threadIdx.x == 0) a.inverse_rms[row] = inverse;
        auto y_of = [&](float h, int i) {
            return __fmul_rn(__fmul_rn(h, inverse), load_weight(a.weight, a.weight_kind, i));
        };
        auto finish = [&](int i, float scale) {
            float h[1] = {h_at(i)};
            float y[1] = {y_of(h[0], i)};
            bad |= is_non_finite(y[0]);
            if (a.payload != nullptr) encode_group<1>(y, scale, a.payload + base + i);
            if (a.residual_out != nullptr) store_group<1>(static_cast<T*>(a.residual_out) + base + i, h);
            if (a.y != nullptr) store_y<1>(a.y, a.y_kind, base + i, y);
        };
        if (a.payload == nullptr || a.block == a.width) {
            float scale = 1.0f;
            if (a.payload != nullptr) {
                float largest = 0.0f;
                for (int i = threadIdx.x; i < a.width; i += kLoopThreads) largest = fmaxf(largest, fabsf(y_of(h_at(i), i)));
                scale = scale_from_maximum_fast(over_cta<true>(largest, sums));
                if (threadIdx.x == 0) a.scales[row] = scale;
            }
            for (int i = threadIdx.x; i < a.width; i += kLoopThreads) finish(i, scale);
            continue;
        }
        const int blocks = a.width / a.block;
        for (int b = warp; b < blocks; b += warps) {
            float largest = 0.0f;
            for (int i = b * a.block + lane; i < (b + 1) * a.block; i += 32) largest = fmaxf(largest, fabsf(y_of(h_at(i), i)));
            const float scale = scale_from_maximum_fast(group_max<32>(largest));
            if (lane == 0) a.scales[row * blocks + b] = scale;
            for (int i = b * a.block + lane; i < (b + 1) * a.block; i += 32) finish(i, scale);
        }
    }
    if (a.finite_status != nullptr && __any_sync(0xffffffffu, bad) && lane == 0) atomicExch(a.finite_status, 1);
}

// ---- backward -----------------------------------------------------------------

struct BackwardArguments {
    const void* y_gradient;
    const void* residual_gradient;     // null: nothing is added to dx
    const void* h;
    const void* weight;
    const float* inverse_rms;
    void* x_gradient;
    float* partials;                   // [CTAs][width]
    long long rows, y_stride, residual_stride, h_stride;
    int width, weight_kind;
    bool weight_aligned;
    float reciprocal_width;
};

template <typename T, int kVec, int kGroups>
__global__ void __launch_bounds__(kRowThreads)
rms_norm_backward_kernel(BackwardArguments a) {
    __shared__ float slots[2][kRowThreads / 32];
    RowSum sums{slots, 0};
    let_next_start();
    constexpr bool kKeep = keeps_weights<kVec, kGroups>();
    float kept[kKeep ? kGroups : 1][kVec] = {}, dw[kGroups][kVec] = {};
    if (kKeep) {
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int column = column_of<kVec, kGroups>(g);
            if (column < a.width) load_weights<kVec>(a.weight, a.weight_kind, a.weight_aligned, column, kept[kKeep ? g : 0]);
        }
    }
    extern __shared__ uint4 ring_words[];
    using Ring = RowRing<T, kVec, kGroups, 3>;
    const Ring ring{ring_words};
    constexpr int kStages = Ring::kStages;
    Raw<T, kVec> dy[kGroups], h[kGroups];
    auto copy = [&](long long row, int stage) {
        if (row < a.rows) {
            ring.copy(stage, 0, a.y_gradient, row, a.y_stride, a.width);
            ring.copy(stage, 1, a.h, row, a.h_stride, a.width);
            if (a.residual_gradient != nullptr) ring.copy(stage, 2, a.residual_gradient, row, a.residual_stride, a.width);
        }
        close_copies();                          // an empty one too: the waits count them
    };
    int stage = 0;
    float inverse_ahead = blockIdx.x < a.rows ? a.inverse_rms[blockIdx.x] : 0.0f;
    if constexpr (kStages > 0) {
        #pragma unroll
        for (int s = 0; s < kStages - 1; ++s) copy(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
    }
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float inverse = inverse_ahead;
        if (row + gridDim.x < a.rows) inverse_ahead = a.inverse_rms[row + gridDim.x];
        if constexpr (kStages > 0) {
            copy(row + static_cast<long long>(kStages - 1) * gridDim.x, stage == 0 ? kStages - 1 : stage - 1);
            wait_copies<kStages - 1>();
            ring.read(stage, 0, dy);
            ring.read(stage, 1, h);
        } else {
            load_row<T, kVec, kGroups>(a.y_gradient, row, a.y_stride, a.width, dy);
            load_row<T, kVec, kGroups>(a.h, row, a.h_stride, a.width, h);
        }
        float d[kGroups][kVec], n[kGroups][kVec];
        float along = 0.0f;
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int column = column_of<kVec, kGroups>(g);
            #pragma unroll
            for (int i = 0; i < kVec; ++i) d[g][i] = n[g][i] = 0.0f;
            if (column < a.width) {
                unpack<T, kVec>(dy[g], d[g]);
                unpack<T, kVec>(h[g], n[g]);
            }
            float w[kVec] = {};
            if (!kKeep && column < a.width) load_weights<kVec>(a.weight, a.weight_kind, a.weight_aligned, column, w);
            #pragma unroll
            for (int i = 0; i < kVec; ++i) {
                n[g][i] = __fmul_rn(n[g][i], inverse);
                dw[g][i] = __fmaf_rn(d[g][i], n[g][i], dw[g][i]);
                d[g][i] = __fmul_rn(d[g][i], kKeep ? kept[kKeep ? g : 0][i] : w[i]);
                along = __fmaf_rn(d[g][i], n[g][i], along);
            }
        }
        const float mean = __fmul_rn(over_cta<false>(along, sums), a.reciprocal_width);
        Raw<T, kVec> added[kGroups];
        if constexpr (kStages > 0) {
            if (a.residual_gradient != nullptr) ring.read(stage, 2, added);
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        #pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int column = column_of<kVec, kGroups>(g);
            if (column >= a.width) continue;
            float v[kVec] = {};
            if (a.residual_gradient != nullptr) {
                if constexpr (kStages == 0)
                    load_raw<T, kVec>(static_cast<const T*>(a.residual_gradient) + row * a.residual_stride + column, added[g]);
                unpack<T, kVec>(added[g], v);
            }
            #pragma unroll
            for (int i = 0; i < kVec; ++i) d[g][i] = __fmaf_rn(inverse, __fmaf_rn(-n[g][i], mean, d[g][i]), v[i]);
            store_group<kVec>(static_cast<T*>(a.x_gradient) + row * a.width + column, d[g]);
        }
    }
    float* partial = a.partials + static_cast<long long>(blockIdx.x) * a.width;
    #pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int column = column_of<kVec, kGroups>(g);
        #pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (column < a.width) partial[column + i] = dw[g][i];
    }
}

// Any width and alignment: the row is read twice, the partial weight gradient
// is kept in memory; a thread always has the same columns.
template <typename T>
__global__ void __launch_bounds__(kLoopThreads)
rms_norm_backward_loop_kernel(BackwardArguments a) {
    __shared__ float slots[2][kRowThreads / 32];
    RowSum sums{slots, 0};
    float* partial = a.partials + static_cast<long long>(blockIdx.x) * a.width;
    for (int i = threadIdx.x; i < a.width; i += kLoopThreads) partial[i] = 0.0f;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* dy = static_cast<const T*>(a.y_gradient) + row * a.y_stride;
        const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
        const float inverse = a.inverse_rms[row];
        float along = 0.0f;
        for (int i = threadIdx.x; i < a.width; i += kLoopThreads) {
            const float d = load_value(dy + i), n = __fmul_rn(load_value(h + i), inverse);
            partial[i] = __fmaf_rn(d, n, partial[i]);
            along = __fmaf_rn(__fmul_rn(d, load_weight(a.weight, a.weight_kind, i)), n, along);
        }
        const float mean = __fmul_rn(over_cta<false>(along, sums), a.reciprocal_width);
        for (int i = threadIdx.x; i < a.width; i += kLoopThreads) {
            const float g = __fmul_rn(load_value(dy + i), load_weight(a.weight, a.weight_kind, i));
            const float n = __fmul_rn(load_value(h + i), inverse);
            const float r = a.residual_gradient == nullptr
                ? 0.0f : load_value(static_cast<const T*>(a.residual_gradient) + row * a.residual_stride + i);
            const float dx[1] = {__fmaf_rn(inverse, __fmaf_rn(-n, mean, g), r)};
            store_group<1>(static_cast<T*>(a.x_gradient) + row * a.width + i, dx);
        }
    }
}

// dw (+)= sum of the partials, in a fixed order: 64 threads share a column.
__global__ void __launch_bounds__(kJoinColumns * kJoinRows)
rms_norm_join_kernel(const float* partials, int count, int width, void* weight_gradient, int kind, bool accumulate) {
    __shared__ float sums[kJoinRows][kJoinColumns];
    const int x = threadIdx.x % kJoinColumns, y = threadIdx.x / kJoinColumns;
    const int column = blockIdx.x * kJoinColumns + x;
    wait_for_previous();
    float sum = 0.0f;
    if (column < width) {
        #pragma unroll 8
        for (int r = y; r < count; r += kJoinRows) sum = __fadd_rn(sum, partials[static_cast<long long>(r) * width + column]);
    }
    sums[y][x] = sum;
    for (int half = kJoinRows / 2; half > 0; half /= 2) {
        __syncthreads();
        if (y < half) sums[y][x] = __fadd_rn(sums[y][x], sums[y + half][x]);
    }
    if (y != 0 || column >= width) return;
    if (kind == 0) {
        float* out = static_cast<float*>(weight_gradient) + column;
        *out = accumulate ? __fadd_rn(*out, sums[0][x]) : sums[0][x];
    } else {
        unsigned short* out = static_cast<unsigned short*>(weight_gradient) + column;
        *out = bf16_bits(accumulate ? __fadd_rn(bf16_value(*out), sums[0][x]) : sums[0][x]);
    }
}

// ---- launch shapes ---------------------------------------------------------------

// One resident wave of kKernel with `threads` threads and the shared memory that
// goes with them.
template <auto kKernel>
int resident_grid(int threads, int shared, long long rows) {
    static std::atomic<int> known[kRowThreads / 32 + 1];
    std::atomic<int>& slot = known[threads / 32];
    int fit = slot.load(std::memory_order_relaxed);
    if (fit == 0) {
        if (reported(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kKernel, threads, shared)) != cudaSuccess || fit < 1)
            return grid_for(rows, 1);            // not kept: the next call asks again
        slot.store(fit, std::memory_order_relaxed);
    }
    return grid_for(rows, fit);
}

struct RowShape {
    int groups, threads;               // groups 0: the row does not fit registers
};

int threads_for(int units, int groups) { return ((units + groups - 1) / groups + 31) / 32 * 32; }

// Threads and groups per thread for a row of `units` groups of 8 values.  32
// bytes of an input a thread (two groups of bf16, one of fp32) where there are
// rows for all SMs, so that few warps share a row's barriers and its own
// arithmetic (16384 x 1536 bf16: 41 us with 96 threads, 43 us with 192, 58 us
// with 64; its gradient 65, 72 and 140 us for twice the rows), more where the row
// is longer than 256 threads then.
template <typename T>
RowShape row_shape(int units, long long rows) {
    const bool wide = sizeof(T) == 2 && units > 64 && rows >= sm_count();
    for (int groups = wide ? 2 : 1; groups <= 4; groups *= 2) {
        const int threads = threads_for(units, groups);
        if (threads <= kStagedThreads || (groups == 4 && threads <= kRowThreads)) return {groups, threads};
    }
    return {0, 0};
}

// A staged row's kStagedThreads threads have at most 48 KB in flight: with the
// reduction's slots a little more than a launch may ask for by itself.  The limit
// belongs to the kernel on the device, not to a launch, so it is always set to the
// most that the kernel can ask for: set to each launch's own size, it made the
// launches of another host thread with a wider row fail.
template <auto kKernel, int kThreadBytes>
cudaError_t allow_shared() {
    constexpr int kMost = kStagedThreads * kThreadBytes;
    if constexpr (kMost < (40 << 10)) return cudaSuccess;
    else return reported(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
}

template <typename T, int kVec, int kGroups, int kBlock>
cudaError_t launch_forward(const ForwardArguments& a, int threads, cudaStream_t stream) {
    constexpr auto kKernel = rms_norm_forward_kernel<T, kVec, kGroups, kBlock>;
    constexpr int kThreadBytes = RowRing<T, kVec, kGroups, 2>::kThreadBytes;
    static_assert(kThreadBytes == 0 || kGroups < 4, "four groups a thread may have kRowThreads threads");
    const int shared = threads * kThreadBytes;
    const cudaError_t e = allow_shared<kKernel, kThreadBytes>();
    if (e != cudaSuccess) return e;
    return launch(kKernel, dim3(resident_grid<kKernel>(threads, shared, a.rows)), threads, shared, stream, a);
}

template <typename T, int kVec, int kGroups>
cudaError_t forward_by_block(const ForwardArguments& a, int threads, cudaStream_t stream) {
    if (a.payload == nullptr) return launch_forward<T, kVec, kGroups, -1>(a, threads, stream);
    if (a.block == a.width) return launch_forward<T, kVec, kGroups, 0>(a, threads, stream);
    if (a.block == 32) return launch_forward<T, kVec, kGroups, 32>(a, threads, stream);
    if constexpr (kVec == 8) {
        if (a.block == 64) return launch_forward<T, kVec, kGroups, 64>(a, threads, stream);
        return launch_forward<T, kVec, kGroups, 128>(a, threads, stream);
    }
    return cudaErrorInvalidValue;
}

// Rows in registers: blocks of 32, 64, 128 or the row on the 16-byte grid up to
// 16384 values, blocks of 32 or the row off it up to 8192.  All else goes value by
// value through memory: other blocks that divide the width, 64 and 128 off the grid,
// longer rows.  It is right for all of them and several times slower (16384 x 1536
// bf16 with residual: block 32 on the grid 38 us, off it 134 us; in the loop block 96
// 162 us, 256 140 us, 64 off the grid 176 us; 2048 x 16384 in registers 55 us, 2048 x
// 16416 in the loop 123 us).
template <typename T>
cudaError_t run_forward(const ForwardArguments& a, bool vector_ok, cudaStream_t stream) {
    const bool whole = a.payload == nullptr || a.block == a.width;
    if (vector_ok && (whole || a.block == 32 || a.block == 64 || a.block == 128)) {
        const RowShape s = row_shape<T>(a.width / 8, a.rows);
        if (s.groups == 1) return forward_by_block<T, 8, 1>(a, s.threads, stream);
        if (s.groups == 2) return forward_by_block<T, 8, 2>(a, s.threads, stream);
        if (s.groups == 4) return forward_by_block<T, 8, 4>(a, s.threads, stream);
    } else if (whole || a.block == 32) {
        // 16 values a thread past one warp's: the barriers and the row's own arithmetic are shared by fewer warps
        // (771 fp32, one scale a row: 3001 rows 11.7 us with 4 values, 10.3 us with 16, 10001 rows 32 and 26.5 us)
        if (a.width <= 512) return forward_by_block<T, 1, 4>(a, threads_for(a.width, 4), stream);
        if (a.width <= 16 * kRowThreads) return forward_by_block<T, 1, 16>(a, threads_for(a.width, 16), stream);
    }
    constexpr auto kKernel = rms_norm_forward_loop_kernel<T>;
    return launch(kKernel, dim3(resident_grid<kKernel>(kLoopThreads, 0, a.rows)), kLoopThreads, 0, stream, a);
}

template <typename T, int kVec, int kGroups>
cudaError_t launch_backward(const BackwardArguments& a, int threads, int& grid, cudaStream_t stream) {
    constexpr auto kKernel = rms_norm_backward_kernel<T, kVec, kGroups>;
    constexpr int kThreadBytes = RowRing<T, kVec, kGroups, 3>::kThreadBytes;
    static_assert(kThreadBytes == 0 || kGroups < 4, "four groups a thread may have kRowThreads threads");
    const int shared = threads * kThreadBytes;
    const cudaError_t e = allow_shared<kKernel, kThreadBytes>();
    if (e != cudaSuccess) return e;
    grid = resident_grid<kKernel>(threads, shared, a.rows);
    if (grid > kMostPartials) grid = kMostPartials;
    return launch(kKernel, dim3(grid), threads, shared, stream, a);
}

template <typename T>
cudaError_t run_backward(const BackwardArguments& a, bool vector_ok, int& grid, cudaStream_t stream) {
    if (vector_ok) {
        const RowShape s = row_shape<T>(a.width / 8, a.rows);
        if (s.groups == 1) return launch_backward<T, 8, 1>(a, s.threads, grid, stream);
        if (s.groups == 2) return launch_backward<T, 8, 2>(a, s.threads, grid, stream);
        if (s.groups == 4) return launch_backward<T, 8, 4>(a, s.threads, grid, stream);
    } else {
        if (a.width <= 4 * kRowThreads) return launch_backward<T, 1, 4>(a, threads_for(a.width, 4), grid, stream);
        if (a.width <= 16 * kRowThreads) return launch_backward<T, 1, 16>(a, threads_for(a.width, 16), grid, stream);
    }
    constexpr auto kKernel = rms_norm_backward_loop_kernel<T>;
    grid = resident_grid<kKernel>(kLoopThreads, 0, a.rows);
    if (grid > kMostPartials) grid = kMostPartials;
    return launch(kKernel, dim3(grid), kLoopThreads, 0, stream, a);
}

// Rows of `kind` at `p`, `stride` values apart: 128-bit accesses possible?
bool rows_aligned(const void* p, int kind, long long stride) {
    return aligned_for(p, 16) && stride * (kind == 0 ? 4 : 2) % 16 == 0;
}
bool typed(const void* p, int kind) { return aligned_for(p, kind == 0 ? 4 : 2); }
bool is_kind(int kind) { return kind == 0 || kind == 1; }

constexpr long long kMostRows = 1ll << 40;
constexpr int kMostWidth = 1 << 24;
long long partial_count(long long rows) { return rows < kMostPartials ? rows : kMostPartials; }

int forward(int device, int kind, const void* x, long long x_stride, const void* residual, long long residual_stride,
            const void* weight, int weight_kind, long long rows, int width, float epsilon, void* residual_out, void* y,
            int y_kind, signed char* payload, float* scales, int block_size, float* inverse_rms, int* finite_status,
            cudaStream_t stream) {
    if (!is_kind(kind) || !is_kind(weight_kind) || !is_kind(y_kind) || rows < 0 || rows > kMostRows || width < 1 ||
        width > kMostWidth || block_size < 0 || !(epsilon >= 0.0f) || std::isinf(epsilon) || x_stride < width ||
        (residual && residual_stride < width))
        return static_cast<int>(cudaErrorInvalidValue);
    const int block = block_size == 0 || block_size > width ? width : block_size;
    if (!weight || (rows > 0 && !y && !payload) || (payload && (!scales || width % block != 0)) || (residual_out && !residual) ||
        (rows > 0 && !x) || !typed(x, kind) || !typed(residual, kind) || !typed(weight, weight_kind) ||
        !typed(residual_out, kind) || !typed(y, y_kind) || !aligned_for(scales, 4) || !aligned_for(inverse_rms, 4) ||
        !aligned_for(finite_status, 4))
        return static_cast<int>(cudaErrorInvalidValue);
    if (rows == 0) return static_cast<int>(cudaSuccess);
    const DeviceScope scope(device);
    if (scope.status() != cudaSuccess) return scope.status();
    const ForwardArguments a{x, residual, weight, residual_out, y, payload, scales, inverse_rms, finite_status,
                             rows, x_stride, residual_stride, width, block, weight_kind, y_kind, aligned_for(weight, 16), epsilon, 1.0f / static_cast<float>(width)};
    const bool vector_ok = width % 8 == 0 && rows_aligned(x, kind, x_stride) &&
                           (!residual || rows_aligned(residual, kind, residual_stride)) &&
                           aligned_for(residual_out, 16) && aligned_for(y, 16) && aligned_for(payload, 8);
    return static_cast<int>(kind == 0 ? run_forward<float>(a, vector_ok, stream)
                                      : run_forward<unsigned short>(a, vector_ok, stream));
}

int backward(int device, int kind, const void* y_gradient, long long y_stride, const void* residual_gradient,
             long long residual_stride, const void* h, long long h_stride, const void* weight, int weight_kind,
             const float* inverse_rms, long long rows, int width, void* x_gradient, void* weight_gradient,
             int weight_gradient_kind, int accumulate, void* workspace, long long workspace_bytes, cudaStream_t stream) {
    if (!is_kind(kind) || !is_kind(weight_kind) || !is_kind(weight_gradient_kind) || rows < 0 || rows > kMostRows ||
        width < 1 || width > kMostWidth || y_stride < width || h_stride < width ||
        (residual_gradient && residual_stride < width))
        return static_cast<int>(cudaErrorInvalidValue);
    if (!weight || !weight_gradient || (rows > 0 && (!y_gradient || !h || !inverse_rms || !x_gradient || !workspace)) ||
        !typed(y_gradient, kind) || !typed(residual_gradient, kind) || !typed(h, kind) || !typed(x_gradient, kind) ||
        !typed(weight, weight_kind) || !typed(weight_gradient, weight_gradient_kind) || !aligned_for(inverse_rms, 4) ||
        !aligned_for(workspace, 4) || workspace_bytes < partial_count(rows) * width * 4)
        return static_cast<int>(cudaErrorInvalidValue);
    const DeviceScope scope(device);
    if (scope.status() != cudaSuccess) return scope.status();
    int grid = 0;
    cudaError_t e = cudaSuccess;
    if (rows > 0) {
        const BackwardArguments a{y_gradient, residual_gradient, h, weight, inverse_rms, x_gradient,
                                  static_cast<float*>(workspace), rows, y_stride, residual_stride, h_stride, width, weight_kind, aligned_for(weight, 16), 1.0f / static_cast<float>(width)};
        const bool vector_ok = width % 8 == 0 && rows_aligned(y_gradient, kind, y_stride) && rows_aligned(h, kind, h_stride) &&
                               (!residual_gradient || rows_aligned(residual_gradient, kind, residual_stride)) &&
                               aligned_for(x_gradient, 16);
        e = kind == 0 ? run_backward<float>(a, vector_ok, grid, stream) : run_backward<unsigned short>(a, vector_ok, grid, stream);
    }
    if (e == cudaSuccess)
        e = launch_dependent(rms_norm_join_kernel, (width + kJoinColumns - 1) / kJoinColumns, kJoinColumns * kJoinRows, 0,
                             stream, static_cast<const float*>(workspace), grid, width, weight_gradient,
                             weight_gradient_kind, accumulate != 0);
    return static_cast<int>(e);
}

}  // namespace
}  // namespace ngb

using namespace ngb;

NNTRAIN_EXPORT int nntrain_rms_norm_forward(
    int device, int kind, const void* x, long long x_stride, const void* residual, long long residual_stride,
    const void* weight, int weight_kind, long long rows, int width, float epsilon, void* residual_out, void* y, int y_kind,
    signed char* payload, float* scales, int block_size, float* inverse_rms, int* finite_status, nntrain_stream_t stream) {
    return complete(kOpRmsNorm, device,
                    forward(device, kind, x, x_stride, residual, residual_stride, weight, weight_kind, rows, width, epsilon,
                            residual_out, y, y_kind, payload, scales, block_size, inverse_rms, finite_status,
                            static_cast<cudaStream_t>(stream)));
}

NNTRAIN_EXPORT int nntrain_rms_norm_backward_workspace(long long rows, int width, long long* bytes) {
    if (rows < 0 || rows > kMostRows || width < 1 || width > kMostWidth || !bytes)
        return complete(kOpRmsNorm, -1, static_cast<int>(cudaErrorInvalidValue));
    *bytes = partial_count(rows) * width * 4;
    return static_cast<int>(cudaSuccess);
}

NNTRAIN_EXPORT int nntrain_rms_norm_backward(
    int device, int kind, const void* y_gradient, long long y_stride, const void* residual_gradient,
    long long residual_stride, const void* h, long long h_stride, const void* weight, int weight_kind,
    const float* inverse_rms, long long rows, int width, void* x_gradient, void* weight_gradient, int weight_gradient_kind,
    int accumulate, void* workspace, long long workspace_bytes, nntrain_stream_t stream) {
    return complete(kOpRmsNorm, device,
                    backward(device, kind, y_gradient, y_stride, residual_gradient, residual_stride, h, h_stride, weight,
                             weight_kind, inverse_rms, rows, width, x_gradient, weight_gradient, weight_gradient_kind,
                             accumulate, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)));
}
