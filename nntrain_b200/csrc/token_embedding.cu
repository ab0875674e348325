// Rows of a token table, and the table's gradient (ABI minor 36).
//
//   out[t]  = scale * T[token_t]            T in fp32, bf16 or BFP8
//   dT[v]   = scale * sum over t with token_t = v of dout[t]   (+ dT[v])
//
// The table is the largest tensor of the published parameters and its gradient
// the largest of the arena.  The lookup decodes the rows it needs from the
// encoded table (code * scale_b, the codec's multiply, then the scale); no
// decoded copy of the table exists.
//
// The gradient is a sum over equal tokens.  Atomics on the table would add in
// another order every time, so the tokens are sorted (stable) and every row is
// summed in the order in which its tokens occur, the same bits every time:
//
//   sort    one cluster of 8 CTAs: a stable radix sort of (token, position),
//           9 bits a pass, digit counts exchanged through distributed shared
//           memory, the cluster's barriers between the passes; no grid-wide wait
//   rows    a warp takes 32 sorted positions x 256 columns and walks them; a
//           token that lies inside the 32 is finished, of one that crosses the
//           border a partial sum goes to scratch.  Further CTAs write the zeros
//           of the rows no token names (not when adding to what is there)
//   join    a CTA per crossing token adds its partials in order
//
// so a token that is half of the batch is summed by as many warps as its
// positions are long, and one that occurs once costs one row read and written.
// Sums are fp32, multiplied by the scale and rounded once.
//
// Bound: HBM.  dout is read once, the table's gradient written once (adding:
// the named rows read and written).
#include "operator_launch.cuh"

#include "nntrain_grad_abi.h"

#include <cooperative_groups.h>

namespace ngb {
namespace {

namespace cg = cooperative_groups;

enum TableKind : int { kTableF32 = 0, kTableBf16 = 1, kTableBfp8 = 2 };

struct Tokens {
    const void* values;
    int bytes;                         // 4 or 8
    long long padding;                 // no token: a row of zeros, no gradient
    long long vocab;

    // The token at i, or -1 for none; `bad` when it is neither a row nor padding.
    __device__ __forceinline__ long long at(long long i, bool& bad) const {
        const long long token = bytes == 8 ? __ldg(static_cast<const long long*>(values) + i)
                                           : static_cast<long long>(__ldg(static_cast<const int*>(values) + i));
        if (token == padding) return -1;
        if (token < 0 || token >= vocab) {
            bad = true;
            return -1;
        }
        return token;
    }
};

// ---- lookup -------------------------------------------------------------------

struct LookupArguments {
    Tokens tokens;
    const void* table;
    const float* scales;
    void* out;
    int* status;
    long long count, out_stride, first_value, block;
    int width, slices, block_shift;    // block_shift < 0: block is not a power of two; block 0: one scale
    float scale;
};

constexpr int kLookupGroups = 2;       // groups of 8 values per lane: a warp covers 512 columns

__device__ __forceinline__ float table_scale(const LookupArguments& a, long long value) {
    if (a.block == 0) return __ldg(a.scales);
    const long long at = a.first_value + value;
    return __ldg(a.scales + (a.block_shift >= 0 ? at >> a.block_shift : at / a.block));
}

// One warp: one token's row, 512 columns of it.  kVector: 8 neighbouring values
// per lane and access (of BFP8: in one block); otherwise single values.
template <int kTable, typename T, bool kVector>
__global__ void __launch_bounds__(kThreads)
embedding_lookup_kernel(LookupArguments a) {
    const int lane = threadIdx.x & 31;
    const long long task = static_cast<long long>(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5);
    const long long position = task / a.slices;
    if (position >= a.count) return;
    const int first = static_cast<int>(task - position * a.slices) * (kLookupGroups * 256);
    bool bad = false;
    const long long token = a.tokens.at(position, bad);
    if (bad && a.status != nullptr && lane == 0) atomicExch(a.status, 1);
    T* out = static_cast<T*>(a.out) + position * a.out_stride;
    const long long row = token * a.width;
    if constexpr (kVector) {
        float v[kLookupGroups][8] = {};
        #pragma unroll
        for (int g = 0; g < kLookupGroups; ++g) {
            const int column = first + (g * 32 + lane) * 8;
            if (column >= a.width || token < 0) continue;
            if constexpr (kTable == kTableF32) {
                const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.table) + row + column);
                const float4 x = __ldg(p), y = __ldg(p + 1);
                v[g][0] = x.x; v[g][1] = x.y; v[g][2] = x.z; v[g][3] = x.w;
                v[g][4] = y.x; v[g][5] = y.y; v[g][6] = y.z; v[g][7] = y.w;
            } else if constexpr (kTable == kTableBf16) {
                const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(a.table) + row + column));
                v[g][0] = bf16_low(x.x); v[g][1] = bf16_high(x.x); v[g][2] = bf16_low(x.y); v[g][3] = bf16_high(x.y);
                v[g][4] = bf16_low(x.z); v[g][5] = bf16_high(x.z); v[g][6] = bf16_low(x.w); v[g][7] = bf16_high(x.w);
            } else {
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(static_cast<const signed char*>(a.table) + row + column));
                const float s = table_scale(a, row + column);
                const unsigned low = x.x ^ 0x80808080u, high = x.y ^ 0x80808080u;
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[g][i] = __fmul_rn(byte_to_float(low, i), s);
                    v[g][4 + i] = __fmul_rn(byte_to_float(high, i), s);
                }
            }
        }
        #pragma unroll
        for (int g = 0; g < kLookupGroups; ++g) {
            const int column = first + (g * 32 + lane) * 8;
            if (column >= a.width) continue;
            // zeros times an infinite scale would be NaN: a row of no token is not multiplied
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[g][i] = token < 0 ? 0.0f : __fmul_rn(v[g][i], a.scale);
            if constexpr (sizeof(T) == 4) {
                store_f4(reinterpret_cast<float*>(out) + column, make_float4(v[g][0], v[g][1], v[g][2], v[g][3]));
                store_f4(reinterpret_cast<float*>(out) + column + 4, make_float4(v[g][4], v[g][5], v[g][6], v[g][7]));
            } else {
                *reinterpret_cast<uint4*>(out + column) = make_uint4(pack_bf16(v[g][0], v[g][1]), pack_bf16(v[g][2], v[g][3]),
                                                                     pack_bf16(v[g][4], v[g][5]), pack_bf16(v[g][6], v[g][7]));
            }
        }
    } else {
        #pragma unroll 4
        for (int i = 0; i < kLookupGroups * 8; ++i) {
            const int column = first + i * 32 + lane;
            if (column >= a.width) break;
            float v = 0.0f;
            if (token >= 0) {
                if constexpr (kTable == kTableF32) v = __ldg(static_cast<const float*>(a.table) + row + column);
                else if constexpr (kTable == kTableBf16) v = bf16_value(__ldg(static_cast<const unsigned short*>(a.table) + row + column));
                else v = __fmul_rn(static_cast<float>(static_cast<const signed char*>(a.table)[row + column]), table_scale(a, row + column));
                v = __fmul_rn(v, a.scale);
            }
            if constexpr (sizeof(T) == 4) out[column] = v;
            else out[column] = bf16_bits(v);
        }
    }
}

// ---- sort ---------------------------------------------------------------------

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kSortCluster = 8;                 // CTAs (the portable cluster size)
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortShared = (kSortWarps * kDigits + 2 * kDigits + 32) * 4;

struct SortArguments {
    Tokens tokens;
    unsigned* keys[2];                 // passes take turns; the sorted order ends in [0]
    unsigned* positions[2];
    unsigned* touched;                 // one bit a row, null when not asked for
    unsigned* crossing;                // counter of the rows kernel, cleared here
    int* status;
    unsigned count;
    int passes, bits;                  // bits of a pass
};

// Stable: warps own consecutive stretches of the input, a warp walks its
// stretch 32 at a time, and equal digits keep the order of their lanes.  Keys
// are row numbers; positions without a token get the key `vocab`, behind all
// rows.
__global__ void __launch_bounds__(kSortThreads)
embedding_sort_kernel(SortArguments a) {
    extern __shared__ unsigned shared[];
    unsigned* counts = shared;                               // [warps][digits]
    unsigned* totals = shared + kSortWarps * kDigits;        // [digits], read by the whole cluster
    unsigned* starts = totals + kDigits;                     // [digits]
    unsigned* warp_sums = starts + kDigits;                  // [32]
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), ranks = cluster.num_blocks();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned before = (1u << lane) - 1u;
    const unsigned workers = ranks * kSortWarps;
    const unsigned stretch = ((a.count + workers - 1) / workers + 31u) & ~31u;
    const unsigned long long begin = static_cast<unsigned long long>(rank * kSortWarps + warp) * stretch;
    const unsigned first = begin < a.count ? static_cast<unsigned>(begin) : a.count;
    const unsigned last = begin + stretch < a.count ? static_cast<unsigned>(begin + stretch) : a.count;
    unsigned* mine = counts + warp * kDigits;

    if (a.touched != nullptr) {
        const unsigned words = static_cast<unsigned>((a.tokens.vocab + 31) / 32);
        for (unsigned i = rank * kSortThreads + threadIdx.x; i < words; i += ranks * kSortThreads) a.touched[i] = 0;
        cluster.sync();
    }
    if (rank == 0 && threadIdx.x == 0) *a.crossing = 0;
    bool bad = false;
    for (int pass = 0; pass < a.passes; ++pass) {
        const int out = (a.passes - 1 - pass) & 1, shift = pass * a.bits;
        const unsigned* in_keys = a.keys[out ^ 1];
        const unsigned* in_positions = a.positions[out ^ 1];
        auto key_at = [&](unsigned i) -> unsigned {
            if (pass > 0) return __ldcg(in_keys + i);
            const long long token = a.tokens.at(i, bad);
            return static_cast<unsigned>(token < 0 ? a.tokens.vocab : token);
        };
        const unsigned digit_mask = (1u << a.bits) - 1u;
        for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) counts[i] = 0;
        __syncthreads();
        for (unsigned base = first; base < last; base += 32) {
            const bool here = base + lane < last;
            const unsigned key = here ? key_at(base + lane) : 0;
            const unsigned digit = here ? (key >> shift) & digit_mask : 0xffffffffu;
            const unsigned same = __match_any_sync(0xffffffffu, digit);
            if (here && (same & before) == 0) mine[digit] += __popc(same);
            if (pass == 0 && here && a.touched != nullptr && key < static_cast<unsigned long long>(a.tokens.vocab))
                atomicOr(a.touched + (key >> 5), 1u << (key & 31u));
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x < kDigits) {
            unsigned sum = 0;
            for (int w = 0; w < kSortWarps; ++w) {
                const unsigned n = counts[w * kDigits + threadIdx.x];
                counts[w * kDigits + threadIdx.x] = sum;
                sum += n;
            }
            totals[threadIdx.x] = sum;
        }
        cluster.sync();
        // first place of this CTA's share of each digit
        unsigned below = 0, all = 0, inclusive = 0;
        if (threadIdx.x < kDigits) {
            for (unsigned r = 0; r < ranks; ++r) {
                const unsigned n = *cluster.map_shared_rank(totals + threadIdx.x, r);
                below += r < rank ? n : 0;
                all += n;
            }
            inclusive = all;
            #pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
                const unsigned n = __shfl_up_sync(0xffffffffu, inclusive, offset);
                inclusive += lane >= offset ? n : 0;
            }
            if (lane == 31) warp_sums[warp] = inclusive;
        }
        __syncthreads();
        if (threadIdx.x < kDigits) {
            for (int w = 0; w < warp; ++w) inclusive += warp_sums[w];
            starts[threadIdx.x] = inclusive - all + below;
        }
        __syncthreads();
        for (unsigned base = first; base < last; base += 32) {
            const bool here = base + lane < last;
            const unsigned key = here ? key_at(base + lane) : 0;
            const unsigned position = !here ? 0 : (pass > 0 ? __ldcg(in_positions + base + lane) : base + lane);
            const unsigned digit = here ? (key >> shift) & digit_mask : 0xffffffffu;
            const unsigned same = __match_any_sync(0xffffffffu, digit);
            if (here) {
                const unsigned place = starts[digit] + mine[digit] + __popc(same & before);
                if (place < a.count) {           // always, unless the tokens change while they are sorted
                    a.keys[out][place] = key;
                    a.positions[out][place] = position;
                }
            }
            __syncwarp();
            if (here && (same & before) == 0) mine[digit] += __popc(same);
            __syncwarp();
        }
        cluster.sync();
    }
    if (bad && a.status != nullptr) atomicExch(a.status, 1);
}

// ---- rows and join --------------------------------------------------------------

constexpr int kChunkPositions = 32;             // sorted positions of a warp
constexpr int kSliceColumns = 256;              // columns of a warp: 8 a lane
constexpr int kZeroRows = 32;                   // rows of a CTA that writes zeros: one word of the bitmap

struct RowsArguments {
    const unsigned* keys;
    const unsigned* positions;
    const unsigned* touched;
    unsigned* crossing;                // [0] count, then the chunks in which a crossing token begins
    float* tails;                      // [chunk][width]: sum up to the chunk's end of a token that goes on
    float* heads;                      // [chunk][width]: rest of a token that began in an earlier chunk
    const void* gradient;              // dout
    void* table;
    long long gradient_stride;
    unsigned count, vocab, chunks;
    int width, slices, row_ctas;
    float scale;
    bool accumulate;
};

// Column of the lane's i-th value: 8 neighbours, or every 32nd.
template <bool kVector>
__device__ __forceinline__ int lane_column(int first, int lane, int i) {
    return kVector ? first + lane * 8 + i : first + i * 32 + lane;
}

template <typename T>
__device__ __forceinline__ float value_of(T raw) {
    if constexpr (sizeof(T) == 4) return raw;
    else return bf16_value(raw);
}

// table[row] = scale * sum (+ what is there), rounded once.
template <typename T, bool kVector>
__device__ __forceinline__ void store_row(const RowsArguments& a, unsigned row, int first, int lane, const float (&sum)[8]) {
    T* out = static_cast<T*>(a.table) + static_cast<long long>(row) * a.width;
    float v[8];
    if constexpr (kVector) {
        const int column = lane_column<true>(first, lane, 0);
        if (column >= a.width) return;
        out += column;
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(sum[i], a.scale);
        if constexpr (sizeof(T) == 4) {
            if (a.accumulate) {
                const float4 x = load_f4(out), y = load_f4(out + 4);
                v[0] = __fmaf_rn(sum[0], a.scale, x.x); v[1] = __fmaf_rn(sum[1], a.scale, x.y);
                v[2] = __fmaf_rn(sum[2], a.scale, x.z); v[3] = __fmaf_rn(sum[3], a.scale, x.w);
                v[4] = __fmaf_rn(sum[4], a.scale, y.x); v[5] = __fmaf_rn(sum[5], a.scale, y.y);
                v[6] = __fmaf_rn(sum[6], a.scale, y.z); v[7] = __fmaf_rn(sum[7], a.scale, y.w);
            }
            store_f4(out, make_float4(v[0], v[1], v[2], v[3]));
            store_f4(out + 4, make_float4(v[4], v[5], v[6], v[7]));
        } else {
            if (a.accumulate) {
                const uint4 x = *reinterpret_cast<const uint4*>(out);
                v[0] = __fmaf_rn(sum[0], a.scale, bf16_low(x.x)); v[1] = __fmaf_rn(sum[1], a.scale, bf16_high(x.x));
                v[2] = __fmaf_rn(sum[2], a.scale, bf16_low(x.y)); v[3] = __fmaf_rn(sum[3], a.scale, bf16_high(x.y));
                v[4] = __fmaf_rn(sum[4], a.scale, bf16_low(x.z)); v[5] = __fmaf_rn(sum[5], a.scale, bf16_high(x.z));
                v[6] = __fmaf_rn(sum[6], a.scale, bf16_low(x.w)); v[7] = __fmaf_rn(sum[7], a.scale, bf16_high(x.w));
            }
            *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]),
                                                        pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        }
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int column = lane_column<false>(first, lane, i);
            if (column >= a.width) continue;
            const float x = a.accumulate ? __fmaf_rn(sum[i], a.scale, value_of(out[column])) : __fmul_rn(sum[i], a.scale);
            if constexpr (sizeof(T) == 4) out[column] = x;
            else out[column] = bf16_bits(x);
        }
    }
}

template <bool kVector>
__device__ __forceinline__ void store_partial(float* partials, unsigned chunk, int width, int first, int lane, const float (&sum)[8]) {
    float* out = partials + static_cast<long long>(chunk) * width;
    if constexpr (kVector) {
        const int column = lane_column<true>(first, lane, 0);
        if (column >= width) return;
        store_f4(out + column, make_float4(sum[0], sum[1], sum[2], sum[3]));
        store_f4(out + column + 4, make_float4(sum[4], sum[5], sum[6], sum[7]));
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int column = lane_column<false>(first, lane, i);
            if (column < width) out[column] = sum[i];
        }
    }
}

// The zeros of 32 rows, those that the bitmap does not name.
template <typename T>
__device__ void zero_rows(const RowsArguments& a, unsigned group) {
    const unsigned touched = a.touched[group];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = warp; r < kZeroRows; r += kWarpsPerCta) {
        const long long row = static_cast<long long>(group) * kZeroRows + r;
        if (row >= a.vocab || ((touched >> r) & 1u)) continue;
        T* out = static_cast<T*>(a.table) + row * a.width;
        constexpr int kPerWord = 16 / sizeof(T);
        int head = static_cast<int>((16u - (reinterpret_cast<std::uintptr_t>(out) & 15u)) & 15u) / static_cast<int>(sizeof(T));
        if (head > a.width) head = a.width;
        const int words = (a.width - head) / kPerWord, tail = head + words * kPerWord;
        if (lane < head) out[lane] = T(0);
        for (int i = lane; i < words; i += 32) reinterpret_cast<uint4*>(out + head)[i] = make_uint4(0, 0, 0, 0);
        if (tail + lane < a.width) out[tail + lane] = T(0);
    }
}

template <typename G, typename T, bool kVector>
__global__ void __launch_bounds__(kThreads)
embedding_rows_kernel(RowsArguments a) {
    wait_for_previous();
    let_next_start();
    if (static_cast<int>(blockIdx.x) >= a.row_ctas) {
        zero_rows<T>(a, blockIdx.x - a.row_ctas);
        return;
    }
    const int lane = threadIdx.x & 31;
    const unsigned task = blockIdx.x * kWarpsPerCta + (threadIdx.x >> 5);
    const unsigned chunk = task / a.slices;
    if (chunk >= a.chunks) return;
    const int first = static_cast<int>(task - chunk * a.slices) * kSliceColumns;
    const unsigned base = chunk * kChunkPositions;
    const unsigned key = base + lane < a.count ? a.keys[base + lane] : a.vocab;
    const unsigned position = base + lane < a.count ? a.positions[base + lane] : 0;
    const unsigned key_before = chunk > 0 ? a.keys[base - 1] : a.vocab;
    const unsigned key_behind = base + kChunkPositions < a.count ? a.keys[base + kChunkPositions] : a.vocab;
    const int n = __popc(__ballot_sync(0xffffffffu, key != a.vocab));    // rows come first
    constexpr int kBatch = sizeof(G) == 4 ? 4 : 8;                          // rows whose loads are in flight together
    const G* gradient = static_cast<const G*>(a.gradient);
    float sum[8] = {};
    bool begun_here = __shfl_sync(0xffffffffu, key, 0) != key_before;
    for (int j = 0; j < n; j += kBatch) {
        uint4 raw[kBatch][sizeof(G) / 2];
        G single[kBatch][8];
        #pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const unsigned at = __shfl_sync(0xffffffffu, position, (j + b) & 31);
            if (j + b >= n) continue;
            const G* row = gradient + static_cast<long long>(at) * a.gradient_stride;
            if constexpr (kVector) {
                const int column = lane_column<true>(first, lane, 0);
                #pragma unroll
                for (int h = 0; h < static_cast<int>(sizeof(G)) / 2; ++h)
                    raw[b][h] = column < a.width ? __ldcs(reinterpret_cast<const uint4*>(row + column) + h) : make_uint4(0, 0, 0, 0);
            } else {
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int column = lane_column<false>(first, lane, i);
                    single[b][i] = column < a.width ? __ldcs(row + column) : G(0);
                }
            }
        }
        #pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (j + b >= n) continue;
            const unsigned here = __shfl_sync(0xffffffffu, key, j + b);
            const unsigned next = j + b + 1 < kChunkPositions ? __shfl_sync(0xffffffffu, key, (j + b + 1) & 31) : key_behind;
            if constexpr (kVector) {
                if constexpr (sizeof(G) == 4) {
                    const uint4 x = raw[b][0], y = raw[b][1];
                    const float v[8] = {__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w),
                                        __uint_as_float(y.x), __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w)};
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) sum[i] = __fadd_rn(sum[i], v[i]);
                } else {
                    const uint4 x = raw[b][0];
                    const unsigned w[4] = {x.x, x.y, x.z, x.w};
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sum[2 * i] = __fadd_rn(sum[2 * i], bf16_low(w[i]));
                        sum[2 * i + 1] = __fadd_rn(sum[2 * i + 1], bf16_high(w[i]));
                    }
                }
            } else {
                #pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] = __fadd_rn(sum[i], value_of(single[b][i]));
            }
            if (next == here && j + b + 1 < kChunkPositions) continue;      // the token goes on in this chunk
            const bool goes_on = next == here;
            if (goes_on) {
                store_partial<kVector>(a.tails, chunk, a.width, first, lane, sum);
                if (begun_here && first == 0 && lane == 0) a.crossing[1 + atomicAdd(a.crossing, 1u)] = chunk;
            } else if (!begun_here) {
                store_partial<kVector>(a.heads, chunk, a.width, first, lane, sum);
            } else {
                store_row<T, kVector>(a, here, first, lane, sum);
            }
            begun_here = true;
            #pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
        }
    }
}

// The last chunk that holds `key`, which fills chunk `begin` to its end and
// goes on in the next one.  A warp looks at 32 chunk starts at a time: first at
// the next 32, then at 32 spread over what is left.
__device__ unsigned last_chunk_of(const RowsArguments& a, unsigned key, unsigned begin, int lane) {
    unsigned low = begin + 1, high = a.chunks;       // chunk `low` starts with the key, chunk `high` does not
    unsigned step = 1;
    while (high - low > 1) {
        const unsigned long long probe = low + static_cast<unsigned long long>(step) * (lane + 1);
        const bool holds = probe < high && a.keys[probe * kChunkPositions] == key;
        const unsigned held = __popc(__ballot_sync(0xffffffffu, holds));   // the first `held` probes hold it
        const unsigned long long beyond = low + static_cast<unsigned long long>(step) * (held + 1);
        low += step * held;
        if (beyond < high && held < 32) high = static_cast<unsigned>(beyond);
        step = (high - low + 31) / 32;
    }
    return low;
}

// A CTA per token that crosses chunks (and 256 columns): tails[begin], the
// tails of the chunks between, heads[end]; each of 8 warps adds an eighth of
// them in order, the eighths are added in order.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kThreads)
embedding_join_kernel(RowsArguments a) {
    __shared__ float sums[kWarpsPerCta][kSliceColumns];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    wait_for_previous();
    const unsigned tasks = a.crossing[0] * a.slices;
    for (unsigned task = blockIdx.x; task < tasks; task += gridDim.x) {
        const unsigned begin = a.crossing[1 + task / a.slices];
        const int first = static_cast<int>(task % a.slices) * kSliceColumns;
        const unsigned key = a.keys[begin * kChunkPositions + kChunkPositions - 1];
        const unsigned end = last_chunk_of(a, key, begin, lane);
        const unsigned parts = end - begin + 1, share = (parts + kWarpsPerCta - 1) / kWarpsPerCta;
        const unsigned from = warp * share, to = from + share < parts ? from + share : parts;
        float sum[8] = {};
        #pragma unroll 4
        for (unsigned p = from; p < to; ++p) {
            const float* partial = (begin + p == end ? a.heads : a.tails) + static_cast<long long>(begin + p) * a.width;
            if constexpr (kVector) {
                const int column = lane_column<true>(first, lane, 0);
                if (column < a.width) {
                    const float4 x = load_f4(partial + column), y = load_f4(partial + column + 4);
                    sum[0] = __fadd_rn(sum[0], x.x); sum[1] = __fadd_rn(sum[1], x.y);
                    sum[2] = __fadd_rn(sum[2], x.z); sum[3] = __fadd_rn(sum[3], x.w);
                    sum[4] = __fadd_rn(sum[4], y.x); sum[5] = __fadd_rn(sum[5], y.y);
                    sum[6] = __fadd_rn(sum[6], y.z); sum[7] = __fadd_rn(sum[7], y.w);
                }
            } else {
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int column = lane_column<false>(first, lane, i);
                    if (column < a.width) sum[i] = __fadd_rn(sum[i], partial[column]);
                }
            }
        }
        #pragma unroll
        for (int i = 0; i < 8; ++i) sums[warp][i * 32 + lane] = sum[i];
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < kWarpsPerCta; ++w) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] = __fadd_rn(sum[i], sums[w][i * 32 + lane]);
            }
            store_row<T, kVector>(a, key, first, lane, sum);
        }
        __syncthreads();
    }
}

// ---- entry points ----------------------------------------------------------------

constexpr long long kMostTokens = (1ll << 31) - 64, kMostVocab = 1ll << 31;
constexpr int kMostWidth = 1 << 24;

bool valid_sizes(long long count, long long vocab, int width) {
    return count >= 0 && count <= kMostTokens && vocab >= 1 && vocab <= kMostVocab && width >= 1 && width <= kMostWidth;
}

template <int kTable, typename T>
cudaError_t run_lookup(const LookupArguments& a, bool vector_ok, int grid, cudaStream_t stream) {
    if (vector_ok) embedding_lookup_kernel<kTable, T, true><<<grid, kThreads, 0, stream>>>(a);
    else embedding_lookup_kernel<kTable, T, false><<<grid, kThreads, 0, stream>>>(a);
    return cudaPeekAtLastError();
}

int lookup(int device, int table_kind, const void* table, const float* scales, int block_size, long long first_value,
           long long vocab, int width, const void* tokens, int token_bytes, long long count, long long padding_token,
           float scale, int out_kind, void* out, long long out_stride, int* token_status, cudaStream_t stream) {
    if (!valid_sizes(count, vocab, width) || table_kind < kTableF32 || table_kind > kTableBfp8 || out_kind < 0 || out_kind > 1 ||
        (token_bytes != 4 && token_bytes != 8) || out_stride < width || block_size < 0 || first_value < 0 || !table ||
        (table_kind == kTableBfp8 && !scales) || (count > 0 && (!tokens || !out)))
        return static_cast<int>(cudaErrorInvalidValue);
    const int table_bytes = table_kind == kTableF32 ? 4 : (table_kind == kTableBf16 ? 2 : 1), out_bytes = out_kind == 0 ? 4 : 2;
    if (!aligned_for(table, table_bytes) || !aligned_for(out, out_bytes) || !aligned_for(tokens, token_bytes) ||
        !aligned_for(scales, 4) || !aligned_for(token_status, 4))
        return static_cast<int>(cudaErrorInvalidValue);
    if (count == 0) return static_cast<int>(cudaSuccess);
    constexpr int kColumns = kLookupGroups * 256;
    const int slices = (width + kColumns - 1) / kColumns;
    const long long ctas = (count * slices + kWarpsPerCta - 1) / kWarpsPerCta;
    if (ctas > 2147483647ll) return static_cast<int>(cudaErrorInvalidValue);
    const DeviceScope scope(device);
    if (scope.status() != cudaSuccess) return scope.status();
    int shift = -1;
    if (block_size > 0 && (block_size & (block_size - 1)) == 0)
        for (shift = 0; (1 << shift) < block_size;) ++shift;
    const LookupArguments a{Tokens{tokens, token_bytes, padding_token, vocab}, table, scales, out, token_status, count,
                            out_stride, first_value, block_size, width, slices, shift, scale};
    const bool vector_ok = width % 8 == 0 && aligned_for(table, table_kind == kTableBfp8 ? 8 : 16) && aligned_for(out, 16) &&
                           out_stride * out_bytes % 16 == 0 &&
                           (table_kind != kTableBfp8 || block_size == 0 || (block_size % 8 == 0 && first_value % 8 == 0));
    const int grid = static_cast<int>(ctas);
    if (out_kind == 0) {
        if (table_kind == kTableF32) return static_cast<int>(run_lookup<kTableF32, float>(a, vector_ok, grid, stream));
        if (table_kind == kTableBf16) return static_cast<int>(run_lookup<kTableBf16, float>(a, vector_ok, grid, stream));
        return static_cast<int>(run_lookup<kTableBfp8, float>(a, vector_ok, grid, stream));
    }
    if (table_kind == kTableF32) return static_cast<int>(run_lookup<kTableF32, unsigned short>(a, vector_ok, grid, stream));
    if (table_kind == kTableBf16) return static_cast<int>(run_lookup<kTableBf16, unsigned short>(a, vector_ok, grid, stream));
    return static_cast<int>(run_lookup<kTableBfp8, unsigned short>(a, vector_ok, grid, stream));
}

// Scratch of one gradient call, every part on a 256-byte boundary.
struct GradientScratch {
    long long keys[2], positions[2], touched, crossing, tails, heads, bytes;
    long long chunks;
};

GradientScratch gradient_scratch(long long count, long long vocab, int width) {
    GradientScratch s{};
    auto take = [&](long long bytes) {
        const long long at = s.bytes;
        s.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    s.chunks = (count + kChunkPositions - 1) / kChunkPositions;
    for (int i = 0; i < 2; ++i) {
        s.keys[i] = take(count * 4);
        s.positions[i] = take(count * 4);
    }
    s.touched = take((vocab + 31) / 32 * 4);
    s.crossing = take((s.chunks + 1) * 4);
    s.tails = take(s.chunks * width * 4);
    s.heads = take(s.chunks * width * 4);
    return s;
}

cudaError_t launch_sort(const SortArguments& a, cudaStream_t stream) {
    // a dynamic-shared-memory limit belongs to the device's context; setting it costs a fraction of the launch
    cudaError_t e = cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortShared);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = kSortCluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(kSortCluster);
    config.blockDim = dim3(kSortThreads);
    config.dynamicSmemBytes = kSortShared;
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, embedding_sort_kernel, a);
}

template <typename G, typename T>
cudaError_t run_rows(const RowsArguments& a, bool vector_ok, int grid, cudaStream_t stream) {
    cudaError_t e = vector_ok ? launch_dependent(embedding_rows_kernel<G, T, true>, grid, kThreads, 0, stream, a)
                              : launch_dependent(embedding_rows_kernel<G, T, false>, grid, kThreads, 0, stream, a);
    if (e != cudaSuccess || a.chunks < 2) return e;
    const int join = grid_for(static_cast<long long>(a.chunks - 1) * a.slices, 4);
    return vector_ok ? launch_dependent(embedding_join_kernel<T, true>, join, kThreads, 0, stream, a)
                     : launch_dependent(embedding_join_kernel<T, false>, join, kThreads, 0, stream, a);
}

int gradient(int device, int gradient_kind, const void* out_gradient, long long gradient_stride, const void* tokens,
             int token_bytes, long long count, long long padding_token, float scale, int table_kind, void* table_gradient,
             long long vocab, int width, int accumulate, int* token_status, void* workspace, long long workspace_bytes,
             cudaStream_t stream) {
    if (!valid_sizes(count, vocab, width) || gradient_kind < 0 || gradient_kind > 1 || table_kind < 0 || table_kind > 1 ||
        (token_bytes != 4 && token_bytes != 8) || gradient_stride < width || !table_gradient ||
        (count > 0 && (!tokens || !out_gradient)))
        return static_cast<int>(cudaErrorInvalidValue);
    const GradientScratch s = gradient_scratch(count, vocab, width);
    const int slices = (width + kSliceColumns - 1) / kSliceColumns;
    const long long row_ctas = (s.chunks * slices + kWarpsPerCta - 1) / kWarpsPerCta;
    const long long zero_ctas = accumulate ? 0 : (vocab + kZeroRows - 1) / kZeroRows;
    const int gradient_bytes = gradient_kind == 0 ? 4 : 2, table_bytes = table_kind == 0 ? 4 : 2;
    if (!aligned_for(out_gradient, gradient_bytes) || !aligned_for(table_gradient, table_bytes) ||
        !aligned_for(tokens, token_bytes) || !aligned_for(token_status, 4) || !workspace || !aligned_for(workspace, 16) ||
        workspace_bytes < s.bytes || row_ctas + zero_ctas > 2147483647ll || s.chunks * slices > 2147483647ll)
        return static_cast<int>(cudaErrorInvalidValue);
    if (count == 0 && accumulate) return static_cast<int>(cudaSuccess);
    const DeviceScope scope(device);
    if (scope.status() != cudaSuccess) return scope.status();
    char* scratch = static_cast<char*>(workspace);
    auto words = [&](long long at) { return reinterpret_cast<unsigned*>(scratch + at); };
    int key_bits = 0;                            // of the largest key, `vocab`
    while ((vocab >> key_bits) != 0) ++key_bits;
    const int passes = (key_bits + kDigitBits - 1) / kDigitBits;
    const SortArguments sort{Tokens{tokens, token_bytes, padding_token, vocab}, {words(s.keys[0]), words(s.keys[1])},
                             {words(s.positions[0]), words(s.positions[1])}, accumulate ? nullptr : words(s.touched),
                             words(s.crossing), token_status, static_cast<unsigned>(count), passes,
                             (key_bits + passes - 1) / passes};
    cudaError_t e = launch_sort(sort, stream);
    if (e != cudaSuccess) return static_cast<int>(e);
    const RowsArguments a{words(s.keys[0]), words(s.positions[0]), words(s.touched), words(s.crossing),
                          reinterpret_cast<float*>(scratch + s.tails), reinterpret_cast<float*>(scratch + s.heads),
                          out_gradient, table_gradient, gradient_stride, static_cast<unsigned>(count),
                          static_cast<unsigned>(vocab), static_cast<unsigned>(s.chunks), width, slices,
                          static_cast<int>(row_ctas), scale, accumulate != 0};
    const bool vector_ok = width % 8 == 0 && aligned_for(out_gradient, 16) && gradient_stride * gradient_bytes % 16 == 0 &&
                           aligned_for(table_gradient, 16);
    const int grid = static_cast<int>(row_ctas + zero_ctas);
    if (gradient_kind == 0)
        e = table_kind == 0 ? run_rows<float, float>(a, vector_ok, grid, stream)
                            : run_rows<float, unsigned short>(a, vector_ok, grid, stream);
    else
        e = table_kind == 0 ? run_rows<unsigned short, float>(a, vector_ok, grid, stream)
                            : run_rows<unsigned short, unsigned short>(a, vector_ok, grid, stream);
    return static_cast<int>(e);
}

}  // namespace
}  // namespace ngb

using namespace ngb;

NNTRAIN_EXPORT int nntrain_embedding_lookup(
    int device, int table_kind, const void* table, const float* scales, int block_size, long long first_value,
    long long vocab, int width, const void* tokens, int token_bytes, long long count, long long padding_token, float scale,
    int out_kind, void* out, long long out_stride, int* token_status, nntrain_stream_t stream) {
    return complete(kOpTokenEmbedding, device,
                    lookup(device, table_kind, table, scales, block_size, first_value, vocab, width, tokens, token_bytes,
                           count, padding_token, scale, out_kind, out, out_stride, token_status,
                           static_cast<cudaStream_t>(stream)));
}

NNTRAIN_EXPORT int nntrain_embedding_gradient_workspace(long long count, long long vocab, int width, long long* bytes) {
    if (!valid_sizes(count, vocab, width) || !bytes)
        return complete(kOpTokenEmbedding, -1, static_cast<int>(cudaErrorInvalidValue));
    *bytes = gradient_scratch(count, vocab, width).bytes;
    return static_cast<int>(cudaSuccess);
}

NNTRAIN_EXPORT int nntrain_embedding_gradient(
    int device, int gradient_kind, const void* out_gradient, long long gradient_stride, const void* tokens, int token_bytes,
    long long count, long long padding_token, float scale, int table_kind, void* table_gradient, long long vocab, int width,
    int accumulate, int* token_status, void* workspace, long long workspace_bytes, nntrain_stream_t stream) {
    return complete(kOpTokenEmbedding, device,
                    gradient(device, gradient_kind, out_gradient, gradient_stride, tokens, token_bytes, count, padding_token,
                             scale, table_kind, table_gradient, vocab, width, accumulate, token_status, workspace,
                             workspace_bytes, static_cast<cudaStream_t>(stream)));
}
