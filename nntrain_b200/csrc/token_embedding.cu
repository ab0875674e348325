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
//   sort    pairs (row, position).  Up to 2048 tokens: one CTA, a bitonic sort
//           in shared memory.  More: one cluster of CTAs, a stable radix sort
//           of up to 9 bits a pass, digit counts exchanged through distributed shared
//           memory, the cluster's barriers between the passes.  (When the whole
//           table is written, the other SMs write its zeros in the same launch:
//           they are most of the traffic and take longer than the sort, whose
//           chain of short waits they hide.)
//   rows    a warp takes 16 or 32 sorted positions x 128 or 256 columns and walks
//           them; a token that lies inside them is finished, of one that
//           crosses the border a partial sum goes to scratch
//   join    a warp per crossing token adds its partials in order, a CTA where
//           there are many
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

#include <atomic>

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
    int width, block_shift;            // block_shift < 0: block is not a power of two; 63: one scale
    float scale;
};

__device__ __forceinline__ float table_scale(const LookupArguments& a, long long value) {
    // (one scale: block_shift is 63)
    const long long at = a.first_value + value;
    return __ldg(a.scales + (a.block_shift >= 0 ? at >> a.block_shift : at / a.block));
}

constexpr int kLookupColumns = 256;    // of a warp: 8 values a lane

template <typename T>
__device__ __forceinline__ void store_values(T* out, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        store_f4(out, make_float4(v[0], v[1], v[2], v[3]));
        store_f4(out + 4, make_float4(v[4], v[5], v[6], v[7]));
    } else {
        *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]),
                                                    pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
}

// A warp: 256 columns of kTokens neighbouring positions, all their rows in
// flight together behind one load of the tokens.  kVector: 8 neighbouring
// values per lane and access (of BFP8: in one block); otherwise single values.
template <int kTable, typename T, bool kVector, int kTokens>
__global__ void __launch_bounds__(kThreads)
embedding_lookup_kernel(LookupArguments a) {
    const int lane = threadIdx.x & 31;
    const long long position = (static_cast<long long>(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5)) * kTokens;
    if (position >= a.count) return;
    const int first = static_cast<int>(blockIdx.y) * kLookupColumns;
    const int here = static_cast<int>(a.count - position < kTokens ? a.count - position : kTokens);
    bool bad = false;
    const int mine = lane < here ? static_cast<int>(a.tokens.at(position + lane, bad)) : -1;
    if (bad && a.status != nullptr) atomicExch(a.status, 1);
    T* out = static_cast<T*>(a.out) + position * a.out_stride;
    int token[kTokens];                          // (a row is below 2^31)
    #pragma unroll
    for (int t = 0; t < kTokens; ++t) token[t] = __shfl_sync(0xffffffffu, mine, t);
    if constexpr (kVector) {
        const int column = first + lane * 8;
        if (column >= a.width) return;
        constexpr int kWords = kTable == kTableF32 ? 8 : (kTable == kTableBf16 ? 4 : 2);
        unsigned raw[kTokens][kWords];
        float row_scale[kTokens];
        #pragma unroll
        for (int t = 0; t < kTokens; ++t) {
            if (token[t] < 0) continue;
            const long long at = static_cast<long long>(token[t]) * a.width + column;
            if constexpr (kTable == kTableBfp8) {
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(static_cast<const signed char*>(a.table) + at));
                raw[t][0] = x.x; raw[t][1] = x.y;
                row_scale[t] = table_scale(a, at);
            } else {
                constexpr int kBytes = kTable == kTableF32 ? 4 : 2;
                const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(a.table) + at * kBytes);
                #pragma unroll
                for (int q = 0; q < kWords / 4; ++q) {
                    const uint4 x = __ldg(p + q);
                    raw[t][q * 4] = x.x; raw[t][q * 4 + 1] = x.y; raw[t][q * 4 + 2] = x.z; raw[t][q * 4 + 3] = x.w;
                }
            }
        }
        T* row = out + column;
        #pragma unroll
        for (int t = 0; t < kTokens; ++t) {
            if (t >= here) break;
            float v[8] = {};
            if (token[t] >= 0) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (kTable == kTableF32) v[i] = __uint_as_float(raw[t][i]);
                    else if constexpr (kTable == kTableBf16) v[i] = i & 1 ? bf16_high(raw[t][i / 2]) : bf16_low(raw[t][i / 2]);
                    else v[i] = __fmul_rn(byte_to_float(raw[t][i / 4] ^ 0x80808080u, i & 3), row_scale[t]);
                    v[i] = __fmul_rn(v[i], a.scale);
                }
            }
            store_values(row, v);
            row += a.out_stride;
        }
    } else {
        #pragma unroll
        for (int t = 0; t < kTokens; ++t) {
            if (t >= here) break;
            const long long row = static_cast<long long>(token[t]) * a.width;
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int column = first + i * 32 + lane;
                if (column >= a.width) continue;
                float v = 0.0f;
                if (token[t] >= 0) {
                    if constexpr (kTable == kTableF32) v = __ldg(static_cast<const float*>(a.table) + row + column);
                    else if constexpr (kTable == kTableBf16) v = bf16_value(__ldg(static_cast<const unsigned short*>(a.table) + row + column));
                    else v = __fmul_rn(static_cast<float>(__ldg(static_cast<const signed char*>(a.table) + row + column)), table_scale(a, row + column));
                    v = __fmul_rn(v, a.scale);
                }
                if constexpr (sizeof(T) == 4) out[t * a.out_stride + column] = v;
                else out[t * a.out_stride + column] = bf16_bits(v);
            }
        }
    }
}

// ---- sort ---------------------------------------------------------------------

constexpr int kSmallBits = 11, kSmallSort = 1 << kSmallBits;   // tokens that one CTA sorts
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
// CTAs of the sorting cluster: 8 is the portable size.  16, where the device has
// them, for more tokens than one for each thread of 8 (rows of 512 added to a
// table: 8192 tokens 21.0 us with 8, 22.0 us with 16; 20000: 32.7 and 31.2 us;
// 65536: 68 and 55 us), or beside zeros, which clusters of 16 write more slowly,
// than 8 hold in their registers (30000 tokens and 307 MB of zeros: 84 us with 8,
// 91 us with 16).
constexpr int kClusterSmall = 8, kClusterLarge = 16;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;   // of a pass at most
constexpr int kLeastBits = 5;                   // a warp of digits
// Bytes of shared memory; with one CTA of an SM there is room for masks beside the counts.
template <int kCluster, int kResident>
constexpr int sort_shared() { return (kSortWarps * (kResident == 1 ? 2 : 1) + 2 + kCluster) * kDigits * 4; }
// Zeros of a CTA beside the sort; and from how many bytes on, these and some for
// each token, they take longer than the sort (tables of 933 MB, 8192 tokens: 155 us
// with two CTAs of an SM, 172 us with one; of 197 MB, 8192 tokens: 61.8 and 60.3 us;
// of 307 MB, 30000 tokens: 98 and 84 us; of 98 MB, 65536 tokens: 119 and 102 us).
constexpr long long kClearPiece = 128 << 10, kClearLong = 128ll << 20, kClearToken = 6 << 10;

struct SortArguments {
    Tokens tokens;
    uint2* pairs[2];                   // (row, position); passes take turns, the order ends in [0]
    unsigned* crossing;                // counters of the rows kernel, cleared here
    unsigned* named;                   // a bit for each row, set where a token names it; null when not asked for
    int* status;
    char* clear;                       // bytes that the CTAs behind the sort's clear
    long long clear_bytes, clear_piece;          // all of them, and those of a CTA
    unsigned count;
    int passes, bits;                  // and the bits of a pass's digit
};

// Zeros to the piece number `piece` of a.clear.  (A table is whole values, so
// its unaligned ends are whole 2-byte pieces.)
__device__ void clear_piece(const SortArguments& a, long long piece) {
    char* begin = a.clear + piece * a.clear_piece;
    const long long left = a.clear_bytes - piece * a.clear_piece, bytes = left < a.clear_piece ? left : a.clear_piece;
    const int head = static_cast<int>((16u - (reinterpret_cast<std::uintptr_t>(begin) & 15u)) & 15u);
    const int ends = head < bytes ? head : static_cast<int>(bytes);
    const int words = static_cast<int>((bytes - ends) / 16);
    uint4* body = reinterpret_cast<uint4*>(begin + ends);
    for (int i = threadIdx.x; i < words; i += kSortThreads) body[i] = make_uint4(0, 0, 0, 0);
    unsigned short* pieces = reinterpret_cast<unsigned short*>(begin);
    for (int i = threadIdx.x; i < ends / 2; i += kSortThreads) pieces[i] = 0;
    for (int i = (ends + words * 16) / 2 + threadIdx.x; i < bytes / 2; i += kSortThreads) pieces[i] = 0;
}

// Ascending sort of `n` numbers, a power of two from 64 to kSmallSort, by the
// warps of a CTA that hold them.  Thread t of warp w has the numbers 64 w + lane
// and 64 w + 32 + lane, so that strides of 16 and less are shuffles, 32 is inside
// a thread, and only the longer ones (15 of the 66 steps of 2048 numbers) go
// through shared memory, by turns through two buffers, a barrier each.  Bound by
// the instructions of the shuffles: 10 us for 2048, 18 us with every step in
// shared memory.
template <typename K>
__device__ void sort_cta(K& x, K& y, int n, K (*buffers)[kSmallSort]) {
    const int lane = threadIdx.x & 31, first = (threadIdx.x >> 5) * 64 + lane, second = first + 32;
    const auto keep = [](K mine, K other, bool smaller) {
        const K low = mine < other ? mine : other, high = mine < other ? other : mine;
        return smaller ? low : high;
    };
    int turn = 0;
    for (int k = 2; k <= n; k <<= 1) {
        const bool x_up = (first & k) == 0, y_up = (second & k) == 0;
        for (int j = k >> 1; j > 32; j >>= 1) {
            K* data = buffers[turn];
            turn ^= 1;
            data[first] = x;
            data[second] = y;
            __syncthreads();
            x = keep(x, data[first ^ j], ((first & j) == 0) == x_up);
            y = keep(y, data[second ^ j], ((second & j) == 0) == y_up);
        }
        if (k >= 64) {
            const K low = x < y ? x : y, high = x < y ? y : x;
            x = x_up ? low : high;
            y = x_up ? high : low;
        }
        #pragma unroll
        for (int j = 16; j > 0; j >>= 1) {
            if (j >= k) continue;
            const bool lower = (lane & j) == 0;
            x = keep(x, __shfl_xor_sync(0xffffffffu, x, j), lower == x_up);
            y = keep(y, __shfl_xor_sync(0xffffffffu, y, j), lower == y_up);
        }
    }
}

// Up to kSmallSort tokens, `padded` a power of two.  Positions without a token
// get the row `vocab`, behind all rows.  K holds a row above kPositionBits of
// its position: 32 bits where they suffice.
template <typename K>
__global__ void __launch_bounds__(kSortThreads)
embedding_small_sort_kernel(SortArguments a, int padded) {
    constexpr int kPositionBits = sizeof(K) == 4 ? kSmallBits : 32;
    __shared__ K buffers[2][kSmallSort];
    static_assert(kSmallSort == 2 * kSortThreads && kSmallSort == 1 << kSmallBits, "two numbers for each thread");
    let_next_start();
    if (blockIdx.x > 0) {
        clear_piece(a, blockIdx.x - 1);
        return;
    }
    if (threadIdx.x < 2) a.crossing[threadIdx.x] = 0;
    if (a.named != nullptr) {
        for (long long i = threadIdx.x; i * 32 < a.tokens.vocab; i += kSortThreads) a.named[i] = 0;
        __syncthreads();
    }
    const int first = (threadIdx.x >> 5) * 64 + (threadIdx.x & 31);
    if (first >= padded) return;                 // whole warps; barriers wait for those that are left
    bool bad = false;
    const auto load = [&](int i) {
        const long long token = i < static_cast<int>(a.count) ? a.tokens.at(i, bad) : -1;
        return (static_cast<K>(token < 0 ? a.tokens.vocab : token) << kPositionBits) | static_cast<K>(i);
    };
    K pair[2] = {load(first), load(first + 32)};
    sort_cta<K>(pair[0], pair[1], padded, buffers);
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = first + 32 * h;
        if (at >= static_cast<int>(a.count)) continue;
        const unsigned row = static_cast<unsigned>(pair[h] >> kPositionBits);
        a.pairs[0][at] = make_uint2(row, static_cast<unsigned>(pair[h] & ((static_cast<K>(1) << kPositionBits) - 1)));
        if (a.named != nullptr && row < a.tokens.vocab) atomicOr(a.named + (row >> 5), 1u << (row & 31u));
    }
    if (bad && a.status != nullptr) atomicExch(a.status, 1);
}

// The first kSteps groups of 32 pairs of a warp's stretch.
template <int kSteps>
struct Head {
    uint2 pairs[kSteps];
};

template <int kSteps, typename Load>
__device__ __forceinline__ Head<kSteps> load_head(unsigned from, unsigned to, Load load) {
    Head<kSteps> head;
    #pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const unsigned at = from + s * 32 + (threadIdx.x & 31);
        head.pairs[s] = at < to ? load(at) : make_uint2(0, 0);
    }
    return head;
}

// Walks [from, to) 32 at a time, in order: visit(here, pair).  kSteps groups are
// loaded before the first of them is visited; the first ones are there already.
template <int kSteps, typename Load, typename Visit>
__device__ __forceinline__ void walk(unsigned from, unsigned to, Head<kSteps> head, Load load, Visit visit) {
    const int lane = threadIdx.x & 31;
    for (unsigned base = from; base < to; base += 32 * kSteps) {
        if (base != from) head = load_head<kSteps>(base, to, load);
        #pragma unroll
        for (int s = 0; s < kSteps; ++s)
            if (base + s * 32 < to) visit(base + s * 32 + lane < to, head.pairs[s]);
    }
}

// Lanes that are here and have the lane's digit (of a lane that is not here:
// anything).  With masks, a zero for each digit of the warp's: every lane sets its
// bit, and the first of a digit leaves a zero again; the caller's next __syncwarp()
// ends that.  Without: a vote per bit.  (Votes, of which an SM finishes one in some
// 4 clocks, were what ranking waited for: 131072 tokens of 128 columns added 63 us
// with them, 60 us with masks; a match instruction is no faster than the votes.)
template <bool kMasks>
__device__ __forceinline__ unsigned same_digit(bool here, unsigned digit, int bits, unsigned* masks) {
    if constexpr (kMasks) {
        const unsigned lane = threadIdx.x & 31;
        if (here) atomicOr(masks + digit, 1u << lane);
        __syncwarp();
        const unsigned same = masks[digit];
        __syncwarp();
        if (here && (same & ((1u << lane) - 1u)) == 0) masks[digit] = 0;
        return same;
    } else {
        unsigned same = __ballot_sync(0xffffffffu, here);
        #pragma unroll
        for (int b = 0; b < kDigitBits; ++b) {
            if (b >= bits) break;
            const bool set = (digit >> b) & 1u;
            const unsigned votes = __ballot_sync(0xffffffffu, set);
            same &= set ? votes : ~votes;
        }
        return same;
    }
}

// Stable: warps own consecutive stretches of the input, a warp walks its
// stretch 32 at a time, and equal digits keep the order of their lanes.  A pair
// is stored in one piece: the scattered stores of a few SMs, a 32-byte sector
// each, are most of a pass over many tokens (65536 tokens, 8 CTAs, all digits
// ranked twice: 47 us with rows and positions apart, 35 us so).  A stretch that fits a warp's registers is
// ranked once, when its digits are counted, and only placed afterwards.  Every CTA
// writes its counts into the others' shared memory in front of the barrier that
// it needs anyway, and sums them from its own.
//
// CTAs behind the first cluster clear.  kResident: 2 CTAs of an SM write zeros at
// 7.3 TB/s, one at 6.3 TB/s, but their 32 registers hold no ranks, and the sort
// takes longer; for the tables whose zeros do.
template <int kCluster, int kSteps, int kResident>
__global__ void __launch_bounds__(kSortThreads, kResident)
embedding_sort_kernel(SortArguments a) {
    extern __shared__ __align__(16) unsigned shared[];
    unsigned* counts = shared;                               // [warps][digits]
    unsigned* totals = shared + kSortWarps * kDigits;        // [digits]
    unsigned* starts = totals + kDigits;                     // [digits]
    unsigned* shares = starts + kDigits;                     // [CTAs][digits]: the totals of each
    constexpr bool kMasks = kResident == 1;
    unsigned* masks = shares + kCluster * kDigits + (kMasks ? (threadIdx.x >> 5) * kDigits : 0);
    __shared__ unsigned sums[32];
    let_next_start();
    if (blockIdx.x >= kCluster) {                            // whole clusters of them: no barrier is shared
        const long long piece = blockIdx.x - kCluster;
        if (piece * a.clear_piece < a.clear_bytes) clear_piece(a, piece);
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned below_lane = (1u << lane) - 1u;
    constexpr unsigned kWorkers = kCluster * kSortWarps;
    const unsigned stretch = ((a.count + kWorkers - 1) / kWorkers + 31u) & ~31u;
    const bool held = kResident == 1 && stretch <= 32 * kSteps;
    const unsigned long long begin = static_cast<unsigned long long>(rank * kSortWarps + warp) * stretch;
    const unsigned first = begin < a.count ? static_cast<unsigned>(begin) : a.count;
    const unsigned last = begin + stretch < a.count ? static_cast<unsigned>(begin + stretch) : a.count;
    const int digits = 1 << a.bits;
    unsigned* mine = counts + warp * kDigits;
    if (rank == 0 && threadIdx.x < 2) a.crossing[threadIdx.x] = 0;
    if (a.named != nullptr) {
        for (long long i = rank * kSortThreads + threadIdx.x; i * 32 < a.tokens.vocab; i += kCluster * kSortThreads) a.named[i] = 0;
        cluster.sync();
    }
    if (kMasks)
        for (int i = lane; i < digits; i += 32) masks[i] = 0;
    bool bad = false;
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");        // this CTA's shared memory may be written
    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = pass * a.bits;
        uint2* out = (a.passes - 1 - pass) & 1 ? a.pairs[1] : a.pairs[0];
        const uint2* in = (a.passes - 1 - pass) & 1 ? a.pairs[0] : a.pairs[1];
        const auto load = [&](unsigned i) {
            if (pass > 0) return __ldcg(in + i);
            const long long token = a.tokens.at(i, bad);
            return make_uint2(static_cast<unsigned>(token < 0 ? a.tokens.vocab : token), i);
        };
        const auto digit_of = [&](uint2 pair) { return (pair.x >> shift) & static_cast<unsigned>(digits - 1); };
        const auto name = [&](bool here, uint2 pair) {
            if (pass == 0 && here && a.named != nullptr && pair.x < a.tokens.vocab)
                atomicOr(a.named + (pair.x >> 5), 1u << (pair.x & 31u));
        };
        const Head<kSteps> head = load_head<kSteps>(first, last, load);
        for (int i = threadIdx.x; i < kSortWarps << a.bits; i += kSortThreads)
            counts[(i >> a.bits) * kDigits + (i & (digits - 1))] = 0;
        __syncthreads();
        unsigned places[kSteps];                             // in the warp's share of the digit
        if (held) {
            #pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                if (first + s * 32 >= last) break;
                const bool here = first + s * 32 + lane < last;
                const unsigned digit = digit_of(head.pairs[s]), there = mine[digit];
                const unsigned same = same_digit<kMasks>(here, digit, a.bits, masks), before = same & below_lane;
                places[s] = there + __popc(before);
                if (here && before == 0) mine[digit] = there + __popc(same);
                __syncwarp();
                name(here, head.pairs[s]);
            }
        } else {
            walk<kSteps>(first, last, head, load, [&](bool here, uint2 pair) {
                const unsigned digit = digit_of(pair), same = same_digit<kMasks>(here, digit, a.bits, masks);
                if (here && (same & below_lane) == 0) mine[digit] += __popc(same);
                name(here, pair);
                __syncwarp();
            });
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < digits) {
            unsigned sum = 0;
            #pragma unroll 16
            for (int w = 0; w < kSortWarps; ++w) {
                const unsigned n = counts[w * kDigits + threadIdx.x];
                counts[w * kDigits + threadIdx.x] = sum;
                sum += n;
            }
            totals[threadIdx.x] = sum;
        }
        if (pass == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        __syncthreads();
        for (int i = threadIdx.x; i < kCluster << (a.bits - 2); i += kSortThreads) {
            const int quad = i & (digits / 4 - 1);
            uint4* share = reinterpret_cast<uint4*>(cluster.map_shared_rank(shares + rank * kDigits, i >> (a.bits - 2)));
            share[quad] = reinterpret_cast<const uint4*>(totals)[quad];
        }
        cluster.sync();
        // first place of this CTA's share of each digit
        unsigned below = 0, all = 0, inclusive = 0;
        if (static_cast<int>(threadIdx.x) < digits) {
            #pragma unroll
            for (unsigned r = 0; r < kCluster; ++r) {
                const unsigned n = shares[r * kDigits + threadIdx.x];
                below += r < rank ? n : 0;
                all += n;
            }
            inclusive = all;
            #pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
                const unsigned n = __shfl_up_sync(0xffffffffu, inclusive, offset);
                inclusive += lane >= offset ? n : 0;
            }
            if (lane == 31) sums[warp] = inclusive;
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < digits) {
            inclusive += __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0);
            starts[threadIdx.x] = inclusive - all + below;
        }
        __syncthreads();
        if (held) {
            #pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const bool here = first + s * 32 + lane < last;
                const unsigned digit = digit_of(head.pairs[s]);
                const unsigned place = here ? starts[digit] + mine[digit] + places[s] : a.count;
                if (place < a.count) out[place] = head.pairs[s];         // (it is, unless the tokens are written meanwhile)
            }
        } else {
            walk<kSteps>(first, last, head, load, [&](bool here, uint2 pair) {
                const unsigned digit = digit_of(pair), same = same_digit<kMasks>(here, digit, a.bits, masks);
                const unsigned before = same & below_lane;
                const unsigned place = here ? starts[digit] + mine[digit] + __popc(before) : a.count;
                if (place < a.count) out[place] = pair;
                __syncwarp();                                // everyone has read its place
                if (here && before == 0) mine[digit] += __popc(same);
                __syncwarp();
            });
        }
        // the pass is in memory, and nobody reads these shares (the last pass writes no more of them)
        if (pass + 1 < a.passes) cluster.sync();
    }
    if (bad && a.status != nullptr) atomicExch(a.status, 1);
}

// ---- rows and join --------------------------------------------------------------

// Sorted positions of a warp.  32, so that few tokens cross; 16 where 32 leave
// the 148 SMs less than 64 warps of 256 columns each (added gradients: 500 tokens x
// 1536 13.5 us with 16, 18.1 us with 32; 16384 x 512 24.4 and 28.3 us; 131072 x 768
// 148 and 138 us, 166 us with 8).  The border was measured when the join loaded
// partials one after the other; now 32 would do a little better from about 4000
// such warps on (65536 x 512 55.4 and 53.3 us).
constexpr int kChunkMost = 32, kChunkLeast = 16;
constexpr int kZeroRows = 32;                   // rows of a CTA that writes late zeros: one word of the bitmap
// Columns of a warp: one 128-bit load of a lane, or 8 single values.
template <typename G, bool kVector>
__host__ __device__ constexpr int lane_values() { return kVector && sizeof(G) == 4 ? 4 : 8; }

struct RowsArguments {
    const uint2* pairs;                // sorted (row, position)
    unsigned* crossing;                // tokens that cross chunks: number of short and of long ones, then
    unsigned* crossing_short;          // the chunks in which they begin
    unsigned* crossing_long;
    unsigned* rows_short;              // and their rows, where the sort's second array was
    unsigned* rows_long;
    float* tails;                      // [chunk][width]: sum up to the chunk's end of a token that goes on
    float* heads;                      // [chunk][width]: rest of a token that began in an earlier chunk
    const void* gradient;              // dout
    void* table;
    long long gradient_stride;
    const unsigned* named;             // the sort's bitmap
    long long late;                    // rows from here on were not cleared beside the sort
    unsigned count, vocab, chunk, chunks;    // chunk: positions of one
    int width, slices, row_ctas, long_ctas, join_ctas;
    unsigned late_groups, join_groups; // groups of kZeroRows rows from `late` on, and the first of the join's
    float scale;
    bool accumulate;
};

// Column of the lane's i-th value: neighbours, or every 32nd.
template <int kValues, bool kVector>
__device__ __forceinline__ int lane_column(int first, int lane, int i) {
    return kVector ? first + lane * kValues + i : first + i * 32 + lane;
}

template <typename T>
__device__ __forceinline__ float value_of(T raw) {
    if constexpr (sizeof(T) == 4) return raw;
    else return bf16_value(raw);
}

// What is there in a row of the table, to be added to.
template <typename T, int kValues, bool kVector>
__device__ __forceinline__ void load_old(const RowsArguments& a, unsigned row, int first, int lane, float (&old)[kValues]) {
    const T* p = static_cast<const T*>(a.table) + static_cast<long long>(row) * a.width;
    #pragma unroll
    for (int i = 0; i < kValues; i += kVector ? 4 : 1) {
        const int column = lane_column<kValues, kVector>(first, lane, i);
        if constexpr (!kVector) {
            old[i] = column < a.width ? value_of(p[column]) : 0.0f;
        } else if constexpr (sizeof(T) == 4) {
            const float4 x = column < a.width ? load_f4(p + column) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            old[i] = x.x; old[i + 1] = x.y; old[i + 2] = x.z; old[i + 3] = x.w;
        } else {
            const uint2 x = column < a.width ? *reinterpret_cast<const uint2*>(p + column) : make_uint2(0, 0);
            old[i] = bf16_low(x.x); old[i + 1] = bf16_high(x.x); old[i + 2] = bf16_low(x.y); old[i + 3] = bf16_high(x.y);
        }
    }
}

// table[row] = scale * sum (+ old), rounded once.
template <typename T, int kValues, bool kVector, bool kAdd>
__device__ __forceinline__ void store_row(const RowsArguments& a, unsigned row, int first, int lane, const float (&sum)[kValues],
                                          const float (&old)[kAdd ? kValues : 1]) {
    T* out = static_cast<T*>(a.table) + static_cast<long long>(row) * a.width;
    #pragma unroll
    for (int i = 0; i < kValues; i += kVector ? 4 : 1) {
        const int column = lane_column<kValues, kVector>(first, lane, i);
        if (column >= a.width) continue;
        float x[kVector ? 4 : 1];
        #pragma unroll
        for (int q = 0; q < (kVector ? 4 : 1); ++q) {
            if constexpr (kAdd) x[q] = __fmaf_rn(sum[i + q], a.scale, old[i + q]);
            else x[q] = __fmul_rn(sum[i + q], a.scale);
        }
        if constexpr (!kVector) {
            if constexpr (sizeof(T) == 4) out[column] = x[0];
            else out[column] = bf16_bits(x[0]);
        } else if constexpr (sizeof(T) == 4) {
            store_f4(out + column, make_float4(x[0], x[1], x[2], x[3]));
        } else {
            *reinterpret_cast<uint2*>(out + column) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        }
    }
}

template <int kValues, bool kVector>
__device__ __forceinline__ void store_partial(float* partials, unsigned chunk, int width, int first, int lane,
                                              const float (&sum)[kValues]) {
    float* out = partials + static_cast<long long>(chunk) * width;
    #pragma unroll
    for (int i = 0; i < kValues; i += kVector ? 4 : 1) {
        const int column = lane_column<kValues, kVector>(first, lane, i);
        if (column >= width) continue;
        if constexpr (kVector) store_f4(out + column, make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]));
        else out[column] = sum[i];
    }
}

// The zeros of 32 rows, those that no token names.
template <typename T>
__device__ void zero_rows(const RowsArguments& a, unsigned group) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = warp; r < kZeroRows; r += kWarpsPerCta) {
        const long long row = a.late + static_cast<long long>(group) * kZeroRows + r;
        if (row >= a.vocab || ((a.named[row >> 5] >> (row & 31)) & 1u)) continue;
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

// A token that goes on for this many chunks is long: a CTA adds its partials,
// not a warp.
constexpr unsigned kLongChunks = 16;

template <typename G, typename T, bool kVector, bool kAdd>
__global__ void __launch_bounds__(kThreads)
embedding_rows_kernel(RowsArguments a) {
    constexpr int kValues = lane_values<G, kVector>();
    const int lane = threadIdx.x & 31;
    const unsigned task = blockIdx.x * kWarpsPerCta + (threadIdx.x >> 5);
    const unsigned chunk = task / a.slices, size = a.chunk, base = chunk * size;
    wait_for_previous();
    let_next_start();
    if (static_cast<int>(blockIdx.x) >= a.row_ctas) {
        zero_rows<T>(a, blockIdx.x - a.row_ctas);
        return;
    }
    if (chunk >= a.chunks) return;
    const int first = static_cast<int>(task - chunk * a.slices) * (kValues * 32);
    const uint2 none = make_uint2(a.vocab, 0);
    const uint2 pair = lane < static_cast<int>(size) && base + lane < a.count ? a.pairs[base + lane] : none;
    // (the sort leaves rows and positions; tokens that are written while they are sorted must not lead out of the table)
    const unsigned key = pair.x < a.vocab ? pair.x : a.vocab, position = pair.y < a.count ? pair.y : 0;
    const unsigned key_before = chunk > 0 ? a.pairs[base - 1].x : a.vocab;
    const unsigned key_behind = base + size < a.count ? a.pairs[base + size].x : a.vocab;
    const unsigned named = __ballot_sync(0xffffffffu, key != a.vocab);       // rows come first
    const int n = named == 0xffffffffu ? 32 : __ffs(static_cast<int>(~named)) - 1;
    // Rows whose loads are in flight together; when adding, with the rows of the table that they complete (one after
    // the other these were most of a warp's time: 15 us for 300 tokens, 9 us so).
    constexpr int kBatch = kVector && !kAdd ? 8 : 4;
    const G* gradient = static_cast<const G*>(a.gradient);
    float sum[kValues] = {};
    const unsigned following = __shfl_down_sync(0xffffffffu, key, 1);
    const unsigned next_key = lane + 1 < static_cast<int>(size) ? following : key_behind;
    for (int j = 0; j < n; j += kBatch) {
        uint4 raw[kBatch];
        float old[kBatch][kAdd ? kValues : 1];
        G single[kBatch][kValues];
        #pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const unsigned at = __shfl_sync(0xffffffffu, position, (j + b) & 31);
            const unsigned here = __shfl_sync(0xffffffffu, key, (j + b) & 31), next = __shfl_sync(0xffffffffu, next_key, (j + b) & 31);
            if (j + b >= n) continue;
            if constexpr (kAdd)
                if (here != next && here != key_before) load_old<T, kValues, kVector>(a, here, first, lane, old[b]);
            const G* row = gradient + static_cast<long long>(at) * a.gradient_stride;
            if constexpr (kVector) {
                const int column = lane_column<kValues, true>(first, lane, 0);
                raw[b] = column < a.width ? __ldcs(reinterpret_cast<const uint4*>(row + column)) : make_uint4(0, 0, 0, 0);
            } else {
                #pragma unroll
                for (int i = 0; i < kValues; ++i) {
                    const int column = lane_column<kValues, false>(first, lane, i);
                    single[b][i] = column < a.width ? __ldcs(row + column) : G(0);
                }
            }
        }
        #pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (j + b >= n) continue;
            const unsigned here = __shfl_sync(0xffffffffu, key, j + b), next = __shfl_sync(0xffffffffu, next_key, j + b);
            if constexpr (kVector) {
                const unsigned w[4] = {raw[b].x, raw[b].y, raw[b].z, raw[b].w};
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (sizeof(G) == 4) {
                        sum[i] = __fadd_rn(sum[i], __uint_as_float(w[i]));
                    } else {
                        sum[2 * i] = __fadd_rn(sum[2 * i], bf16_low(w[i]));
                        sum[2 * i + 1] = __fadd_rn(sum[2 * i + 1], bf16_high(w[i]));
                    }
                }
            } else {
                #pragma unroll
                for (int i = 0; i < kValues; ++i) sum[i] = __fadd_rn(sum[i], value_of(single[b][i]));
            }
            if (next == here && j + b + 1 < static_cast<int>(size)) continue;      // the token goes on in this chunk
            const bool begun_before = here == key_before;
            if (next == here) {
                store_partial<kValues, kVector>(a.tails, chunk, a.width, first, lane, sum);
                if (!begun_before && first == 0 && lane == 0) {
                    const unsigned long long far = static_cast<unsigned long long>(chunk + kLongChunks) * size;
                    const bool is_long = far < a.count && a.pairs[far].x == here;
                    const unsigned place = atomicAdd(a.crossing + is_long, 1u);
                    (is_long ? a.crossing_long : a.crossing_short)[place] = chunk;
                    (is_long ? a.rows_long : a.rows_short)[place] = here;
                }
            } else if (begun_before) {
                store_partial<kValues, kVector>(a.heads, chunk, a.width, first, lane, sum);
            } else {
                store_row<T, kValues, kVector, kAdd>(a, here, first, lane, sum, old[b]);
            }
            #pragma unroll
            for (int i = 0; i < kValues; ++i) sum[i] = 0.0f;
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
        const bool holds = probe < high && a.pairs[probe * a.chunk].x == key;
        const unsigned held = __popc(__ballot_sync(0xffffffffu, holds));   // the first `held` probes hold it
        const unsigned long long beyond = low + static_cast<unsigned long long>(step) * (held + 1);
        low += step * held;
        if (beyond < high && held < 32) high = static_cast<unsigned>(beyond);
        step = (high - low + 31) / 32;
    }
    return low;
}

// sum += the partials [from, to) of the token that begins in chunk `begin`: the
// tails of its chunks, the head of the last one.
template <int kValues, bool kVector>
__device__ __forceinline__ void add_partials(const RowsArguments& a, unsigned begin, unsigned end, unsigned from, unsigned to,
                                             int first, int lane, float (&sum)[kValues]) {
    // Partials whose loads are in flight together: all of a short token's where a lane has 4 columns.
    constexpr int kBatch = 64 / kValues;
    for (unsigned p = from; p < to; p += kBatch) {
        float values[kBatch][kValues];
        #pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const unsigned at = begin + p + b;
            const float* partial = (at == end ? a.heads : a.tails) + static_cast<long long>(at) * a.width;
            #pragma unroll
            for (int i = 0; i < kValues; i += kVector ? 4 : 1) {
                const int column = lane_column<kValues, kVector>(first, lane, i);
                const bool here = p + b < to && column < a.width;
                if constexpr (kVector) {
                    const float4 x = here ? load_f4(partial + column) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    values[b][i] = x.x; values[b][i + 1] = x.y; values[b][i + 2] = x.z; values[b][i + 3] = x.w;
                } else {
                    values[b][i] = here ? partial[column] : 0.0f;
                }
            }
        }
        #pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (p + b >= to) break;
            #pragma unroll
            for (int i = 0; i < kValues; ++i) sum[i] = __fadd_rn(sum[i], values[b][i]);
        }
    }
}

// The first CTAs take the long crossing tokens (and a slice of their columns):
// each of 8 warps adds an eighth of the partials in order, the eighths are
// added in order.  In the others a warp takes a short one.
template <typename T, int kValues, bool kVector, bool kAdd>
__global__ void __launch_bounds__(kThreads)
embedding_join_kernel(RowsArguments a) {
    __shared__ float sums[kWarpsPerCta][kValues * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool is_long = static_cast<int>(blockIdx.x) < a.long_ctas;
    wait_for_previous();
    if (static_cast<int>(blockIdx.x) >= a.join_ctas) {
        zero_rows<T>(a, a.join_groups + blockIdx.x - a.join_ctas);
        return;
    }
    const unsigned* list = is_long ? a.crossing_long : a.crossing_short;
    const unsigned* rows = is_long ? a.rows_long : a.rows_short;
    const unsigned long long step = is_long ? a.long_ctas : static_cast<unsigned long long>(a.join_ctas - a.long_ctas) * kWarpsPerCta;
    unsigned long long task = is_long ? blockIdx.x : static_cast<unsigned long long>(blockIdx.x - a.long_ctas) * kWarpsPerCta + warp;
    // (the first entry is loaded beside the number of them, from a place that the list has)
    const unsigned long long places = is_long ? a.chunks / kLongChunks + 1 : a.chunks;
    unsigned long long place = task / a.slices < places ? task / a.slices : 0;
    unsigned begin = list[place], key = rows[place];
    const unsigned long long tasks = static_cast<unsigned long long>(a.crossing[is_long]) * a.slices;
    for (; task < tasks; task += step) {
        if (task >= step) {
            place = task / a.slices;
            begin = list[place];
            key = rows[place];
        }
        const int first = static_cast<int>(task % a.slices) * (kValues * 32);
        const unsigned end = last_chunk_of(a, key, begin, lane), parts = end - begin + 1;
        float sum[kValues] = {}, old[kAdd ? kValues : 1];
        if constexpr (kAdd)
            if (!is_long || warp == 0) load_old<T, kValues, kVector>(a, key, first, lane, old);
        if (!is_long) {
            add_partials<kValues, kVector>(a, begin, end, 0, parts, first, lane, sum);
            store_row<T, kValues, kVector, kAdd>(a, key, first, lane, sum, old);
            continue;
        }
        const unsigned share = (parts + kWarpsPerCta - 1) / kWarpsPerCta;
        const unsigned from = warp * share < parts ? warp * share : parts, to = from + share < parts ? from + share : parts;
        add_partials<kValues, kVector>(a, begin, end, from, to, first, lane, sum);
        #pragma unroll
        for (int i = 0; i < kValues; ++i) sums[warp][i * 32 + lane] = sum[i];
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < kWarpsPerCta; ++w) {
                #pragma unroll
                for (int i = 0; i < kValues; ++i) sum[i] = __fadd_rn(sum[i], sums[w][i * 32 + lane]);
            }
            store_row<T, kValues, kVector, kAdd>(a, key, first, lane, sum, old);
        }
        __syncthreads();
    }
}

// ---- entry points ----------------------------------------------------------------

constexpr long long kLateBytes = 128ll << 20;
constexpr long long kMostTokens = (1ll << 31) - 64, kMostVocab = 1ll << 31;
constexpr int kMostWidth = (1 << 24) - 256;     // 65535 slices of the lookup

bool valid_sizes(long long count, long long vocab, int width) {
    return count >= 0 && count <= kMostTokens && vocab >= 1 && vocab <= kMostVocab && width >= 1 && width <= kMostWidth;
}

template <int kTable, typename T, int kTokens>
cudaError_t launch_lookup(const LookupArguments& a, bool vector_ok, cudaStream_t stream) {
    constexpr int kCtaTokens = kWarpsPerCta * kTokens;
    const dim3 grid(static_cast<unsigned>((a.count + kCtaTokens - 1) / kCtaTokens),
                    static_cast<unsigned>((a.width + kLookupColumns - 1) / kLookupColumns));
    return launch(vector_ok ? embedding_lookup_kernel<kTable, T, true, kTokens> : embedding_lookup_kernel<kTable, T, false, kTokens>,
                  grid, kThreads, 0, stream, a);
}

// Four tokens a warp once that still leaves each SM 16 warps, else one.
template <int kTable, typename T>
cudaError_t run_lookup(const LookupArguments& a, bool vector_ok, cudaStream_t stream) {
    const long long warps = a.count * ((a.width + kLookupColumns - 1) / kLookupColumns);
    return warps >= 64ll * sm_count() ? launch_lookup<kTable, T, 4>(a, vector_ok, stream)
                                      : launch_lookup<kTable, T, 1>(a, vector_ok, stream);
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
    const DeviceScope scope(device);
    if (scope.status() != cudaSuccess) return scope.status();
    int shift = block_size == 0 ? 63 : -1;
    if (block_size > 0 && (block_size & (block_size - 1)) == 0)
        for (shift = 0; (1 << shift) < block_size;) ++shift;
    const LookupArguments a{Tokens{tokens, token_bytes, padding_token, vocab}, table, scales, out, token_status, count,
                            out_stride, first_value, block_size, width, shift, scale};
    const bool vector_ok = width % 8 == 0 && aligned_for(table, table_kind == kTableBfp8 ? 8 : 16) && aligned_for(out, 16) &&
                           out_stride * out_bytes % 16 == 0 &&
                           (table_kind != kTableBfp8 || block_size == 0 || (block_size % 8 == 0 && first_value % 8 == 0));
    if (out_kind == 0) {
        if (table_kind == kTableF32) return static_cast<int>(run_lookup<kTableF32, float>(a, vector_ok, stream));
        if (table_kind == kTableBf16) return static_cast<int>(run_lookup<kTableBf16, float>(a, vector_ok, stream));
        return static_cast<int>(run_lookup<kTableBfp8, float>(a, vector_ok, stream));
    }
    if (table_kind == kTableF32) return static_cast<int>(run_lookup<kTableF32, unsigned short>(a, vector_ok, stream));
    if (table_kind == kTableBf16) return static_cast<int>(run_lookup<kTableBf16, unsigned short>(a, vector_ok, stream));
    return static_cast<int>(run_lookup<kTableBfp8, unsigned short>(a, vector_ok, stream));
}

// Scratch of one gradient call, every part on a 256-byte boundary.
struct GradientScratch {
    long long pairs[2], named, crossing, crossing_short, crossing_long, tails, heads, bytes;
    int chunk;
    long long chunks;
};

GradientScratch gradient_scratch(long long count, long long vocab, int width) {
    GradientScratch s{};
    auto take = [&](long long bytes) {
        const long long at = s.bytes;
        s.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    const long long warps = (count + kChunkMost - 1) / kChunkMost * ((width + 255) / 256);
    s.chunk = warps < 148 * 64 ? kChunkLeast : kChunkMost;
    s.chunks = (count + s.chunk - 1) / s.chunk;
    for (int i = 0; i < 2; ++i) s.pairs[i] = take(count * 8);
    s.named = take((vocab + 31) / 32 * 4);
    s.crossing = take(8);
    s.crossing_short = take(s.chunks * 4);
    s.crossing_long = take((s.chunks / kLongChunks + 1) * 4);
    s.tails = take(s.chunks * width * 4);
    s.heads = take(s.chunks * width * 4);
    return s;
}

using SortKernel = void (*)(SortArguments);

cudaLaunchConfig_t cluster_launch(int cluster, long long ctas, int shared, cudaLaunchAttribute& attribute, cudaStream_t stream) {
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = cluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(ctas));
    config.blockDim = dim3(kSortThreads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return config;
}

// The sorting cluster, and as many more as `pieces` CTAs take.
template <int kCluster, int kResident>
cudaError_t launch_cluster(SortKernel kernel, long long pieces, const SortArguments& a, cudaStream_t stream) {
    // the limit belongs to the device's context; setting it costs a fraction of a launch
    const cudaError_t e =
        reported(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sort_shared<kCluster, kResident>()));
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attribute{};
    const long long ctas = kCluster + (pieces + kCluster - 1) / kCluster * kCluster;
    const cudaLaunchConfig_t config = cluster_launch(kCluster, ctas, sort_shared<kCluster, kResident>(), attribute, stream);
    return reported(cudaLaunchKernelEx(&config, kernel, a));
}

// Whether the current device runs clusters of 16 such CTAs: asked once per
// device, after which the kernels may be launched so.
bool large_clusters() {
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];     // 0: not asked yet, 1: no, 2: yes
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kDevices) return false;
    int answer = known[device].load(std::memory_order_relaxed);
    if (answer == 0) {
        const auto can_run = [](SortKernel kernel) {
            constexpr int kShared = sort_shared<kClusterLarge, 1>();
            cudaLaunchAttribute attribute{};
            const cudaLaunchConfig_t config = cluster_launch(kClusterLarge, kClusterLarge, kShared, attribute, nullptr);
            int clusters = 0;
            return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShared) == cudaSuccess &&
                   cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                   cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) == cudaSuccess && clusters > 0;
        };
        const bool can = can_run(embedding_sort_kernel<kClusterLarge, 4, 1>) && can_run(embedding_sort_kernel<kClusterLarge, 8, 1>);
        if (!can) cudaGetLastError();
        answer = can ? 2 : 1;
        known[device].store(answer, std::memory_order_relaxed);
    }
    return answer == 2;
}

cudaError_t launch_sort(SortArguments a, cudaStream_t stream) {
    const bool small = a.count <= kSmallSort, two_ctas = !small && a.clear_bytes >= kClearLong + kClearToken * a.count;
    a.clear_piece = small || two_ctas ? kClearPiece : 2 * kClearPiece;
    const long long pieces = (a.clear_bytes + a.clear_piece - 1) / a.clear_piece;
    if (pieces > 2147483000ll) return cudaErrorInvalidValue;
    if (small) {
        int padded = 64;
        while (padded < static_cast<int>(a.count)) padded <<= 1;
        const unsigned ctas = static_cast<unsigned>(1 + pieces);
        return launch(a.tokens.vocab < 1ll << (32 - kSmallBits) ? embedding_small_sort_kernel<unsigned>
                                                                : embedding_small_sort_kernel<unsigned long long>,
                      dim3(ctas), kSortThreads, 0, stream, a, padded);
    }
    int bits = 1;                                // of the largest key, `vocab`
    while (a.tokens.vocab >> bits != 0) ++bits;
    a.passes = (bits + kDigitBits - 1) / kDigitBits;
    a.bits = (bits + a.passes - 1) / a.passes;
    if (a.bits < kLeastBits) a.bits = kLeastBits;
    if (two_ctas) return launch_cluster<kClusterSmall, 2>(embedding_sort_kernel<kClusterSmall, 4, 2>, pieces, a, stream);
    if (a.count <= kClusterSmall * kSortThreads * (pieces > 0 ? 4 : 1) || !large_clusters())
        return launch_cluster<kClusterSmall, 1>(embedding_sort_kernel<kClusterSmall, 4, 1>, pieces, a, stream);
    return launch_cluster<kClusterLarge, 1>(a.count > kClusterLarge * kSortThreads * 4 ? embedding_sort_kernel<kClusterLarge, 8, 1>
                                                                                    : embedding_sort_kernel<kClusterLarge, 4, 1>,
                                         pieces, a, stream);
}

template <typename G, typename T, bool kVector, bool kAdd>
cudaError_t run_rows(RowsArguments a, cudaStream_t stream) {
    constexpr int kValues = lane_values<G, kVector>();
    const long long slices = (a.width + kValues * 32 - 1) / (kValues * 32);
    if (a.chunks * slices > 2147483647ll) return cudaErrorInvalidValue;
    a.slices = static_cast<int>(slices);
    a.row_ctas = static_cast<int>((a.chunks * slices + kWarpsPerCta - 1) / kWarpsPerCta);
    const bool join = a.chunks > 1;
    a.join_groups = join ? a.late_groups - a.late_groups / 3 : a.late_groups;
    const cudaError_t e = launch_dependent(embedding_rows_kernel<G, T, kVector, kAdd>, a.row_ctas + static_cast<int>(a.join_groups),
                                           kThreads, 0, stream, a);
    if (e != cudaSuccess || !join) return e;
    a.long_ctas = a.chunks > kLongChunks ? grid_for(a.chunks / kLongChunks * slices, 2) : 0;
    a.join_ctas = a.long_ctas + grid_for(((a.chunks - 1) * slices + kWarpsPerCta - 1) / kWarpsPerCta, 4);
    return launch_dependent(embedding_join_kernel<T, kValues, kVector, kAdd>, a.join_ctas + static_cast<int>(a.late_groups - a.join_groups),
                            kThreads, 0, stream, a);
}

template <typename G, typename T>
cudaError_t run_rows(const RowsArguments& a, bool vector_ok, cudaStream_t stream) {
    if (a.accumulate) return vector_ok ? run_rows<G, T, true, true>(a, stream) : run_rows<G, T, false, true>(a, stream);
    return vector_ok ? run_rows<G, T, true, false>(a, stream) : run_rows<G, T, false, false>(a, stream);
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
    const int gradient_bytes = gradient_kind == 0 ? 4 : 2, table_bytes = table_kind == 0 ? 4 : 2;
    if (!aligned_for(out_gradient, gradient_bytes) || !aligned_for(table_gradient, table_bytes) ||
        !aligned_for(tokens, token_bytes) || !aligned_for(token_status, 4) || !workspace || !aligned_for(workspace, 16) ||
        workspace_bytes < s.bytes)
        return static_cast<int>(cudaErrorInvalidValue);
    if (count == 0 && accumulate) return static_cast<int>(cudaSuccess);
    const DeviceScope scope(device);
    if (scope.status() != cudaSuccess) return scope.status();
    char* scratch = static_cast<char*>(workspace);
    SortArguments sort{};
    sort.tokens = Tokens{tokens, token_bytes, padding_token, vocab};
    for (int i = 0; i < 2; ++i) sort.pairs[i] = reinterpret_cast<uint2*>(scratch + s.pairs[i]);
    sort.crossing = reinterpret_cast<unsigned*>(scratch + s.crossing);
    sort.status = token_status;
    // A quarter of the zeros, 128 MB at most, is left to the rows and join launches, which have their own short waits.
    const long long row_bytes = static_cast<long long>(width) * table_bytes;
    long long late_rows = kLateBytes / row_bytes < vocab / 4 ? kLateBytes / row_bytes : vocab / 4;
    if (accumulate || count == 0) late_rows = 0;
    if (late_rows > 0) sort.named = reinterpret_cast<unsigned*>(scratch + s.named);
    sort.clear = static_cast<char*>(table_gradient);
    sort.clear_bytes = accumulate ? 0 : (vocab - late_rows) * row_bytes;
    sort.count = static_cast<unsigned>(count);
    cudaError_t e = launch_sort(sort, stream);
    if (e != cudaSuccess || count == 0) return static_cast<int>(e);
    RowsArguments a{};
    a.pairs = sort.pairs[0];
    a.crossing = sort.crossing;
    a.crossing_short = reinterpret_cast<unsigned*>(scratch + s.crossing_short);
    a.crossing_long = reinterpret_cast<unsigned*>(scratch + s.crossing_long);
    a.rows_short = reinterpret_cast<unsigned*>(scratch + s.pairs[1]);    // chunks + chunks / 16 + 1 of them: less than pairs
    a.rows_long = a.rows_short + s.chunks;
    a.tails = reinterpret_cast<float*>(scratch + s.tails);
    a.heads = reinterpret_cast<float*>(scratch + s.heads);
    a.gradient = out_gradient;
    a.table = table_gradient;
    a.gradient_stride = gradient_stride;
    a.count = static_cast<unsigned>(count);
    a.vocab = static_cast<unsigned>(vocab);
    a.chunks = static_cast<unsigned>(s.chunks);
    a.width = width;
    a.scale = scale;
    a.accumulate = accumulate != 0;
    a.named = sort.named;
    a.late = vocab - late_rows;
    a.late_groups = static_cast<unsigned>((late_rows + kZeroRows - 1) / kZeroRows);
    a.chunk = static_cast<unsigned>(s.chunk);
    const bool vector_ok = width % 8 == 0 && aligned_for(out_gradient, 16) && gradient_stride * gradient_bytes % 16 == 0 &&
                           aligned_for(table_gradient, 16);
    if (gradient_kind == 0)
        e = table_kind == 0 ? run_rows<float, float>(a, vector_ok, stream) : run_rows<float, unsigned short>(a, vector_ok, stream);
    else
        e = table_kind == 0 ? run_rows<unsigned short, float>(a, vector_ok, stream)
                            : run_rows<unsigned short, unsigned short>(a, vector_ok, stream);
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
