// Tokens sorted by expert and back, with their gradients, and the router's (include/kadan_amd.h).
// The reference goes from expert to expert on the host (MoeLayer::forward,
// IW/src/models/text/qwen_layers.cpp:378-492; IW = services/hikari/inference_worker) and has no
// gradients.
//
//   sort_kernel            rows[p] = x[perm[p] / top_k], place[perm[p]] = p, by positions
//   place_kernel, spread_kernel   the same by tokens (-1 for a slot that perm does not name)
//   combine_kernel         y[t] = residual[t] + sum_i w[t, i] rows[place[t top_k + i]]; without
//                          weights the gradient of sorting
//   combine_grad_kernel    drows[place] = w dy, dw = dy . rows[place]
//   inverse_kernel, zero_kernel   zeros in the rows of drows that no place names
//   route_grad_kernel      dlogits of the renormalised weights of the selection
//
// All of them move memory: a value costs a few operations at most, and up to a few hundred tokens
// a call is its launch.  A lane moves 16 bytes at a time (32 where types differ), from any element
// on: gfx950 loads need no alignment beyond it.  Times below are of single MI355X cards, whose
// 1 GB copy runs at 5.2 TB/s and whose reads alone at 7.  Stores keep the caches' default policy:
// streaming ones shorten what follows where that reads something else (combining 32768 rows of
// 2048 bf16 values and back 90 -> 77 us) and lengthen it where it reads the rows, as the experts'
// products do (back and the down product's gradient 173 -> 183).
#include "kdq_common.hpp"

#include <algorithm>

namespace kdq {
namespace {

constexpr unsigned kThreads = 256, kMost = 8;  // selections of a token

struct Bf16 {
    uint16_t bits;
};
struct F16 {
    uint16_t bits;
};

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float widen(Bf16 v) {
    return __uint_as_float(unsigned(v.bits) << 16);
}
__device__ __forceinline__ float widen(F16 v) {
    return half_hw(v.bits);
}
__device__ __forceinline__ float widen(float v) {
    return v;
}

template <class T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) {
    return v;
}
template <> __device__ __forceinline__ Bf16 narrow<Bf16>(float v) {
    return {__builtin_bit_cast(uint16_t, __bf16(v))};
}
template <> __device__ __forceinline__ F16 narrow<F16>(float v) {
    return {__builtin_bit_cast(uint16_t, _Float16(v))};
}

// N values as they lie, 16 bytes or twice as many.
template <class T, int N> struct Piece {
    u32x4 w[N * sizeof(T) / 16];
};

// Values a lane moves at a time: 16 bytes of the narrower type, so that a wavefront's access is
// whole lines of it.
template <class T, class Y> constexpr int kValues = sizeof(T) == 4 && sizeof(Y) == 4 ? 4 : 8;

template <int N, class T> __device__ __forceinline__ Piece<T, N> load_whole(const T* p) {
    Piece<T, N> v;
#pragma unroll
    for (unsigned i = 0; i < N * sizeof(T) / 16; ++i)
        v.w[i] = load16_a2(reinterpret_cast<const uint8_t*>(p) + 16 * i);
    return v;
}

template <int N, class T> __device__ __forceinline__ void store_whole(T* p, const Piece<T, N>& v) {
#pragma unroll
    for (unsigned i = 0; i < N * sizeof(T) / 16; ++i)
        reinterpret_cast<u32x4_a2*>(p)[i] = u32x4_a2{v.w[i].x, v.w[i].y, v.w[i].z, v.w[i].w};
}

template <int N> __device__ __forceinline__ float value(const Piece<Bf16, N>& v, int i) {
    const unsigned w = v.w[i / 8][i / 2 % 4];
    return __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
}
template <int N> __device__ __forceinline__ float value(const Piece<F16, N>& v, int i) {
    return half_hw((v.w[i / 8][i / 2 % 4] >> (16 * (i % 2))) & 0xffffu);
}
template <int N> __device__ __forceinline__ float value(const Piece<float, N>& v, int i) {
    return __uint_as_float(v.w[i / 4][i % 4]);
}

template <int N> __device__ __forceinline__ void set(Piece<Bf16, N>& v, const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
        v.w[i / 8][i / 2 % 4] =
            __builtin_bit_cast(unsigned, bf16x2{__bf16(f[i]), __bf16(f[i + 1])});
}
template <int N> __device__ __forceinline__ void set(Piece<F16, N>& v, const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
        v.w[i / 8][i / 2 % 4] =
            unsigned(narrow<F16>(f[i]).bits) | unsigned(narrow<F16>(f[i + 1]).bits) << 16;
}
template <int N> __device__ __forceinline__ void set(Piece<float, N>& v, const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        v.w[i / 4][i % 4] = __float_as_uint(f[i]);
}

// A row's values from c on, of which those past its end read as zeros and are not written.
template <int N, class T>
__device__ __forceinline__ Piece<T, N> load_piece(const T* row, unsigned c, unsigned cols) {
    if (c + N <= cols)
        return load_whole<N>(row + c);
    float f[N];
#pragma unroll
    for (unsigned i = 0; i < N; ++i)
        f[i] = c + i < cols ? widen(row[c + i]) : 0.f;
    Piece<T, N> v;
    set(v, f);
    return v;
}

template <int N, class T>
__device__ __forceinline__ void store_piece(T* row, unsigned c, unsigned cols,
                                            const float (&f)[N]) {
    if (c + N <= cols) {
        Piece<T, N> v;
        set(v, f);
        store_whole<N>(row + c, v);
        return;
    }
#pragma unroll
    for (unsigned i = 0; i < N; ++i)
        if (c + i < cols)
            row[c + i] = narrow<T>(f[i]);
}

// From this many bytes of rows on they are written by tokens, in two launches: 32768 rows of 2048
// bf16 values 33.3 us against 38.5 by positions (4.5 TB/s of what has to move, of tensors that are
// not in the caches), 8192 of 2880 (45 MB) 14.2 against 15.5, 8192 of 2048 (32 MB) 11.4 against
// 11.1, 4096 of 2048 (16 MB) 8.5 against 6.7.
constexpr size_t kSpreadBytes = size_t(32) << 20;

// How a launch's workgroups share rows of `cols` values: `across` lanes (a power of two) along a
// row, the others' along further rows.
struct Shape {
    unsigned across, rows, blocks;  // rows of a workgroup, workgroups of a row
};

Shape shape_of(size_t cols, int values) {
    const size_t pieces = (cols + values - 1) / values;
    unsigned across = 1;
    while (across < kThreads && across < pieces)
        across *= 2;
    return {across, kThreads / across, unsigned((pieces + across - 1) / across)};
}

// The inverse of the permutation, -1 for a slot that it does not name.  A workgroup takes kPlaces
// slots through LDS and goes over the whole permutation for them, beside the rows' workgroups: 4
// and 2048 slots of 2880 bf16 values 2.5 and 4.9 us, as without.  Of narrow rows the scan is what
// is seen: 64 values, 4096 slots 4.0 us against 2.5, 16384 6.2, 32768 8.7.  By tokens, which needs
// no scan, those take 7.0 and 7.5, but in two launches, and the second is 3 us of the host.
constexpr unsigned kPlaces = 4096, kOwnPlaces = 32768;

constexpr unsigned places_groups(unsigned slots) {
    return (slots + kPlaces - 1) / kPlaces;
}

// put(value, its index) for each of `count` values, by the workgroup's threads.
template <class F>
__device__ __forceinline__ void for_each(const int32_t* __restrict__ values, unsigned count,
                                         unsigned threads, F&& put) {
    constexpr unsigned kAhead = 4;
    const unsigned turn = kAhead * threads * 4;
    unsigned i0 = 0;
    for (; i0 + turn <= count; i0 += turn) {
        Piece<float, 4> v[kAhead];
#pragma unroll
        for (unsigned i = 0; i < kAhead; ++i)
            v[i] = load_whole<4>(reinterpret_cast<const float*>(values) + i0 +
                                 (i * threads + threadIdx.x) * 4);
#pragma unroll
        for (unsigned i = 0; i < kAhead; ++i)
#pragma unroll
            for (unsigned j = 0; j < 4; ++j)
                put(int32_t(v[i].w[0][j]), i0 + (i * threads + threadIdx.x) * 4 + j);
    }
    int32_t rest[kAhead * 4];
#pragma unroll
    for (unsigned i = 0; i < kAhead * 4; ++i) {
        const unsigned at = i0 + i * threads + threadIdx.x;
        rest[i] = at < count ? values[at] : -1;
    }
#pragma unroll
    for (unsigned i = 0; i < kAhead * 4; ++i)
        put(rest[i], i0 + i * threads + threadIdx.x);  // (negative ones past the last)
}

__device__ __forceinline__ void write_places(const int32_t* __restrict__ perm, unsigned slots,
                                             unsigned first, int32_t* __restrict__ place) {
    __shared__ int32_t at[kPlaces];
    const unsigned mine = min(slots - first, kPlaces);
    for (unsigned s = threadIdx.x; s < mine; s += kThreads)
        at[s] = -1;
    __syncthreads();
    for_each(perm, slots, kThreads, [&](int32_t slot, unsigned p) {
        if (unsigned(slot) < slots && unsigned(slot) - first < mine)
            at[unsigned(slot) - first] = int32_t(p);
    });
    __syncthreads();
    for (unsigned s = threadIdx.x; s < mine; s += kThreads)
        place[first + s] = at[s];
}

// A copy, so bits and no values.  By positions: a row of x is read for each of its places, from
// the caches but for the first time.  The first of the workgroups take the places.
template <class U>
__global__ __launch_bounds__(kThreads) void sort_kernel(const U* __restrict__ x, size_t x_stride,
                                                        unsigned slots, unsigned cols,
                                                        unsigned top_k, Shape s,
                                                        const int32_t* __restrict__ perm,
                                                        U* __restrict__ rows, size_t rows_stride,
                                                        int32_t* __restrict__ place) {
    constexpr unsigned N = kValues<U, U>;
    const unsigned own = places_groups(slots);
    if (blockIdx.x < own) {
        if (blockIdx.y == 0)
            write_places(perm, slots, blockIdx.x * kPlaces, place);
        return;
    }
    const unsigned p = (blockIdx.x - own) * s.rows + threadIdx.x / s.across;
    const unsigned c = (blockIdx.y * s.across + threadIdx.x % s.across) * N;
    if (p >= slots || c >= cols)
        return;
    const unsigned slot = unsigned(perm[p]);
    U* to = rows + size_t(p) * rows_stride + c;
    const bool some = slot < slots;  // (no slot: a row of zeros)
    const U* from = x + size_t(some ? slot / top_k : 0) * x_stride + c;
    if (c + N <= cols) {
        store_whole<N>(to, some ? load_whole<N>(from) : Piece<U, N>{});
    } else {
        for (unsigned i = 0; c + i < cols; ++i)
            to[i] = some ? from[i] : U{};
    }
}

// The same by tokens, once the places are known: a row of x is read once.
__global__ __launch_bounds__(kThreads) void place_kernel(const int32_t* __restrict__ perm,
                                                         unsigned slots,
                                                         int32_t* __restrict__ place) {
    const unsigned p = blockIdx.x * kThreads + threadIdx.x;
    if (p < slots && unsigned(perm[p]) < slots)
        place[perm[p]] = int32_t(p);
}

template <class U>
__global__ __launch_bounds__(kThreads) void spread_kernel(const U* __restrict__ x, size_t x_stride,
                                                          unsigned tokens, unsigned cols,
                                                          unsigned top_k, Shape s,
                                                          const int32_t* __restrict__ perm,
                                                          int32_t* place, U* __restrict__ rows,
                                                          size_t rows_stride) {
    constexpr unsigned N = kValues<U, U>;
    const unsigned t = blockIdx.x * s.rows + threadIdx.x / s.across;
    const unsigned c = (blockIdx.y * s.across + threadIdx.x % s.across) * N;
    if (t >= tokens || c >= cols)
        return;
    const unsigned slots = tokens * top_k;
    const bool whole = c + N <= cols;
    const U* from = x + size_t(t) * x_stride + c;
    Piece<U, N> v;
    if (whole)
        v = load_whole<N>(from);
    bool holes = false;
    for (unsigned i = 0; i < top_k; ++i) {
        const unsigned slot = t * top_k + i, p = unsigned(place[slot]);
        holes |= unsigned(perm[slot]) >= slots;
        if (p >= slots || unsigned(perm[p]) != slot) {  // a slot that perm does not name
            if (c == 0)
                place[slot] = -1;  // (another lane finds either value to be none)
            continue;
        }
        U* to = rows + size_t(p) * rows_stride + c;
        if (whole) {
            store_whole<N>(to, v);
        } else {
            for (unsigned j = 0; c + j < cols; ++j)
                to[j] = from[j];
        }
    }
    if (holes) [[unlikely]]  // entries that are no slot: rows of zeros
        for (unsigned p = t * top_k; p < (t + 1) * top_k; ++p)
            if (unsigned(perm[p]) >= slots) {
                U* to = rows + size_t(p) * rows_stride + c;
                if (whole) {
                    store_whole<N>(to, Piece<U, N>{});
                } else {
                    for (unsigned j = 0; c + j < cols; ++j)
                        to[j] = U{};
                }
            }
}

// Sums in fp32, in the order of the selection, and one rounding.  Every row of a token is asked for
// at once.  32768 rows of 2048 bf16 values to 4096 tokens 33 us (4.6 TB/s), with weights and a
// residual 43 (3.9), of tensors that are not in the caches; a few tokens 3.4 us, the launch and two
// loads, one behind the other.
template <class T, class Y>
__global__ __launch_bounds__(kThreads) void combine_kernel(
    const T* __restrict__ rows, size_t rows_stride, const int32_t* __restrict__ place,
    const float* __restrict__ weights, unsigned tokens, unsigned top_k, unsigned cols, Shape s,
    const Y* residual, size_t residual_stride, Y* y, size_t y_stride) {
    constexpr int N = kValues<T, Y>;
    const unsigned t = blockIdx.x * s.rows + threadIdx.x / s.across;
    const unsigned c = (blockIdx.y * s.across + threadIdx.x % s.across) * N;
    if (t >= tokens || c >= cols)
        return;
    const unsigned slots = tokens * top_k;
    unsigned at[kMost];
    float w[kMost];
#pragma unroll
    for (unsigned i = 0; i < kMost; ++i)
        if (i < top_k) {
            at[i] = unsigned(place[t * top_k + i]);
            w[i] = weights ? weights[t * top_k + i] : 1.0f;
        }
    Piece<T, N> v[kMost];
#pragma unroll
    for (unsigned i = 0; i < kMost; ++i)
        if (i < top_k && at[i] < slots)
            v[i] = load_piece<N>(rows + size_t(at[i]) * rows_stride, c, cols);
    float sum[N] = {};
    if (residual) {
        const Piece<Y, N> r = load_piece<N>(residual + size_t(t) * residual_stride, c, cols);
#pragma unroll
        for (int e = 0; e < N; ++e)
            sum[e] = value(r, e);
    }
#pragma unroll
    for (unsigned i = 0; i < kMost; ++i)
        if (i < top_k && at[i] < slots)
#pragma unroll
            for (int e = 0; e < N; ++e)
                sum[e] = fmaf(w[i], value(v[i], e), sum[e]);
    store_piece<N>(y + size_t(t) * y_stride, c, cols, sum);
}

// Zeros in every row from `first` on whose lane asks for them, by the whole wavefront.
template <class T>
__device__ __forceinline__ void zero_rows(bool mine, unsigned first, unsigned cols, T* rows,
                                          size_t stride) {
    constexpr int N = kValues<T, T>;
    const float zeros[N] = {};
    for (uint64_t left = __builtin_amdgcn_ballot_w64(mine); left; left &= left - 1) {
        T* row = rows + size_t(first + unsigned(__builtin_ctzll(left))) * stride;
        for (unsigned c = threadIdx.x % 64 * N; c < cols; c += 64 * N)
            store_piece<N>(row, c, cols, zeros);
    }
}

// Rows of drows that no place names (as many as selections are dropped) get zeros.  Up to
// kMostMarked slots this is the tokens' launch: a workgroup goes over all the places and marks
// which of its kMarked positions they name.  20 slots of 2880 bf16 values 6.0 us against 5.3
// without, 4096 of 2048 10.0 against 9.1, 16384 of 512 14.2 against 9.1, in three launches 12.9 and
// 6 us more of the host; 32768 of 2048 in three launches 51 against 47, in one 57.
constexpr unsigned kMarked = 64, kMostMarked = 16384;

template <class T>
__device__ __forceinline__ void zero_unnamed(const int32_t* __restrict__ place, unsigned slots,
                                             unsigned first, unsigned cols, T* drows,
                                             size_t drows_stride) {
    __shared__ uint8_t named[kMarked];
    if (threadIdx.x < kMarked)
        named[threadIdx.x] = 0;
    __syncthreads();
    for_each(place, slots, blockDim.x, [&](int32_t p, unsigned) {
        if (unsigned(p) < slots && unsigned(p) - first < kMarked)
            named[unsigned(p) - first] = 1;
    });
    __syncthreads();
    const unsigned waves = blockDim.x / 64, share = (kMarked + waves - 1) / waves;
    const unsigned lane = threadIdx.x % 64, at = threadIdx.x / 64 * share;
    zero_rows(lane < share && at + lane < kMarked && first + at + lane < slots && !named[at + lane],
              first + at, cols, drows, drows_stride);
}

// The same ahead of the tokens' launch, by the places' inverse, which goes where the weights'
// gradients will be.  It needs no clearing: what is left there of another use does not lead back.
// A wavefront takes kZeroed positions.
constexpr unsigned kZeroed = 8;

__global__ __launch_bounds__(kThreads) void inverse_kernel(const int32_t* __restrict__ place,
                                                           unsigned slots,
                                                           int32_t* __restrict__ slot) {
    const unsigned s = blockIdx.x * kThreads + threadIdx.x;
    if (s < slots && unsigned(place[s]) < slots)
        slot[place[s]] = int32_t(s);
}

template <class T>
__global__ __launch_bounds__(kThreads) void zero_kernel(const int32_t* __restrict__ place,
                                                        const int32_t* __restrict__ slot,
                                                        unsigned slots, unsigned cols,
                                                        T* __restrict__ drows,
                                                        size_t drows_stride) {
    const unsigned lane = threadIdx.x % 64;
    const unsigned first = (blockIdx.x * kThreads + threadIdx.x) / 64 * kZeroed, p = first + lane;
    const bool mine = lane < kZeroed && p < slots;
    const unsigned of = mine ? unsigned(slot[p]) : 0;
    zero_rows(mine && (of >= slots || unsigned(place[of]) != p), first, cols, drows, drows_stride);
}

// A workgroup takes a token: its dy is read once for all of its rows, and one pass over those gives
// both gradients; dot products are summed lane by lane, then over lanes and wavefronts in their
// order, so results do not depend on the run.  32768 rows of 2048 bf16 values 48 us (6.0 TB/s).
template <class T, class Y, bool ZEROES>
__global__ __launch_bounds__(kThreads) void combine_grad_kernel(
    const T* __restrict__ rows, size_t rows_stride, const Y* __restrict__ dy, size_t dy_stride,
    const int32_t* __restrict__ place, const float* __restrict__ weights, unsigned tokens,
    unsigned top_k, unsigned cols, T* __restrict__ drows, size_t drows_stride,
    float* __restrict__ dweights) {
    constexpr int N = kValues<T, Y>;
    __shared__ float sums[kThreads / 64][kMost];
    const unsigned slots = tokens * top_k;
    const unsigned zeroing = ZEROES ? (slots + kMarked - 1) / kMarked : 0;
    if (blockIdx.x < zeroing) {  // (the first, so that none is waited for in the end)
        zero_unnamed(place, slots, blockIdx.x * kMarked, cols, drows, drows_stride);
        return;
    }
    const unsigned t = blockIdx.x - zeroing;
    const unsigned lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    unsigned at[kMost];
    float w[kMost], dot[kMost] = {};
#pragma unroll
    for (unsigned i = 0; i < kMost; ++i)
        if (i < top_k) {
            at[i] = unsigned(place[t * top_k + i]);
            w[i] = weights[t * top_k + i];
        }
    for (unsigned c = threadIdx.x * N; c < cols; c += blockDim.x * N) {
        const Piece<Y, N> d = load_piece<N>(dy + size_t(t) * dy_stride, c, cols);
        Piece<T, N> v[kMost];
#pragma unroll
        for (unsigned i = 0; i < kMost; ++i)
            if (i < top_k && at[i] < slots)
                v[i] = load_piece<N>(rows + size_t(at[i]) * rows_stride, c, cols);
#pragma unroll
        for (unsigned i = 0; i < kMost; ++i)
            if (i < top_k && at[i] < slots) {
                float f[N];
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float g = value(d, e);
                    dot[i] = fmaf(g, value(v[i], e), dot[i]);
                    f[e] = w[i] * g;
                }
                store_piece<N>(drows + size_t(at[i]) * drows_stride, c, cols, f);
            }
    }
#pragma unroll
    for (unsigned i = 0; i < kMost; ++i)
        if (i < top_k) {
            const float sum = wave_sum(dot[i]);
            if (lane == 0)
                sums[wave][i] = sum;
        }
    __syncthreads();
    if (threadIdx.x < top_k) {
        float sum = 0.f;
        for (unsigned i = 0; i < blockDim.x / 64; ++i)
            sum += sums[i][threadIdx.x];
        dweights[t * top_k + threadIdx.x] = sum;
    }
}

// w = softmax over the selected logits, so dlogit = w (dw - sum w dw) there and 0 elsewhere.  A
// wavefront takes a token: lane i its selection i, then lanes go along the experts.  4096 tokens of
// 128 experts 3.7 us, of which 2.5 are the launch.
__global__ __launch_bounds__(kThreads) void route_grad_kernel(
    const int32_t* __restrict__ idx, const float* __restrict__ weights,
    const float* __restrict__ dweights, unsigned tokens, unsigned experts, unsigned top_k,
    float* __restrict__ dlogits) {
    const unsigned t = blockIdx.x * (kThreads / 64) + threadIdx.x / 64, lane = threadIdx.x % 64;
    if (t >= tokens)
        return;
    const bool chosen = lane < top_k;
    const int e = chosen ? idx[t * top_k + lane] : -1;
    const float w = chosen ? weights[t * top_k + lane] : 0.f;
    const float d = chosen ? dweights[t * top_k + lane] : 0.f;
    float sum = w * d;  // (of lanes 0 to 7, in every one of them)
#pragma unroll
    for (int offset = 4; offset > 0; offset >>= 1)
        sum += __shfl_xor(sum, offset, 64);
    const float g = w * (d - sum);
    for (unsigned c = lane; c < experts; c += 64) {
        float out = 0.f;
#pragma unroll
        for (unsigned i = 0; i < kMost; ++i)
            if (i < top_k &&
                unsigned(__builtin_amdgcn_readlane(e, int(i))) == c)
                out = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), int(i)));
        dlogits[size_t(t) * experts + c] = out;
    }
}

// ------------------------------------------------------------------ arguments

constexpr size_t kMaxTokens = size_t(1) << 20, kMaxCols = size_t(1) << 20;

size_t size_of(int type) {
    return type == KDQ_F32 ? 4 : type == KDQ_F16 || type == KDQ_BF16 ? 2 : 0;
}

// Rows of a call: their bytes from the first value to the last.
struct Rows {
    const void* p;
    size_t stride, count;
    int type;
    size_t bytes(size_t cols) const {
        return ((count - 1) * stride + cols) * size_of(type);
    }
};

int check_sizes(size_t tokens, size_t top_k, size_t cols) {
    if (!tokens || !top_k || !cols)
        return KDQ_ERR_ARGUMENT;
    return tokens > kMaxTokens || top_k > kMost || cols > kMaxCols ? KDQ_ERR_SHAPE : KDQ_OK;
}

int check_rows(const Rows& r, size_t cols) {
    if (!size_of(r.type))
        return KDQ_ERR_UNSUPPORTED;
    if (r.stride < cols || r.stride > (SIZE_MAX >> 4) / r.count)
        return KDQ_ERR_SHAPE;
    return misaligned(r.p, size_of(r.type)) ? KDQ_ERR_ALIGNMENT : KDQ_OK;
}

int check_words(const void* p) {
    return misaligned(p, 4) ? KDQ_ERR_ALIGNMENT : KDQ_OK;
}

#define KDQ_TRY(check)              \
    do {                            \
        if (const int rc_ = (check)) \
            return rc_;             \
    } while (0)

// f with a value of the C++ type of `type`, and (two types) one of the second: the first's or
// fp32.
template <class F> int by_type(int type, F&& f) {
    switch (type) {
    case KDQ_BF16:
        return f(Bf16{});
    case KDQ_F16:
        return f(F16{});
    default:
        return f(0.f);
    }
}

template <class F> int by_types(int type, int second, F&& f) {
    return by_type(type, [&](auto t) {
        return second == type ? f(t, t) : f(t, 0.f);
    });
}

int combine(const Rows& rows, const int32_t* place, const float* weights, size_t tokens,
            size_t top_k, size_t cols, const Rows& residual, const Rows& y, hipStream_t st) {
    return by_types(rows.type, y.type, [&](auto t, auto u) {
        using T = decltype(t);
        using Y = decltype(u);
        const Shape s = shape_of(cols, kValues<T, Y>);
        hipLaunchKernelGGL((combine_kernel<T, Y>),
                           dim3(unsigned((tokens + s.rows - 1) / s.rows), s.blocks),
                           dim3(kThreads), 0, st, static_cast<const T*>(rows.p), rows.stride,
                           place, weights, unsigned(tokens), unsigned(top_k), unsigned(cols), s,
                           static_cast<const Y*>(residual.p), residual.stride,
                           static_cast<Y*>(const_cast<void*>(y.p)), y.stride);
        KDQ_HIP(hipGetLastError());
        return int(KDQ_OK);
    });
}
}  // namespace
}  // namespace kdq

using namespace kdq;

extern "C" int kdq_moe_sort(int type, const void* x, size_t x_stride, size_t tokens, size_t cols,
                            size_t top_k, const int32_t* perm, void* rows, size_t rows_stride,
                            int32_t* place, void* stream) {
    if (!x || !perm || !rows || !place)
        return KDQ_ERR_ARGUMENT;
    KDQ_TRY(check_sizes(tokens, top_k, cols));
    const size_t slots = tokens * top_k;
    const Rows in{x, x_stride, tokens, type}, out{rows, rows_stride, slots, type};
    KDQ_TRY(check_rows(in, cols));
    KDQ_TRY(check_rows(out, cols));
    KDQ_TRY(check_words(perm));
    KDQ_TRY(check_words(place));
    const Range to[] = {{rows, out.bytes(cols)}, {place, slots * 4}},
                from[] = {{x, in.bytes(cols)}, {perm, slots * 4}};
    if (any_overlap(to, from))
        return KDQ_ERR_ALIAS;
    const auto st = static_cast<hipStream_t>(stream);
    const auto launch = [&](auto u) {
        using U = decltype(u);
        const Shape s = shape_of(cols, kValues<U, U>);
        const auto blocks = [&](size_t count) {
            return dim3(unsigned((count + s.rows - 1) / s.rows), s.blocks);
        };
        if (slots > kOwnPlaces || (top_k > 1 && slots * cols * size_of(type) >= kSpreadBytes)) {
            hipLaunchKernelGGL(place_kernel, dim3(unsigned((slots + kThreads - 1) / kThreads)),
                               dim3(kThreads), 0, st, perm, unsigned(slots), place);
            hipLaunchKernelGGL(spread_kernel<U>, blocks(tokens), dim3(kThreads), 0, st,
                               static_cast<const U*>(x), x_stride, unsigned(tokens),
                               unsigned(cols), unsigned(top_k), s, perm, place,
                               static_cast<U*>(rows), rows_stride);
        } else {
            dim3 grid = blocks(slots);
            grid.x += places_groups(unsigned(slots));
            hipLaunchKernelGGL(sort_kernel<U>, grid, dim3(kThreads), 0, st,
                               static_cast<const U*>(x), x_stride, unsigned(slots),
                               unsigned(cols), unsigned(top_k), s, perm, static_cast<U*>(rows),
                               rows_stride, place);
        }
        KDQ_HIP(hipGetLastError());
        return int(KDQ_OK);
    };
    return type == KDQ_F32 ? launch(0.f) : launch(Bf16{});
}

extern "C" int kdq_moe_sort_backward(int type, const void* drows, size_t drows_stride,
                                     const int32_t* place, size_t tokens, size_t cols,
                                     size_t top_k, void* dx, size_t dx_stride, void* stream) {
    if (!drows || !place || !dx)
        return KDQ_ERR_ARGUMENT;
    KDQ_TRY(check_sizes(tokens, top_k, cols));
    const size_t slots = tokens * top_k;
    const Rows in{drows, drows_stride, slots, type}, out{dx, dx_stride, tokens, type};
    KDQ_TRY(check_rows(in, cols));
    KDQ_TRY(check_rows(out, cols));
    KDQ_TRY(check_words(place));
    const Range to[] = {{dx, out.bytes(cols)}},
                from[] = {{drows, in.bytes(cols)}, {place, slots * 4}};
    if (any_overlap(to, from))
        return KDQ_ERR_ALIAS;
    return combine(in, place, nullptr, tokens, top_k, cols, Rows{}, out,
                   static_cast<hipStream_t>(stream));
}

extern "C" int kdq_moe_combine(int type, const void* rows, size_t rows_stride,
                               const int32_t* place, const float* weights, size_t tokens,
                               size_t cols, size_t top_k, int y_type, const void* residual,
                               size_t residual_stride, void* y, size_t y_stride, void* stream) {
    if (!rows || !place || !weights || !y)
        return KDQ_ERR_ARGUMENT;
    KDQ_TRY(check_sizes(tokens, top_k, cols));
    if (y_type != type && y_type != KDQ_F32)
        return KDQ_ERR_UNSUPPORTED;
    const size_t slots = tokens * top_k;
    const Rows in{rows, rows_stride, slots, type}, out{y, y_stride, tokens, y_type},
        add{residual, residual ? residual_stride : cols, tokens, y_type};
    KDQ_TRY(check_rows(in, cols));
    KDQ_TRY(check_rows(out, cols));
    KDQ_TRY(check_rows(add, cols));
    KDQ_TRY(check_words(place));
    KDQ_TRY(check_words(weights));
    // (y may be the residual itself: a lane reads what it then writes)
    const bool in_place = residual == y && residual_stride == y_stride;
    const Range to[] = {{y, out.bytes(cols)}},
                from[] = {{rows, in.bytes(cols)},
                          {place, slots * 4},
                          {weights, slots * 4},
                          {in_place ? nullptr : residual, add.bytes(cols)}};
    if (any_overlap(to, from))
        return KDQ_ERR_ALIAS;
    return combine(in, place, weights, tokens, top_k, cols, add, out,
                   static_cast<hipStream_t>(stream));
}

extern "C" int kdq_moe_combine_backward(int type, const void* rows, size_t rows_stride,
                                        const int32_t* place, const float* weights, size_t tokens,
                                        size_t cols, size_t top_k, int dy_type, const void* dy,
                                        size_t dy_stride, void* drows, size_t drows_stride,
                                        float* dweights, void* stream) {
    if (!rows || !place || !weights || !dy || !drows || !dweights)
        return KDQ_ERR_ARGUMENT;
    KDQ_TRY(check_sizes(tokens, top_k, cols));
    if (dy_type != type && dy_type != KDQ_F32)
        return KDQ_ERR_UNSUPPORTED;
    const size_t slots = tokens * top_k;
    const Rows in{rows, rows_stride, slots, type}, of{dy, dy_stride, tokens, dy_type},
        out{drows, drows_stride, slots, type};
    KDQ_TRY(check_rows(in, cols));
    KDQ_TRY(check_rows(of, cols));
    KDQ_TRY(check_rows(out, cols));
    for (const void* p : {static_cast<const void*>(place), static_cast<const void*>(weights),
                          static_cast<const void*>(dweights)})
        KDQ_TRY(check_words(p));
    const Range to[] = {{drows, out.bytes(cols)}, {dweights, slots * 4}},
                from[] = {{rows, in.bytes(cols)},
                          {dy, of.bytes(cols)},
                          {place, slots * 4},
                          {weights, slots * 4}};
    if (any_overlap(to, from))
        return KDQ_ERR_ALIAS;
    const unsigned threads = unsigned(std::min<size_t>(kThreads, (cols + 511) / 512 * 64));
    return by_types(type, dy_type, [&](auto t, auto u) {
        using T = decltype(t);
        using Y = decltype(u);
        const auto st = static_cast<hipStream_t>(stream);
        const bool marked = slots <= kMostMarked;
        const unsigned zeroing = marked ? unsigned((slots + kMarked - 1) / kMarked) : 0;
        if (!marked) {
            auto* slot = reinterpret_cast<int32_t*>(dweights);
            const auto grid = [&](unsigned each) {  // positions of a workgroup
                return dim3(unsigned((slots + each - 1) / each));
            };
            hipLaunchKernelGGL(inverse_kernel, grid(kThreads), dim3(kThreads), 0, st, place,
                               unsigned(slots), slot);
            hipLaunchKernelGGL(zero_kernel<T>, grid(kThreads / 64 * kZeroed), dim3(kThreads), 0,
                               st, place, slot, unsigned(slots), unsigned(cols),
                               static_cast<T*>(drows), drows_stride);
        }
        const auto kernel =
            marked ? combine_grad_kernel<T, Y, true> : combine_grad_kernel<T, Y, false>;
        hipLaunchKernelGGL(kernel, dim3(unsigned(tokens) + zeroing), dim3(threads), 0, st,
                           static_cast<const T*>(rows), rows_stride, static_cast<const Y*>(dy),
                           dy_stride, place, weights, unsigned(tokens), unsigned(top_k),
                           unsigned(cols), static_cast<T*>(drows), drows_stride, dweights);
        KDQ_HIP(hipGetLastError());
        return int(KDQ_OK);
    });
}

extern "C" int kdq_moe_route_backward(const int32_t* idx, const float* weights,
                                      const float* dweights, size_t tokens, size_t experts,
                                      size_t top_k, float* dlogits, void* stream) {
    if (!idx || !weights || !dweights || !dlogits || !experts)
        return KDQ_ERR_ARGUMENT;
    KDQ_TRY(check_sizes(tokens, top_k, experts));
    if (experts > 256 || top_k > experts)
        return KDQ_ERR_SHAPE;
    for (const void* p : {static_cast<const void*>(idx), static_cast<const void*>(weights),
                          static_cast<const void*>(dweights), static_cast<const void*>(dlogits)})
        KDQ_TRY(check_words(p));
    const size_t bytes = tokens * top_k * 4;
    const Range to[] = {{dlogits, tokens * experts * 4}},
                from[] = {{idx, bytes}, {weights, bytes}, {dweights, bytes}};
    if (any_overlap(to, from))
        return KDQ_ERR_ALIAS;
    hipLaunchKernelGGL(route_grad_kernel, dim3(unsigned((tokens + 3) / 4)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), idx, weights, dweights, unsigned(tokens),
                       unsigned(experts), unsigned(top_k), dlogits);
    KDQ_HIP(hipGetLastError());
    return KDQ_OK;
}
