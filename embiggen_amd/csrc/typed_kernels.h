// Products of rows with the weights of their type (node / edge types of a graph, or the adapters of a
// batch of requests): y[r] = x[r] W[t_r] + b[t_r], the low-rank form y[r] = x[r] W + b + (x[r] A[t_r])
// B[t_r], and the gradients of both.  float32 and bfloat16 rows, every sum in float32.
//
// Rows are worked on in the order of their types (a stable counting sort: the plan), through their
// row ids, so that no sorted copy of the rows exists: a tile is up to 64 rows of ONE type, gathered,
// and a type's weights are an ordinary right operand.  MFMA operands are exchanged (C^T = W^T x^T): a
// lane then holds four consecutive output columns of one row and stores them in one instruction.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gn2v {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 64;     // rows of a product tile
constexpr int kMaxTypes = 32768;  // the plan counts the types in LDS: 128 KB
constexpr int kSmallPlan = 512;   // rows one workgroup sorts in LDS

// ------------------------------------------------------------------------------------ the plan
// int32 words: order[rows] (row id at every position), row_types[rows] (type at every position;
// n_types = unknown: any id outside [0, n_types); those rows come last), offsets[n_types + 2]
// (first position of every type, of the unknown rows, rows), tile_first[n_types + 2] (the same in
// tiles: a type of c rows has ceil(c / 64) of them).
struct PlanView {
    int *order, *row_types, *offsets, *tile_first;
    uint32_t rows, types;
};

template <typename I>
__device__ __forceinline__ int type_at(const I *types, uint32_t row, uint32_t n_types) {
    const I t = types[row];
    return t >= 0 && (uint64_t)t < (uint64_t)n_types ? (int)t : (int)n_types;
}

// Up to 512 rows: one workgroup sorts (type << 10 | row) in LDS -- one launch, bound by the sort's
// barriers (64 rows 6 us, 512 rows 10 us: as long as the three launches below).
template <typename I>
__global__ __launch_bounds__(kSmallPlan) void plan_small_kernel(const I *__restrict__ types, PlanView p) {
    __shared__ uint32_t key[kSmallPlan];
    __shared__ int tiles[kSmallPlan + 1];  // tile starts before every position
    __shared__ int wave_sum[kSmallPlan / 64];
    const uint32_t i = threadIdx.x;
    key[i] = i < p.rows ? (uint32_t)type_at(types, i, p.types) << 10 | i : 0xFFFFFFFFu;
    uint32_t n = 64;  // the sort covers the smallest power of two
    while (n < p.rows) n <<= 1;
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (uint32_t step = size >> 1; step; step >>= 1) {
            __syncthreads();
            const uint32_t j = i ^ step;
            if (i < n && j > i) {
                const uint32_t a = key[i], b = key[j];
                if ((a > b) == ((i & size) == 0)) {
                    key[i] = b;
                    key[j] = a;
                }
            }
        }
    __syncthreads();
    auto first_of = [&](uint32_t type) {  // positions of smaller types
        uint32_t lo = 0, hi = p.rows;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (key[mid] >> 10 < type)
                lo = mid + 1;
            else
                hi = mid;
        }
        return lo;
    };
    bool starts = false;
    if (i < p.rows) {
        const uint32_t type = key[i] >> 10;
        p.order[i] = (int)(key[i] & 1023u);
        p.row_types[i] = (int)type;
        starts = (i - first_of(type)) % kTileRows == 0;
    }
    const unsigned long long ballot = __ballot(starts);
    if ((i & 63) == 0) wave_sum[i >> 6] = __popcll(ballot);
    __syncthreads();
    int at = __popcll(ballot & ((1ull << (i & 63)) - 1));
    for (uint32_t w = 0; w < i >> 6; ++w) at += wave_sum[w];
    tiles[i] = at;
    if (i == kSmallPlan - 1) tiles[kSmallPlan] = at + starts;
    __syncthreads();
    for (uint32_t t = i; t < p.types + 2; t += kSmallPlan) {
        const uint32_t first = t <= p.types ? first_of(t) : p.rows;
        p.offsets[t] = (int)first;
        p.tile_first[t] = tiles[first];
    }
}

// More rows: a workgroup per stripe of rows counts its types in LDS; the counts of the stripes before
// it and of the smaller types say where its rows go.  Equal types keep their rows' order (a wave
// takes a part of the stripe in order and ranks 64 rows at a time by ballots over the bits of their
// types), so sums over a type's rows have the same order in every run.  Three launches of latency: 169 343
// rows of 40 types 12 us, 1 M rows of 20 types 19 us (its 8 bytes read and 8 written a row: 3 us).
template <typename I>
__global__ __launch_bounds__(256) void plan_count_kernel(const I *__restrict__ types, uint32_t rows,
                                                         uint32_t n_types, uint32_t stripe,
                                                         int *__restrict__ counts) {
    extern __shared__ int count[];
    for (uint32_t t = threadIdx.x; t <= n_types; t += blockDim.x) count[t] = 0;
    __syncthreads();
    const uint64_t first = (uint64_t)blockIdx.x * stripe;
    const uint64_t last = first + stripe < rows ? first + stripe : rows;
    for (uint64_t r = first + threadIdx.x; r < last; r += blockDim.x)
        atomicAdd(&count[type_at(types, (uint32_t)r, n_types)], 1);
    __syncthreads();
    for (uint32_t t = threadIdx.x; t <= n_types; t += blockDim.x)
        counts[(uint64_t)t * gridDim.x + blockIdx.x] = count[t];
}

// counts[type][stripe] -> sums over the stripes before; totals[type].  A wave per type, kStripes
// counts at most.
constexpr uint32_t kStripes = 1024;
__global__ __launch_bounds__(256) void plan_scan_kernel(int *__restrict__ counts, uint32_t stripes,
                                                        uint32_t groups, int *__restrict__ totals) {
    constexpr int N = kStripes / 64;
    const uint32_t t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= groups) return;
    const int lane = threadIdx.x & 63;
    int *row = counts + (uint64_t)t * stripes, own[N], carry = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) own[i] = 64u * i + lane < stripes ? row[64 * i + lane] : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (64u * i >= stripes) break;
        int sum = own[i];
        for (int step = 1; step < 64; step <<= 1) {
            const int other = __shfl_up(sum, step);
            if (lane >= step) sum += other;
        }
        if (64u * i + lane < stripes) row[64 * i + lane] = carry + sum - own[i];
        carry += __shfl(sum, 63);
    }
    if (lane == 0) totals[t] = carry;
}

// LDS: next[parts][n_types + 1].  The first `parts` waves place rows, all of them sum over the types.
template <typename I>
__global__ __launch_bounds__(1024) void plan_place_kernel(const I *__restrict__ types, PlanView p,
                                                          uint32_t stripe, uint32_t stripes,
                                                          const int *__restrict__ counts, int bits,
                                                          const int *__restrict__ totals, uint32_t parts) {
    extern __shared__ int next[];
    __shared__ int sums[2][16];
    const uint32_t groups = p.types + 1, threads = blockDim.x, waves = threads >> 6;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t t = threadIdx.x; t < groups * parts; t += threads) next[t] = 0;
    __syncthreads();
    // the rows of the wave's own part of the stripe
    const uint64_t first = (uint64_t)blockIdx.x * stripe;
    const uint64_t last = first + stripe < p.rows ? first + stripe : p.rows;
    const uint32_t part = ((stripe + parts - 1) / parts + 63) / 64 * 64;
    const uint64_t from = wave < (int)parts ? min(first + (uint64_t)wave * part, last) : last;
    const uint64_t to = min(from + part, last);
    if (parts > 1)
        for (uint64_t r = from + lane; r < to; r += 64)
            atomicAdd(&next[wave * groups + type_at(types, (uint32_t)r, p.types)], 1);
    __syncthreads();
    int carry = 0, carry_tiles = 0;
    for (uint32_t base = 0; base < groups; base += threads) {
        const uint32_t t = base + threadIdx.x;
        int before = 0, total = 0;
        if (t < groups) {
            before = counts[(uint64_t)t * stripes + blockIdx.x];
            total = totals[t];
        }
        const int own_tiles = (int)(((uint32_t)total + kTileRows - 1) / kTileRows);
        int rows = total, tiles = own_tiles;
        for (int step = 1; step < 64; step <<= 1) {
            const int a = __shfl_up(rows, step), b = __shfl_up(tiles, step);
            if (lane >= step) {
                rows += a;
                tiles += b;
            }
        }
        if (lane == 63) {
            sums[0][wave] = rows;
            sums[1][wave] = tiles;
        }
        __syncthreads();
        int start = carry + rows - total, start_tiles = carry_tiles + tiles - own_tiles;
        for (uint32_t w = 0; w < waves; ++w) {
            if ((int)w < wave) {
                start += sums[0][w];
                start_tiles += sums[1][w];
            }
            carry += sums[0][w];
            carry_tiles += sums[1][w];
        }
        if (t < groups) {
            if (blockIdx.x == 0) {
                p.offsets[t] = start;
                p.tile_first[t] = start_tiles;
            }
            int at = start + before;
            for (uint32_t w = 0; w < parts; ++w) {
                const int own = next[w * groups + t];
                next[w * groups + t] = at;
                at += own;
            }
        }
        __syncthreads();
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.offsets[groups] = carry;
        p.tile_first[groups] = carry_tiles;
    }
    // every such wave walks its own part: its counters belong to no other wave
    volatile int *mine = next + wave * groups;
    for (uint64_t base = from; base < to; base += 256) {
        int type4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t r = base + 64 * i + lane;
            type4[i] = r < to ? type_at(types, (uint32_t)r, p.types) : 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t r = base + 64 * i + lane;
            const int type = type4[i];
            const bool live = r < to;
            unsigned long long same = __ballot(live);
            for (int b = 0; b < bits; ++b) {
                const unsigned long long set = __ballot(type >> b & 1);
                same &= type >> b & 1 ? set : ~set;
            }
            const unsigned long long below = same & ((1ull << lane) - 1);
            const int at = live ? mine[type] : 0;
            __builtin_amdgcn_wave_barrier();  // every lane has read its counter
            if (live) {
                p.order[at + __popcll(below)] = (int)r;
                p.row_types[at + __popcll(below)] = type;
                if (below == 0) mine[type] = at + __popcll(same);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// The plan's words at indexes that are uniform in the wave, through the scalar cache: a vector load would
// have to be waited for together with the rows that are being fetched ahead.
__device__ __forceinline__ int plan_word(const int *p, int i) {
    typedef const __attribute__((address_space(4))) int *scalar_ptr;
    return ((scalar_ptr)(uintptr_t)p)[__builtin_amdgcn_readfirstlane(i)];
}

// Where a tile lies: its type, first position, and the position behind its type's last row.
struct TileAt {
    int type, start, end;
    __device__ __forceinline__ int count() const { return min(kTileRows, end - start); }
};

// Tile number `t` (uniform in the wave): 64 lanes look at 64 types at a time.
__device__ __forceinline__ TileAt find_tile(const PlanView &p, int t, int lane) {
    int lo = 0, hi = (int)p.types + 1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) >> 6, i = lo + lane * step;
        const int c = __popcll(__ballot(i < hi && p.tile_first[i < hi ? i : lo] <= t));
        lo += (c - 1) * step;
        hi = min(lo + step, hi);
    }
    TileAt at;
    at.type = __builtin_amdgcn_readfirstlane(lo);
    at.start = plan_word(p.offsets, at.type) + (t - plan_word(p.tile_first, at.type)) * kTileRows;
    at.end = plan_word(p.offsets, at.type + 1);
    return at;
}
// the tile behind it: at the end of a type that of the next type with rows
__device__ __forceinline__ TileAt tile_behind(const PlanView &p, TileAt at) {
    at.start += kTileRows;
    if (at.start >= at.end) {
        at.start = at.end;
        if (at.start < (int)p.rows) {
            at.type = plan_word(p.row_types, at.start);
            at.end = plan_word(p.offsets, at.type + 1);
        }
    }
    return at;
}

// ------------------------------------------------------------------------------- rows and tiles
template <typename T> struct Tile;
template <> struct Tile<float> {
    static constexpr int kChunk = 4;  // elements of 16 bytes
    static constexpr int kDepth = 32; // inner elements per LDS stage: 128 B of a row
    static constexpr int kSlab = 16;  // inner elements per step of MFMAs (four of depth 4)
    static constexpr int kPad = 4;    // row stride 36 words: 16 rows start in 16 different banks
};
template <> struct Tile<__bf16> {
    static constexpr int kChunk = 8;
    static constexpr int kDepth = 64;
    static constexpr int kSlab = 32;  // one MFMA of depth 32
    static constexpr int kPad = 8;
};

// How the 16-byte chunks of a row are loaded, chosen on the host for all rows of an operand: kWhole
// where every row starts on 16 bytes and its length is a multiple of them, kWords where that holds for 4
// bytes, kElements (bfloat16) else.
enum ChunkMode : int { kWhole = 0, kWords = 1, kElements = 2 };

// Elements k .. of a row of `length` elements, zeros behind its end or where the row is not `live`.
// Loads are masked, never corrected afterwards: nothing here waits for what it loads (kElements does),
// so that a caller can fetch ahead.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T *row, int k, int length, int mode, bool live = true) {
    constexpr int E = Tile<T>::kChunk;
    u32x4 v = {0, 0, 0, 0};
    if (!live || k >= length) return v;
    const T *p = row + k;
    const int valid = length - k;
    if (valid >= E) {
        if (mode == kWhole) return *reinterpret_cast<const u32x4 *>(p);
        if (mode == kWords) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = reinterpret_cast<const uint32_t *>(p)[i];
            return v;
        }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < valid) v[i] = __float_as_uint(p[i]);
    } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < valid) v[i >> 1] |= (uint32_t)h[i] << (16 * (i & 1));
    }
    return v;
}

// nearest bfloat16 (ties to even; NaN stays NaN)
__device__ __forceinline__ __bf16 to_bf16(float v) { return (__bf16)v; }

// A float as two bfloat16 parts: its upper half, and what that leaves, rounded to nearest (2^-16 of it left out
// at most).  Where nothing is left, or less than a normal number, the parts are two halves of the upper half: both
// have its sign and neither is zero, so that an infinite factor makes the same infinity of both, not a NaN, and
// their sum is the value.  That holds from 2^-125 on, and the 2^-16 from 2^-110 on; below, 2^-126 of it is left out.
__device__ __forceinline__ void split(float v, __bf16 &high, __bf16 &rest) {
    const float upper = __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
    const float left = v - upper, half = 0.5f * upper;  // exact; `left` is NaN of an infinity
    const bool both = __builtin_fabsf(left) >= 0x1p-126f;
    high = __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(both ? upper : half) >> 16));
    rest = to_bf16(both ? left : half);
}

// four consecutive output elements, `valid` of them inside the row
__device__ __forceinline__ void store4(float *p, f32x4 v, int valid, bool vec) {
    if (vec && valid >= 4) {
        *reinterpret_cast<f32x4 *>(p) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < valid) p[i] = v[i];
}
__device__ __forceinline__ void store4(__bf16 *p, f32x4 v, int valid, bool vec) {
    bf16x4 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = to_bf16(v[i]);
    if (vec && valid >= 4) {
        *reinterpret_cast<bf16x4 *>(p) = h;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < valid) p[i] = h[i];
}

// eight consecutive output elements, `valid` of them inside the row; `align`: bytes the rows are
// aligned to
__device__ __forceinline__ void store8(float *p, const float *v, int valid, int align) {
    store4(p, f32x4{v[0], v[1], v[2], v[3]}, valid, align == 16);
    store4(p + 4, f32x4{v[4], v[5], v[6], v[7]}, valid - 4, align == 16);
}
__device__ __forceinline__ void store8(__bf16 *p, const float *v, int valid, int align) {
    if (align == 16 && valid >= 8) {
        bf16x8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = to_bf16(v[i]);
        *reinterpret_cast<bf16x8 *>(p) = h;
        return;
    }
    store4(p, f32x4{v[0], v[1], v[2], v[3]}, valid, align >= 8);
    store4(p + 4, f32x4{v[4], v[5], v[6], v[7]}, valid - 4, align >= 8);
}

__device__ __forceinline__ bf16x4 read_transposed(const __bf16 *p) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(p));
    return __builtin_bit_cast(bf16x4, v);
}
__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Tiles dealt out evenly, in order, to at most as many ranges as there are tiles, so that none is empty:
// the first tile of range r, the range of tile t.
__device__ __forceinline__ int range_first(uint32_t r, int tiles, uint32_t ranges) {
    return (int)((uint64_t)r * (uint32_t)tiles / ranges);
}
__device__ __forceinline__ int range_of(int t, int tiles, uint32_t ranges) {
    return (int)(((uint64_t)(t + 1) * ranges - 1) / (uint32_t)tiles);
}

// The 16 outer x kSlab inner operand fragment of a wave.  Inner elements are dealt to the lanes in an
// order of our own, the same for both operands: lane group g = lane / 16 holds, of every 16 inner
// elements, 4 g .. 4 g + 3.
template <typename T> struct Frag;
template <> struct Frag<float> {
    f32x4 v;
    // rows of inner elements: s[outer][inner]
    __device__ __forceinline__ void rows(const float *s, int stride, int outer, int inner, int lane) {
        v = *reinterpret_cast<const f32x4 *>(s + (outer + (lane & 15)) * stride + inner + 4 * (lane >> 4));
    }
    __device__ __forceinline__ void rank_row(const float *s, int stride, int outer, int lane) {
        rows(s, stride, outer, 0, lane);
    }
    // rows of outer elements: s[inner][outer]
    __device__ __forceinline__ void columns(const float *s, int stride, int outer, int inner, int lane) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = s[(inner + 4 * (lane >> 4) + i) * stride + outer + (lane & 15)];
    }
    __device__ __forceinline__ float sum() const { return (v[0] + v[1]) + (v[2] + v[3]); }
    __device__ __forceinline__ void clear() { v = f32x4{0.f, 0.f, 0.f, 0.f}; }
};
template <> struct Frag<__bf16> {
    bf16x8 v;
    __device__ __forceinline__ void rows(const __bf16 *s, int stride, int outer, int inner, int lane) {
        const __bf16 *p = s + (outer + (lane & 15)) * stride + inner + 4 * (lane >> 4);
        v = join(*reinterpret_cast<const bf16x4 *>(p), *reinterpret_cast<const bf16x4 *>(p + 16));
    }
    // 16 inner elements, for the high parts of the other operand and again for its low parts
    __device__ __forceinline__ void rank_row(const __bf16 *s, int stride, int outer, int lane) {
        const bf16x4 q = *reinterpret_cast<const bf16x4 *>(s + (outer + (lane & 15)) * stride + 4 * (lane >> 4));
        v = join(q, q);
    }
    __device__ __forceinline__ void columns(const __bf16 *s, int stride, int outer, int inner, int lane) {
        const int g = lane >> 4, i = lane & 15;
        const __bf16 *p = s + (inner + 4 * g + (i >> 2)) * stride + outer + 4 * (i & 3);
        v = join(read_transposed(p), read_transposed(p + 16 * stride));
    }
    __device__ __forceinline__ float sum() const {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += (float)v[i];
        return s;
    }
    __device__ __forceinline__ void clear() { v = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0}); }
};
__device__ __forceinline__ f32x4 mma(const Frag<float> &a, const Frag<float> &b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma(const Frag<__bf16> &a, const Frag<__bf16> &b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}

// Weights of every type: element (k, n) of type t at t * type + k * inner + n * outer; one of the two
// strides is 1.
struct WeightView {
    const void *data;
    int64_t type, inner, outer;
    int mode;  // ChunkMode of its contiguous rows
};

struct ProductArgs {
    const void *x;
    int64_t ldx;
    int x_mode;
    WeightView w;
    const void *bias;  // [type][N] or [N] (adapted form), may be NULL
    int64_t bias_type;
    void *y;           // rows at their ids; `sorted`: float32 rows at their positions
    int64_t ldy;
    int y_align, sorted;
    float scale;       // of the product (before the bias); narrow_product_kernel, adapted form: of x down
    PlanView plan;
    int K, N;
    // adapted form: low[position][rank] float32 times the `up` weights of the row's type
    const float *low;
    int rank;
    WeightView up;
    // narrow_product_kernel, adapted form: x down, times `scale`, is made on the way and kept in
    // low_out[position][rank] where that is not NULL
    WeightView down;
    float *low_out;
    uint32_t ranges;  // workgroups that share the tiles
};

// 8 XCDs, each with an L2 of its own, take workgroups in turn: the column blocks of a tile follow one
// another on ONE of them, so that its rows come from HBM once.
__device__ __forceinline__ bool tile_of_block(uint32_t tiles, uint32_t columns, uint32_t *tile,
                                              uint32_t *column) {
    const uint32_t xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
    *tile = i / columns * 8 + xcd;
    *column = i % columns;
    return *tile < tiles;
}

// y tile of up to 64 rows x BN columns in one workgroup of four waves.  WT: the weights' inner
// elements are contiguous (the transposed product of the backward pass).  ADAPT: tiles are 64
// consecutive positions of any types; the weights are shared and the rows of every type in the tile
// get their low-rank part in further steps of the same accumulators.
//
// One stage of the inner axis is multiplied while the next one's loads are under way; four workgroups per CU
// take turns at the barriers.  float32 is bound by the matrix instructions (300 000 rows of 512 -> 512: 1 423
// us, 0.72 of the 154 TFLOP/s that a large product reaches), bfloat16 by what the fragments take from LDS, 6 KB
// for eight 16-cycle instructions (368 us, 427 TFLOP/s).  Tiles of 128 rows, eight waves and two buffers an
// operand gave the same in bfloat16 (365 us) and in float32 left too few workgroups to hide a barrier
// behind another (400 000 rows of 256 -> 256: 712 us instead of 506).
template <typename T, int BN, bool WT, bool ADAPT>
__global__ __launch_bounds__(256, 4) void product_kernel(ProductArgs a) {
    constexpr int E = Tile<T>::kChunk, BK = Tile<T>::kDepth, SLAB = Tile<T>::kSlab;
    constexpr int XS = BK + Tile<T>::kPad;
    constexpr int WS = WT ? XS : BN + (sizeof(T) == 4 ? 4 : 16);
    constexpr int WAVES_N = BN / 32, WAVES_M = 4 / WAVES_N;
    constexpr int MI = 4 / WAVES_M, NI = 2;
    constexpr int XL = 64 * BK / E / 256, WL = BN * BK / E / 256;
    __shared__ __align__(16) T xs[64 * XS];
    __shared__ __align__(16) T ws[WT ? BN * XS : BK * WS];
    __shared__ int ids[64], types[64];
    uint32_t tile, column;
    const uint32_t tiles = ADAPT ? (a.plan.rows + 63) / 64 : (uint32_t)plan_word(a.plan.tile_first, (int)a.plan.types + 1);
    if (!tile_of_block(tiles, (uint32_t)((a.N + BN - 1) / BN), &tile, &column)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = (int)column * BN;
    int type = 0, start, count;
    if (ADAPT) {
        start = (int)(tile * 64);
        count = min(64, (int)(a.plan.rows - tile * 64));
    } else {
        const TileAt at = find_tile(a.plan, (int)tile, lane);
        type = at.type;
        start = at.start;
        count = at.count();
    }
    if (tid < 64) {
        ids[tid] = tid < count ? a.plan.order[start + tid] : 0;
        if (ADAPT) types[tid] = tid < count ? a.plan.row_types[start + tid] : (int)a.plan.types;
    }
    __syncthreads();
    const int wn = wave % WAVES_N, m0 = wave / WAVES_N * MI * 16;
    f32x4 acc[MI][NI] = {};
    const bool unknown = !ADAPT && type == (int)a.plan.types;
    if (unknown && a.sorted) return;  // nobody reads the low-rank rows of unknown types
    if (!unknown) {
        const T *w = (const T *)a.w.data + (ADAPT ? 0 : (int64_t)type * a.w.type);
        u32x4 xr[XL], wr[WL];
        auto fetch_x = [&](int k0) {
#pragma unroll
            for (int i = 0; i < XL; ++i) {
                const int c = tid + 256 * i, row = c / (BK / E), k = k0 + c % (BK / E) * E;
                // rows behind the tile's last stand for row 0: nobody stores what they give
                xr[i] = load_chunk((const T *)a.x + (int64_t)ids[row] * a.ldx, k, a.K, a.x_mode);
            }
        };
        auto fetch_w = [&](const T *p, const WeightView &v, int k0, int depth) {
#pragma unroll
            for (int i = 0; i < WL; ++i) {
                const int c = tid + 256 * i;
                if (WT) {
                    const int n = c / (BK / E), k = k0 + c % (BK / E) * E;
                    // columns behind the last one likewise
                    wr[i] = load_chunk(p + (int64_t)min(n0 + n, a.N - 1) * v.outer, k, depth, v.mode);
                } else {
                    const int k = k0 + c / (BN / E), n = n0 + c % (BN / E) * E;
                    wr[i] = load_chunk(p + (int64_t)k * v.inner, n, a.N, v.mode, k < depth);
                }
            }
        };
        auto put_x = [&]() {
#pragma unroll
            for (int i = 0; i < XL; ++i) {
                const int c = tid + 256 * i;
                *reinterpret_cast<u32x4 *>(xs + c / (BK / E) * XS + c % (BK / E) * E) = xr[i];
            }
        };
        auto put_w = [&]() {
#pragma unroll
            for (int i = 0; i < WL; ++i) {
                const int c = tid + 256 * i;
                T *to = WT ? ws + c / (BK / E) * XS + c % (BK / E) * E : ws + c / (BN / E) * WS + c % (BN / E) * E;
                *reinterpret_cast<u32x4 *>(to) = wr[i];
            }
        };
        auto weights = [&](Frag<T> &f, int ni, int inner) {
            if (WT)
                f.rows(ws, XS, wn * 32 + ni * 16, inner, lane);
            else
                f.columns(ws, WS, wn * 32 + ni * 16, inner, lane);
        };
        fetch_x(0);
        fetch_w(w, a.w, 0, a.K);
        for (int k0 = 0; k0 < a.K; k0 += BK) {
            put_x();
            put_w();
            __syncthreads();
            if (k0 + BK < a.K) {
                fetch_x(k0 + BK);
                fetch_w(w, a.w, k0 + BK, a.K);
            }
#pragma unroll
            for (int slab = 0; slab < BK / SLAB; ++slab) {
                Frag<T> xf[MI], wf[NI];
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) xf[mi].rows(xs, XS, m0 + mi * 16, slab * SLAB, lane);
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) weights(wf[ni], ni, slab * SLAB);
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mma(wf[ni], xf[mi], acc[mi][ni]);
            }
            __syncthreads();
        }
        if (ADAPT) {
            // the tile's runs of one type, known types only
            const int own = types[lane];
            const bool begins = own < (int)a.plan.types && (lane == 0 || types[lane - 1] != own);
            unsigned long long runs = __ballot(begins);
            // Measured on 32 768 rows of 512 -> 256 (rank 16) and 1 024 -> 1 024 (rank 32), float32 and
            // bfloat16: 16 runs a tile 381 / 1 593 / 169 / 628 us this way, 423 / 1 584 / 205 / 867 the other;
            // 64 runs 1 183 / 4 160 / 571 / 1 877 and 1 079 / 2 567 / 510 / 1 137.
            if (__popcll(runs) <= 16) {
                // Few runs: 32 rank columns at a time.  A run is a product in sums of its own, which only its
                // rows take: weights that are infinite or NaN reach no row of another type.  In bfloat16
                // the low-rank rows enter as a high and a low part.
                for (; runs; runs &= runs - 1) {
                    const int t = types[__ffsll(runs) - 1];
                    const T *up = (const T *)a.up.data + (int64_t)t * a.up.type;
                    for (int j0 = 0; j0 < a.rank; j0 += 32) {
                        fetch_w(up, a.up, j0, min(a.rank, j0 + 32));
                        for (int i = tid; i < 64 * 32; i += 256) {
                            const int row = i >> 5, j = j0 + (i & 31);
                            const float v = row < count && types[row] == t && j < a.rank
                                                ? a.low[(int64_t)(start + row) * a.rank + j]
                                                : 0.f;
                            if constexpr (sizeof(T) == 4) {
                                xs[row * XS + (i & 31)] = v;
                            } else {
                                __bf16 high, rest;
                                split(v, high, rest);
                                xs[row * XS + (i & 31)] = high;
                                xs[row * XS + 32 + (i & 31)] = rest;
                            }
                        }
                        put_w();
                        __syncthreads();
#pragma unroll
                        for (int mi = 0; mi < MI; ++mi) {
                            const bool mine = types[m0 + mi * 16 + (lane & 15)] == t;
                            if (!__any(mine)) continue;
                            f32x4 part[NI] = {};
#pragma unroll
                            for (int slab = 0; slab < 2; ++slab) {
                                if (sizeof(T) == 4 && j0 + slab * 16 >= a.rank) break;
                                Frag<T> xf;
                                xf.rows(xs, XS, m0 + mi * 16, slab * SLAB, lane);
#pragma unroll
                                for (int ni = 0; ni < NI; ++ni) {
                                    Frag<T> wf;
                                    weights(wf, ni, sizeof(T) == 4 ? slab * SLAB : 0);
                                    part[ni] = mma(wf, xf, part[ni]);
                                }
                            }
#pragma unroll
                            for (int ni = 0; ni < NI; ++ni)
                                if (mine) acc[mi][ni] += part[ni];
                        }
                        __syncthreads();
                    }
                }
            } else {
                // Many types, few rows each: every lane adds its row's part from its row's weights.
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) {
                    const int row = m0 + mi * 16 + (lane & 15), t = types[row];
                    if (t >= (int)a.plan.types) continue;
                    const float *low = a.low + (int64_t)(start + row) * a.rank;
                    const T *up = (const T *)a.up.data + (int64_t)t * a.up.type;
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) {
                        const int n = n0 + wn * 32 + ni * 16 + 4 * (lane >> 4);
                        for (int j = 0; j < a.rank; ++j) {
                            const float v = low[j];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (n + i < a.N)
                                    acc[mi][ni][i] += v * (float)up[j * a.up.inner + (n + i) * a.up.outer];
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
        const int n = n0 + wn * 32 + ni * 16 + 4 * (lane >> 4);
        f32x4 bias = {0.f, 0.f, 0.f, 0.f};
        if (a.bias && !unknown) {
            const T *b = (const T *)a.bias + (int64_t)type * a.bias_type;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < a.N) bias[i] = (float)b[n + i];
        }
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            const int row = m0 + mi * 16 + (lane & 15);
            if (row >= count) continue;
            const f32x4 v = acc[mi][ni] * a.scale + bias;
            if (a.sorted)
                store4((float *)a.y + (int64_t)(start + row) * a.ldy + n, v, a.N - n, a.y_align == 16);
            else
                store4((T *)a.y + (int64_t)ids[row] * a.ldy + n, v, a.N - n, a.y_align >= (int)(4 * sizeof(T)));
        }
    }
}

// ------------------------------------------------------------------------- rows of some hundred bytes
// The same product where a row's inner elements fit one LDS tile (128 floats, 256 bfloat16 elements):
// what an embedding table has.  A workgroup of eight waves takes consecutive tiles of the plan, keeps the
// weights of the current type in its registers -- 16 columns per wave -- and has the next tile's rows
// under way while it multiplies.  ADAPT: the weights are shared and stay for the whole launch; a tile's
// low-rank rows x A are made from the tile itself (one more MFMA column block), go through LDS and are
// multiplied by B as one more step: x is read once.
//
// What a CU can have under way towards its L2 bounds both the rows and the weights (some 20 KB a
// microsecond): weights are therefore read once per workgroup, whole lines at a time, and dealt out
// through the LDS of the rows.  2.4 M bfloat16 rows of 128 -> 128, 16 types: 248 us, 5.0 TB/s (450 us in the
// kernel above); 169 343 float32 rows of 128 -> 128, 40 types: 70 us, where the bytes take 36 us and the
// matrix instructions 36 us, and a workgroup's five or six tiles leave a quarter of the time to its start
// and to the last tile.
constexpr int kFusedRank = 16;
constexpr int kNarrowThreads = 512;

// Rows multiplied at a time: half a tile where LDS would else hold one workgroup per CU.
constexpr int narrow_rows(int slabs, bool adapt) { return slabs == 8 && adapt ? 32 : 64; }

// 16-column blocks per wave.  Two, whose columns a lane holds in turn, make the stores of a bfloat16 row
// 64 bytes long instead of 32 (a launch of 2.4 M rows of 128: 250 us instead of 299); longer rows leave
// no registers for it, and float rows need no help.
constexpr int narrow_blocks(int size, int slabs) { return size == 2 && slabs < 6 ? 2 : 1; }

// Slabs of weights that go through LDS at a time, where it has room for `fit` of them.
constexpr int narrow_step(int slabs, int fit) {
    int step = slabs;
    while (step > fit) step = step % 2 ? 1 : step / 2;
    return step;
}

template <typename T, int SLABS, int BN, bool WT, bool ADAPT>
__global__ __launch_bounds__(kNarrowThreads, 4) void narrow_product_kernel(ProductArgs a) {
    constexpr int E = Tile<T>::kChunk, SLAB = Tile<T>::kSlab, DEPTH = SLABS * SLAB;
    constexpr int XS = DEPTH + Tile<T>::kPad, CHUNKS = DEPTH / E;
    constexpr int NI = narrow_blocks(sizeof(T), SLABS), WAVES_N = BN / (16 * NI), WAVES_M = 8 / WAVES_N;
    constexpr int ROWS = narrow_rows(SLABS, ADAPT), MI = ROWS / 16 / WAVES_M;
    constexpr int XL = ROWS * CHUNKS / kNarrowThreads;
    static_assert(MI >= 1 && XL >= 1, "every wave has rows, every thread a chunk");
    constexpr int LS = sizeof(T) == 4 ? 20 : 40;  // low-rank rows in LDS: 16 floats, or 16 + 16 halves
    // the weights' way through LDS: STEP slabs at a time, inner elements or columns as rows
    constexpr int WS = BN + (sizeof(T) == 4 ? 4 : 16);
    constexpr int LDS_X = 2 * ROWS * XS, LDS_W = LDS_X > 17408 / (int)sizeof(T) ? LDS_X : 17408 / (int)sizeof(T);
    constexpr int FIT = LDS_W / (WT ? BN * (SLAB + Tile<T>::kPad) : SLAB * WS);
    constexpr int STEP = narrow_step(SLABS, FIT);
    constexpr int WTS = STEP * SLAB + Tile<T>::kPad;
    static_assert((WT ? BN * WTS : STEP * SLAB * WS) <= LDS_W, "weights in passes");
    __shared__ __align__(16) T xs[LDS_W];
    __shared__ __align__(16) T ls[ADAPT ? ROWS * LS : 1];
    __shared__ __align__(16) T as[ADAPT ? 16 * XS : 1];
    __shared__ __align__(16) T us[ADAPT ? BN * 20 : 1];  // rows of 16 rank elements and a gap
    __shared__ int ids[3][64];
    uint32_t range, column;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (!tile_of_block(a.ranges, (uint32_t)((a.N + BN - 1) / BN), &range, &column)) return;
    const int tiles = plan_word(a.plan.tile_first, (int)a.plan.types + 1);
    const uint32_t ranges = min(a.ranges, (uint32_t)tiles);
    if (range >= ranges) return;
    const int first = range_first(range, tiles, ranges), last = range_first(range + 1, tiles, ranges);
    // Waves behind the last column have nothing to multiply; which they are takes turns among the workgroups
    // of a CU, and so do the SIMDs that they leave.
    const int turn = (wave + (int)(range >> 8)) & 7;
    const int wn = turn % WAVES_N, m0 = turn / WAVES_N * MI * 16, nb = (int)column * BN, n0 = nb + wn * 16 * NI;
    const int n = n0 + 4 * NI * (lane >> 4);  // the lane's 4 * NI output columns
    const int unknown = (int)a.plan.types;
    u32x4 xr[XL];
    auto fetch = [&](const int *id) {  // ids behind a tile's last row are 0: nobody stores what they give
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int c = tid + kNarrowThreads * i;
            xr[i] = load_chunk((const T *)a.x + (int64_t)id[c / CHUNKS] * a.ldx, c % CHUNKS * E, a.K, a.x_mode);
        }
    };
    Frag<T> wf[SLABS][NI];
    // The workgroup's columns of one type's weights, STEP slabs at a time through the rows' LDS; with
    // two blocks per wave the even columns of 32 go in front of the odd ones.
    auto load_weights = [&](const T *w) {
#pragma unroll
        for (int s0 = 0; s0 < SLABS; s0 += STEP) {
            if (s0 * SLAB >= a.K) {
#pragma unroll
                for (int s = s0; s < s0 + STEP; ++s)
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) wf[s][ni].clear();
                continue;
            }
            constexpr int LINE = WT ? STEP * SLAB / E : BN / E, COUNT = WT ? BN * LINE : STEP * SLAB * LINE;
            __syncthreads();  // the rows have been multiplied, or the last pass has been read
#pragma unroll 8
            for (int c = tid; c < COUNT; c += kNarrowThreads) {
                const int line = c / LINE, at = c % LINE * E;
                u32x4 q;
                if (WT)
                    q = load_chunk(w + (int64_t)min(nb + line, a.N - 1) * a.w.outer, s0 * SLAB + at, a.K, a.w.mode);
                else
                    q = load_chunk(w + (int64_t)(s0 * SLAB + line) * a.w.inner, nb + at, a.N, a.w.mode,
                                   s0 * SLAB + line < a.K);
                if constexpr (NI == 2 && WT) {
                    const int to = (line & ~31) + (line & 1) * 16 + (line & 31) / 2;
                    *reinterpret_cast<u32x4 *>(xs + to * WTS + at) = q;
                } else if constexpr (NI == 2) {
                    T *to = xs + line * WS + (at & ~31) + (at & 31) / 2;
                    const uint2 even = {(q[0] & 0xFFFFu) | q[1] << 16, (q[2] & 0xFFFFu) | q[3] << 16};
                    const uint2 odd = {q[0] >> 16 | (q[1] & 0xFFFF0000u), q[2] >> 16 | (q[3] & 0xFFFF0000u)};
                    *reinterpret_cast<uint2 *>(to) = even;
                    *reinterpret_cast<uint2 *>(to + 16) = odd;
                } else {
                    *reinterpret_cast<u32x4 *>(xs + line * (WT ? WTS : WS) + at) = q;
                }
            }
            __syncthreads();
#pragma unroll
            for (int s = 0; s < STEP; ++s)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) {
                    if (WT)
                        wf[s0 + s][ni].rows(xs, WTS, (wn * NI + ni) * 16, s * SLAB, lane);
                    else
                        wf[s0 + s][ni].columns(xs, WS, (wn * NI + ni) * 16, s * SLAB, lane);
                }
        }
        __syncthreads();
    };
    float bias[4 * NI] = {};
    auto load_bias = [&](const T *b) {
        if (!a.bias) return;
#pragma unroll
        for (int i = 0; i < 4 * NI; ++i) bias[i] = (float)b[min(n + i, a.N - 1)];
    };
    auto id_of = [&](const TileAt &at) { return tid < at.count() ? a.plan.order[at.start + tid] : 0; };
    TileAt at = find_tile(a.plan, first, lane), ahead = at, ahead2;
    if (first + 1 < last) ahead = tile_behind(a.plan, at);
    ahead2 = ahead;
    if (first + 2 < last) ahead2 = tile_behind(a.plan, ahead);
    if (tid < 64) {
        ids[0][tid] = id_of(at);
        ids[1][tid] = id_of(ahead);
    }
    __syncthreads();
    int loaded = -1;
    fetch(ids[0]);
    if (ADAPT) {
        load_bias((const T *)a.bias);
        load_weights((const T *)a.w.data);
    }
    int slot = 0, buffer = 0;
    for (int t = first; t < last; ++t) {
        const bool known = at.type != unknown;
        if (at.type != loaded && known) {
            loaded = at.type;
            if (!ADAPT) {
                load_bias((const T *)a.bias + (int64_t)at.type * a.bias_type);
                load_weights((const T *)a.w.data + (int64_t)at.type * a.w.type);
            } else {
                // A and B in LDS, their rank elements as rows and within rows, B's columns in the order of
                // the weights'
                const T *down = (const T *)a.down.data + (int64_t)at.type * a.down.type;
                const T *up = (const T *)a.up.data + (int64_t)at.type * a.up.type;
                __syncthreads();  // the last tile has been multiplied
#pragma unroll 4
                for (int i = tid; i < 16 * DEPTH; i += kNarrowThreads) {
                    const int j = WT ? i / DEPTH : i & 15, k = WT ? i % DEPTH : i >> 4;
                    const T q = down[min(k, a.K - 1) * a.down.inner + min(j, a.rank - 1) * a.down.outer];
                    as[j * XS + k] = k < a.K && j < a.rank ? q : (T)0.f;
                }
#pragma unroll 4
                for (int i = tid; i < 16 * BN; i += kNarrowThreads) {
                    const int j = WT ? i & 15 : i / BN, c = WT ? i >> 4 : i % BN;
                    const T q = up[min(j, a.rank - 1) * a.up.inner + min(nb + c, a.N - 1) * a.up.outer];
                    const int to = NI == 2 ? (c & ~31) + (c & 1) * 16 + (c & 31) / 2 : c;
                    us[to * 20 + j] = j < a.rank ? q : (T)0.f;
                }
            }
        }
        const int count = at.count(), start = at.start;
        const int *id = ids[slot];
        const int next = slot == 2 ? 0 : slot + 1, free = next == 2 ? 0 : next + 1;
        at = ahead;
        for (int r0 = 0; r0 < count; r0 += ROWS) {
            T *x = xs + buffer * ROWS * XS;  // its last readers are behind the last barrier
            buffer ^= 1;
#pragma unroll
            for (int i = 0; i < XL; ++i) {
                const int c = tid + kNarrowThreads * i;
                *reinterpret_cast<u32x4 *>(x + c / CHUNKS * XS + c % CHUNKS * E) = xr[i];
            }
            __syncthreads();
            // the ids of the tile behind the next, the next rows: of this tile or of the next one
            const bool ends = r0 + ROWS >= count;
            int id_ahead = 0;
            if (ends && t + 2 < last && tid < 64) id_ahead = id_of(ahead2);
            if (!ends || t + 1 < last) fetch(ends ? ids[next] : id + r0 + ROWS);
            // 16-row blocks of this wave that hold rows
            const int live = n0 < a.N ? (count - r0 - m0 + 15) >> 4 : 0;
            f32x4 acc[MI][NI] = {};
            if (ADAPT || known) {
#pragma unroll
                for (int s = 0; s < SLABS; ++s)
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi)
                        if (mi < live) {
                            Frag<T> xf;
                            xf.rows(x, XS, m0 + mi * 16, s * SLAB, lane);
#pragma unroll
                            for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mma(wf[s][ni], xf, acc[mi][ni]);
                        }
                if (ADAPT && known) {
                    if (wave * 16 < ROWS && r0 + wave * 16 < count) {
                        // row block `wave`; lane: rank columns 4 (lane / 16) .. + 3 of row lane % 16
                        f32x4 low = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int s = 0; s < SLABS; ++s) {
                            Frag<T> xf, af;
                            xf.rows(x, XS, wave * 16, s * SLAB, lane);
                            af.rows(as, XS, 0, s * SLAB, lane);
                            low = mma(af, xf, low);
                        }
                        const int row = wave * 16 + (lane & 15), j = 4 * (lane >> 4);
                        // columns behind the rank stay zero, also where the row holds an infinity
#pragma unroll
                        for (int i = 0; i < 4; ++i) low[i] = j + i < a.rank ? low[i] * a.scale : 0.f;
                        if (a.low_out && column == 0 && r0 + row < count)
                            store4(a.low_out + (int64_t)(start + r0 + row) * a.rank + j, low, a.rank - j,
                                   (a.rank & 3) == 0);
                        if constexpr (sizeof(T) == 4) {
                            *reinterpret_cast<f32x4 *>(ls + row * LS + j) = low;
                        } else {
                            bf16x4 high, rest;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                __bf16 h, r;
                                split(low[i], h, r);
                                high[i] = h;
                                rest[i] = r;
                            }
                            *reinterpret_cast<bf16x4 *>(ls + row * LS + j) = high;
                            *reinterpret_cast<bf16x4 *>(ls + row * LS + 16 + j) = rest;
                        }
                    }
                    __syncthreads();
                    Frag<T> uf[NI];
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) uf[ni].rank_row(us, 20, (wn * NI + ni) * 16, lane);
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi)
                        if (mi < live) {
                            Frag<T> lf;
                            lf.rows(ls, LS, m0 + mi * 16, 0, lane);
#pragma unroll
                            for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mma(uf[ni], lf, acc[mi][ni]);
                        }
                }
            }
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) {
                const int row = r0 + m0 + mi * 16 + (lane & 15);
                if (row >= count) continue;
                T *y = (T *)a.y + (int64_t)id[row] * a.ldy + n;
                float v[4 * NI];
#pragma unroll
                for (int i = 0; i < 4 * NI; ++i)
                    v[i] = ADAPT   ? acc[mi][i % NI][i / NI] + bias[i]
                           : known ? acc[mi][i % NI][i / NI] * a.scale + bias[i]
                                   : 0.f;
                if constexpr (NI == 2)
                    store8(y, v, a.N - n, a.y_align);
                else
                    store4(y, f32x4{v[0], v[1], v[2], v[3]}, a.N - n, a.y_align >= (int)(4 * sizeof(T)));
            }
            if (ends && tid < 64) ids[free][tid] = id_ahead;
        }
        slot = next;
        ahead = ahead2;
        if (t + 3 < last) ahead2 = tile_behind(a.plan, ahead2);
    }
}

// --------------------------------------------------------------------------------- few rows
// One workgroup per row and 64 columns: lanes read 16 bytes of a weight row each, the workgroup's
// 256 / (64 / kChunk) row groups split the inner axis and are joined in LDS.  No plan, one launch.  Bound by
// latency while there are fewer workgroups than CUs (64 rows of 128 -> 128 float32: 3.8 us), then by the
// weights that every row reads through L2 (512 rows of 512 -> 256: 268 MB in 15.7 us).
constexpr int kFewDepth = 4096;  // inner elements a workgroup keeps in LDS
constexpr int kMaxRank = 64;

struct FewArgs {
    const void *x;
    int64_t ldx;
    WeightView w;  // outer elements contiguous; type stride 0: shared
    const void *bias;
    int64_t bias_type;
    void *y;
    int64_t ldy;
    const void *types;  // int32 / int64 per row, or NULL: the plan's
    int type_bytes;
    PlanView plan;
    int K, N, rank;
    float scale;
    WeightView down, up;  // adapted form; outer elements contiguous
};

template <typename T, bool ADAPT>
__global__ __launch_bounds__(256) void few_rows_kernel(FewArgs a) {
    constexpr int E = Tile<T>::kChunk, LANES = 64 / E, SPLIT = 256 / LANES;
    __shared__ float xs[kFewDepth];
    __shared__ float part[SPLIT * 64];
    __shared__ float low[kMaxRank];
    const int tid = threadIdx.x, n0 = blockIdx.x * 64;
    int row = (int)blockIdx.y, type;
    if (a.types) {
        type = a.type_bytes == 8 ? type_at((const int64_t *)a.types, row, a.plan.types)
                                 : type_at((const int32_t *)a.types, row, a.plan.types);
    } else {
        type = a.plan.row_types[row];
        row = a.plan.order[row];
    }
    const bool known = type < (int)a.plan.types;
    T *y = (T *)a.y + (int64_t)row * a.ldy;
    if (!ADAPT && !known) {
        if (tid < 64 && n0 + tid < a.N) y[n0 + tid] = (T)0.f;
        return;
    }
    for (int k = tid; k < a.K; k += 256) xs[k] = (float)((const T *)a.x)[(int64_t)row * a.ldx + k];
    __syncthreads();
    const int split = tid / LANES, c = tid % LANES * E;
    float acc[E] = {};
    auto accumulate = [&](const T *w, const WeightView &v, const float *vec, int depth) {
#pragma unroll 8
        for (int k = split; k < depth; k += SPLIT) {
            const u32x4 q = load_chunk(w + (int64_t)k * v.inner, n0 + c, a.N, v.mode);
            const float f = vec[k];
#pragma unroll
            for (int i = 0; i < E; ++i)
                acc[i] += f * (sizeof(T) == 4 ? __uint_as_float(q[i & 3])
                                              : __uint_as_float(i & 1 ? q[i / 2] & 0xFFFF0000u : q[i / 2] << 16));
        }
    };
    accumulate((const T *)a.w.data + (ADAPT ? 0 : (int64_t)type * a.w.type), a.w, xs, a.K);
    if (ADAPT && known) {
        // x A: the rank's next power of two lanes side by side, the inner axis split over the others
        int width = 1;
        while (width < a.rank) width <<= 1;
        const int j = tid & (width - 1), splits = 256 / width;
        const T *down = (const T *)a.down.data + (int64_t)type * a.down.type;
        float sum = 0.f;
        if (j < a.rank) {
#pragma unroll 8
            for (int k = tid / width; k < a.K; k += splits)
                sum += xs[k] * (float)down[(int64_t)k * a.down.inner + j];
        }
        part[tid] = sum;
        __syncthreads();
        if (tid < a.rank) {
            float s = 0.f;
            for (int i = 0; i < splits; ++i) s += part[i * width + tid];
            low[tid] = s * a.scale;
        }
        __syncthreads();
        accumulate((const T *)a.up.data + (int64_t)type * a.up.type, a.up, low, a.rank);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) part[split * 64 + c + i] = acc[i];
    __syncthreads();
    if (tid < 64 && n0 + tid < a.N) {
        float s = 0.f;
        for (int i = 0; i < SPLIT; ++i) s += part[i * 64 + tid];
        if (!ADAPT) s *= a.scale;
        if (a.bias) s += (float)((const T *)a.bias)[(ADAPT ? 0 : (int64_t)type * a.bias_type) + n0 + tid];
        y[n0 + tid] = (T)s;
    }
}

// ------------------------------------------------------------------------- weights' gradients
// dW[t] = sum over the rows of type t of x[r]^T dy[r].  The tiles of the plan are dealt out evenly, in
// order, to `ranges` workgroups per block of dW; a workgroup adds the outer products of one type's rows
// in registers.  A type whose tiles lie in one range is written at once.  A range leaves the sums of
// a type that began before it in its first slot, those of a type that goes on behind it in its second; a
// second launch joins them in order (no atomics: the same bits in every run).  Either operand may be
// float32 rows at their positions (the low-rank rows), which enter bfloat16 products as a high and a
// low part.  Both operands lie in LDS with the rows as the inner axis, which is what a transposed read
// (bfloat16) or four words (float32) take.  Bound by HBM: 2.4 M bfloat16 rows of 128 x 128 262 us, 4.7 TB/s.
enum GradSpan : int { kKnownTiles = 0, kRowBlocks = 1, kAllTiles = 2 };

struct GradArgs {
    const void *x, *dy;
    int64_t ldx, ldy;
    int x_mode, y_mode;
    PlanView plan;
    int span;        // what is dealt out: the known types' tiles, 64 rows after the other, all tiles
    int shared;      // one gradient of all of it, not one per type
    uint32_t ranges;
    int K, N;
    // sums of a range, float32: [range][2][stride], `first` of them for `dw`, and from second_at (a
    // multiple of 4) `second` for `db`
    float *partial;
    int64_t stride, first, second, second_at;
    void *dw;        // [type][first]; NULL when only the bias is asked for (K = 0)
    void *db;        // [type][second] or NULL
};
__device__ __forceinline__ int grad_tiles(const GradArgs &a) {
    return a.span == kRowBlocks ? (int)((a.plan.rows + kTileRows - 1) / kTileRows)
                                : plan_word(a.plan.tile_first, (int)a.plan.types + (a.span == kAllTiles));
}

// waves per SIMD that the registers of a block's sums leave room for
constexpr int grad_waves(int mi, int ni) { return mi * ni >= 8 ? 2 : 4; }

template <typename T, int MI, int NI, bool XLOW, bool YLOW>
__global__ __launch_bounds__(256, grad_waves(MI, NI)) void grad_kernel(GradArgs a) {
    constexpr int E = Tile<T>::kChunk, R = Tile<T>::kDepth, STEP = Tile<T>::kSlab;
    constexpr int STAGES = kTileRows / R;  // a tile is one stage (bfloat16) or two (float)
    constexpr int BM = 32 * MI, BN = 32 * NI;
    constexpr bool SPLITX = XLOW && sizeof(T) == 2, SPLITY = YLOW && sizeof(T) == 2;
    // row strides that keep the four lane groups, four rows apart, in different banks: 4 words more
    // than a multiple of 32 (float), 8 words more (bfloat16, read in transposed blocks of 4 rows)
    constexpr int PAD = sizeof(T) == 4 ? 4 : 16;
    constexpr int XW = BM * (SPLITX ? 2 : 1) + PAD, YW = BN * (SPLITY ? 2 : 1) + PAD;
    constexpr int XL = R * BM / E / 256, YL = R * BN / E / 256;
    static_assert(XL >= 1 && YL >= 1, "a block of at least 32 x 32");
    __shared__ __align__(16) T xss[2][R * XW];
    __shared__ __align__(16) T yss[2][R * YW];
    __shared__ int ids[3][kTileRows];
    const uint32_t kb = a.K > 0 ? (uint32_t)((a.K + BM - 1) / BM) : 1, nb = (uint32_t)((a.N + BN - 1) / BN);
    uint32_t range, block;
    if (!tile_of_block(a.ranges, kb * nb, &range, &block)) return;
    const int k0 = (int)(block / nb) * BM, n0 = (int)(block % nb) * BN;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int tiles = grad_tiles(a);
    const uint32_t ranges = min(a.ranges, (uint32_t)tiles);
    if (range >= ranges) return;
    const int first = range_first(range, tiles, ranges), last = range_first(range + 1, tiles, ranges);
    const int wm = wave >> 1, wn = wave & 1;
    f32x4 acc[MI][NI] = {};
    float sums[NI] = {};
    const bool want_sums = a.db && k0 == 0 && wm == 0;
    u32x4 xr[XL], yr[YL], xr2[SPLITX ? XL : 1], yr2[SPLITY ? YL : 1];
    // float32 rows in a bfloat16 product: 8 floats -> 8 high and 8 low parts
    auto fetch_low = [&](const float *row, int k, int length, int mode, bool live, u32x4 &high, u32x4 &low) {
        const u32x4 q0 = load_chunk(row, k, length, mode, live), q1 = load_chunk(row, k + 4, length, mode, live);
        bf16x8 h, l;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            __bf16 upper, rest;
            split(__uint_as_float(i < 4 ? q0[i & 3] : q1[i & 3]), upper, rest);
            h[i] = upper;
            l[i] = rest;
        }
        high = __builtin_bit_cast(u32x4, h);
        low = __builtin_bit_cast(u32x4, l);
    };
    // rows r0 .. of a tile, `id` = its ids; rows behind its last count as zeros
    auto fetch = [&](const TileAt &at, const int *id, int r0) {
        const int count = at.count();
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int c = tid + 256 * i, row = r0 + c / (BM / E), k = k0 + c % (BM / E) * E;
            const int64_t r = XLOW ? at.start + row : id[row];
            if constexpr (SPLITX)
                fetch_low((const float *)a.x + r * a.ldx, k, a.K, a.x_mode, row < count, xr[i], xr2[i]);
            else
                xr[i] = load_chunk((const T *)a.x + r * a.ldx, k, a.K, a.x_mode, row < count);
        }
#pragma unroll
        for (int i = 0; i < YL; ++i) {
            const int c = tid + 256 * i, row = r0 + c / (BN / E), n = n0 + c % (BN / E) * E;
            const int64_t r = YLOW ? at.start + row : id[row];
            if constexpr (SPLITY)
                fetch_low((const float *)a.dy + r * a.ldy, n, a.N, a.y_mode, row < count, yr[i], yr2[i]);
            else
                yr[i] = load_chunk((const T *)a.dy + r * a.ldy, n, a.N, a.y_mode, row < count);
        }
    };
    auto id_at = [&](const TileAt &at) {
        return tid >= at.count() ? 0 : a.shared ? at.start + tid : a.plan.order[at.start + tid];
    };
    auto behind = [&](TileAt at) {
        if (!a.shared) return tile_behind(a.plan, at);
        at.start += kTileRows;
        return at;
    };
    TileAt at;
    if (a.shared) {
        at.type = 0;
        at.start = first * kTileRows;
        at.end = (int)a.plan.rows;
    } else {
        at = find_tile(a.plan, first, lane);
    }
    TileAt ahead = at, ahead2;
    if (first + 1 < last) ahead = behind(at);
    ahead2 = ahead;
    if (first + 2 < last) ahead2 = behind(ahead);
    if (tid < kTileRows) {
        ids[0][tid] = id_at(at);
        ids[1][tid] = id_at(ahead);
    }
    __syncthreads();
    fetch(at, ids[0], 0);
    int slot = 0, buffer = 0;
    for (int t = first; t < last; ++t) {
        const TileAt now = at;
        const int next = slot == 2 ? 0 : slot + 1, free = next == 2 ? 0 : next + 1;
#pragma unroll
        for (int stage = 0; stage < STAGES; ++stage) {
            // a wave that writes this buffer has passed the barrier behind its last readers
            T *xs = xss[buffer], *ys = yss[buffer];
            buffer ^= 1;
#pragma unroll
            for (int i = 0; i < XL; ++i) {
                const int c = tid + 256 * i;
                T *to = xs + c / (BM / E) * XW + c % (BM / E) * E;
                *reinterpret_cast<u32x4 *>(to) = xr[i];
                if constexpr (SPLITX) *reinterpret_cast<u32x4 *>(to + BM) = xr2[i];
            }
#pragma unroll
            for (int i = 0; i < YL; ++i) {
                const int c = tid + 256 * i;
                T *to = ys + c / (BN / E) * YW + c % (BN / E) * E;
                *reinterpret_cast<u32x4 *>(to) = yr[i];
                if constexpr (SPLITY) *reinterpret_cast<u32x4 *>(to + BN) = yr2[i];
            }
            __syncthreads();
            // the ids of the tile behind the next, the next rows: of this tile or of the next one
            const bool ends = stage + 1 == STAGES;
            int id_ahead = 0;
            if (ends && t + 2 < last && tid < kTileRows) id_ahead = id_at(ahead2);
            if (!ends || t + 1 < last) fetch(ends ? ahead : now, ids[ends ? next : slot], ends ? 0 : R * (stage + 1));
#pragma unroll
            for (int r = 0; r < R; r += STEP) {
                Frag<T> yf[NI], yl[SPLITY ? NI : 1];
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) {
                    yf[ni].columns(ys, YW, wn * NI * 16 + ni * 16, r, lane);
                    if constexpr (SPLITY) yl[ni].columns(ys, YW, BN + wn * NI * 16 + ni * 16, r, lane);
                    if (want_sums) sums[ni] += yf[ni].sum();
                }
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) {
                    Frag<T> xf;
                    xf.columns(xs, XW, wm * MI * 16 + mi * 16, r, lane);
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) {
                        acc[mi][ni] = mma(yf[ni], xf, acc[mi][ni]);
                        if constexpr (SPLITY) acc[mi][ni] = mma(yl[ni], xf, acc[mi][ni]);
                    }
                    if constexpr (SPLITX) {
                        xf.columns(xs, XW, BM + wm * MI * 16 + mi * 16, r, lane);
#pragma unroll
                        for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mma(yf[ni], xf, acc[mi][ni]);
                    }
                }
            }
            if (ends && tid < kTileRows) ids[free][tid] = id_ahead;
        }
        slot = next;
        at = ahead;
        ahead = ahead2;
        if (t + 3 < last) ahead2 = behind(ahead2);
        if (t + 1 < last && at.type == now.type) continue;
        // the type or the range ends here: its sums are whole, or one range's share of them
        const int type_first = a.shared ? 0 : plan_word(a.plan.tile_first, now.type);
        const int type_last = a.shared ? tiles : plan_word(a.plan.tile_first, now.type + 1);
        const bool whole = type_first >= first && type_last <= last;
        float *part = a.partial + (int64_t)(2 * range + (type_first >= first)) * a.stride;
        // lane: row k = lane % 16 of the block, four consecutive columns n
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            const int k = k0 + wm * MI * 16 + mi * 16 + (lane & 15);
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                const int n = n0 + wn * NI * 16 + ni * 16 + 4 * (lane >> 4);
                const bool vec = (a.N & 3) == 0;
                if (k < a.K) {
                    if (whole)
                        store4((T *)a.dw + ((int64_t)now.type * a.K + k) * a.N + n, acc[mi][ni], a.N - n, vec);
                    else
                        store4(part + (int64_t)k * a.N + n, acc[mi][ni], a.N - n, vec);
                }
                acc[mi][ni] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
        if (want_sums) {
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                float s = sums[ni];
                s += __shfl_xor(s, 16);
                s += __shfl_xor(s, 32);
                const int n = n0 + wn * NI * 16 + ni * 16 + lane;
                if (lane < 16 && n < a.N) {
                    if (whole)
                        ((T *)a.db)[(int64_t)now.type * a.N + n] = (T)s;
                    else
                        part[a.second_at + n] = s;
                }
                sums[ni] = 0.f;
            }
        }
    }
}

// All gradients of the adapted form at once, for rows and outputs of up to 128 elements and ranks of up
// to 16: d_down[t] = sum of x[r]^T back[r], d_up[t] = sum of low[r]^T dy[r] over the rows of type t, and
// (WANT_W) dW = sum of x[r]^T dy[r], db = sum of dy[r] over all rows.  The low-rank rows are further
// columns of the two LDS tiles, so that x and dy are read once instead of three times (1 M bfloat16 rows
// of 128 x 128, rank 16: 205 us with the joins instead of 331).  `types` has the sums per type (dw: d_down,
// db: d_up), `all` those of the shared weights.  640 MB in 195 us, 3.3 TB/s: waves wait 0.69 of their cycles,
// 0.02 for LDS, so what bounds it is how many rows are under way -- 32 a workgroup, as many workgroups as
// fit the LDS.
struct AdaptedGradArgs {
    GradArgs types, all;
    const float *low, *back;  // [position][rank]
    int rank, low_mode;
};

// workgroups per CU that registers and LDS leave room for
constexpr int adapted_grad_groups(int size) { return size == 2 ? 3 : 2; }

template <typename T, int MI, int NI, bool WANT_W>
__global__ __launch_bounds__(256, adapted_grad_groups(sizeof(T))) void adapted_grad_kernel(AdaptedGradArgs a) {
    constexpr int E = Tile<T>::kChunk, R = 32, STEP = Tile<T>::kSlab;
    constexpr int BM = 32 * MI, BN = 32 * NI, LOW = sizeof(T) == 4 ? 16 : 32;  // floats, or high | low
    // row strides as in grad_kernel: lane groups four rows apart fall into different banks
    constexpr int XW = BM + LOW + (sizeof(T) == 4 ? 4 : 16), YW = BN + LOW + (sizeof(T) == 4 ? 4 : 16);
    constexpr int XL = R * BM / E / 256, YL = R * BN / E / 256;
    static_assert(XL >= 1 && YL >= 1, "a block of at least 64 x 64");
    __shared__ __align__(16) T xss[2][R * XW];
    __shared__ __align__(16) T yss[2][R * YW];
    __shared__ int ids[3][kTileRows];
    const GradArgs &g = a.types;
    const int tiles = grad_tiles(g);
    const uint32_t ranges = min(g.ranges, (uint32_t)tiles), range = blockIdx.x;
    if (range >= ranges) return;
    const int first = range_first(range, tiles, ranges), last = range_first(range + 1, tiles, ranges);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, unknown = (int)g.plan.types;
    f32x4 acc[WANT_W ? MI : 1][WANT_W ? NI : 1] = {}, acc_down[MI / 2] = {}, acc_up[NI / 2] = {};
    float sums[WANT_W ? NI : 1] = {};
    u32x4 xr[XL], yr[YL], lr;
    // half the threads hold four elements of a row of `low`, half of `back`
    const float *rank_rows = tid < 128 ? a.low : a.back;
    const int rank_row = (tid & 127) >> 2, rank_at = (tid & 3) * 4;
    auto fetch = [&](const TileAt &at, const int *id, int r0) {
        const int count = at.count();
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int c = tid + 256 * i, row = r0 + c / (BM / E);
            xr[i] = load_chunk((const T *)g.x + (int64_t)id[row] * g.ldx, c % (BM / E) * E, g.K, g.x_mode, row < count);
        }
#pragma unroll
        for (int i = 0; i < YL; ++i) {
            const int c = tid + 256 * i, row = r0 + c / (BN / E);
            yr[i] = load_chunk((const T *)g.dy + (int64_t)id[row] * g.ldy, c % (BN / E) * E, g.N, g.y_mode, row < count);
        }
        lr = load_chunk(rank_rows + (int64_t)(at.start + r0 + rank_row) * a.rank, rank_at, a.rank, a.low_mode,
                        r0 + rank_row < count && at.type != unknown);
    };
    auto id_at = [&](const TileAt &at) { return tid < at.count() ? g.plan.order[at.start + tid] : 0; };
    TileAt at = find_tile(g.plan, first, lane), ahead = at, ahead2;
    if (first + 1 < last) ahead = tile_behind(g.plan, at);
    ahead2 = ahead;
    if (first + 2 < last) ahead2 = tile_behind(g.plan, ahead);
    if (tid < kTileRows) {
        ids[0][tid] = id_at(at);
        ids[1][tid] = id_at(ahead);
    }
    __syncthreads();
    fetch(at, ids[0], 0);
    int slot = 0, buffer = 0;
    for (int t = first; t < last; ++t) {
        const TileAt now = at;
        const int next = slot == 2 ? 0 : slot + 1, free = next == 2 ? 0 : next + 1, count = now.count();
        for (int r0 = 0; r0 < count; r0 += R) {
            // a wave that writes this buffer has passed the barrier behind its last readers
            T *xs = xss[buffer], *ys = yss[buffer];
            buffer ^= 1;
#pragma unroll
            for (int i = 0; i < XL; ++i) {
                const int c = tid + 256 * i;
                *reinterpret_cast<u32x4 *>(xs + c / (BM / E) * XW + c % (BM / E) * E) = xr[i];
            }
#pragma unroll
            for (int i = 0; i < YL; ++i) {
                const int c = tid + 256 * i;
                *reinterpret_cast<u32x4 *>(ys + c / (BN / E) * YW + c % (BN / E) * E) = yr[i];
            }
            T *to = (tid < 128 ? xs + BM + rank_row * XW : ys + BN + rank_row * YW) + rank_at;
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<u32x4 *>(to) = lr;
            } else {
                bf16x4 high, rest;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    __bf16 h, r;
                    split(__uint_as_float(lr[i]), h, r);
                    high[i] = h;
                    rest[i] = r;
                }
                *reinterpret_cast<bf16x4 *>(to) = high;
                *reinterpret_cast<bf16x4 *>(to + 16) = rest;
            }
            __syncthreads();
            const bool ends = r0 + R >= count;
            int id_ahead = 0;
            if (ends && t + 2 < last && tid < kTileRows) id_ahead = id_at(ahead2);
            if (!ends || t + 1 < last) fetch(ends ? ahead : now, ids[ends ? next : slot], ends ? 0 : r0 + R);
#pragma unroll
            for (int r = 0; r < R; r += STEP) {
                if (WANT_W) {
                    Frag<T> yf[NI];
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) {
                        yf[ni].columns(ys, YW, (wn * NI + ni) * 16, r, lane);
                        if (wm == 0 && a.all.db) sums[WANT_W ? ni : 0] += yf[ni].sum();
                    }
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi) {
                        Frag<T> xf;
                        xf.columns(xs, XW, (wm * MI + mi) * 16, r, lane);
#pragma unroll
                        for (int ni = 0; ni < NI; ++ni)
                            acc[WANT_W ? mi : 0][WANT_W ? ni : 0] = mma(yf[ni], xf, acc[WANT_W ? mi : 0][WANT_W ? ni : 0]);
                    }
                }
                if (now.type == unknown) continue;
                // the waves share the blocks of x's and of dy's columns between them
                Frag<T> lf;
                lf.columns(ys, YW, BN, r, lane);
#pragma unroll
                for (int i = 0; i < MI / 2; ++i) {
                    Frag<T> xf;
                    xf.columns(xs, XW, (wave * MI / 2 + i) * 16, r, lane);
                    acc_down[i] = mma(lf, xf, acc_down[i]);
                    if constexpr (sizeof(T) == 2) {
                        Frag<T> rest;
                        rest.columns(ys, YW, BN + 16, r, lane);
                        acc_down[i] = mma(rest, xf, acc_down[i]);
                    }
                }
                lf.columns(xs, XW, BM, r, lane);
#pragma unroll
                for (int i = 0; i < NI / 2; ++i) {
                    Frag<T> yf;
                    yf.columns(ys, YW, (wave * NI / 2 + i) * 16, r, lane);
                    acc_up[i] = mma(yf, lf, acc_up[i]);
                    if constexpr (sizeof(T) == 2) {
                        Frag<T> rest;
                        rest.columns(xs, XW, BM + 16, r, lane);
                        acc_up[i] = mma(yf, rest, acc_up[i]);
                    }
                }
            }
            if (ends && tid < kTileRows) ids[free][tid] = id_ahead;
        }
        slot = next;
        at = ahead;
        ahead = ahead2;
        if (t + 3 < last) ahead2 = tile_behind(g.plan, ahead2);
        if ((t + 1 < last && at.type == now.type) || now.type == unknown) continue;
        // the type or the range ends here: the type's sums are whole, or one range's share of them
        const int type_first = plan_word(g.plan.tile_first, now.type);
        const int type_last = plan_word(g.plan.tile_first, now.type + 1);
        const bool whole = type_first >= first && type_last <= last;
        float *part = g.partial + (int64_t)(2 * range + (type_first >= first)) * g.stride;
#pragma unroll
        for (int i = 0; i < MI / 2; ++i) {
            // lane: rank columns 4 (lane / 16) .. + 3 of row k
            const int k = (wave * MI / 2 + i) * 16 + (lane & 15), j = 4 * (lane >> 4);
            const bool vec = (a.rank & 3) == 0;
            if (k < g.K && whole)
                store4((T *)g.dw + (int64_t)now.type * g.first + k * a.rank + j, acc_down[i], a.rank - j, vec);
            else if (k < g.K)
                store4(part + k * a.rank + j, acc_down[i], a.rank - j, vec);
            acc_down[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int i = 0; i < NI / 2; ++i) {
            // lane: columns n .. n + 3 of rank row j
            const int j = lane & 15, n = (wave * NI / 2 + i) * 16 + 4 * (lane >> 4);
            const bool vec = (g.N & 3) == 0;
            if (j < a.rank && whole)
                store4((T *)g.db + (int64_t)now.type * g.second + j * g.N + n, acc_up[i], g.N - n, vec);
            else if (j < a.rank)
                store4(part + g.second_at + j * g.N + n, acc_up[i], g.N - n, vec);
            acc_up[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    if (WANT_W) {
        const GradArgs &w = a.all;
        const bool whole = ranges == 1;
        float *part = w.partial + (int64_t)(2 * range + (range == 0)) * w.stride;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            const int k = (wm * MI + mi) * 16 + (lane & 15);
            if (k >= w.K || !w.dw) continue;
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                const int n = (wn * NI + ni) * 16 + 4 * (lane >> 4);
                const bool vec = (w.N & 3) == 0;
                const f32x4 v = acc[WANT_W ? mi : 0][WANT_W ? ni : 0];
                if (whole)
                    store4((T *)w.dw + (int64_t)k * w.N + n, v, w.N - n, vec);
                else
                    store4(part + (int64_t)k * w.N + n, v, w.N - n, vec);
            }
        }
        if (wm == 0 && w.db) {
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                float s = sums[WANT_W ? ni : 0];
                s += __shfl_xor(s, 16);
                s += __shfl_xor(s, 32);
                const int n = (wn * NI + ni) * 16 + lane;
                if (lane < 16 && n < w.N) {
                    if (whole)
                        ((T *)w.db)[n] = (T)s;
                    else
                        part[w.second_at + n] = s;
                }
            }
        }
    }
}

// Joins the ranges of a type in their order: the workgroup's waves sum an equal share of them each, 256
// elements at a time.  Types without rows get zeros; types inside one range are done.  `first_block`: of the
// workgroups of all types, where this launch's begin.
template <typename T>
__global__ __launch_bounds__(1024) void grad_join_kernel(GradArgs a, uint64_t first_block) {
    __shared__ f32x4 part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const uint64_t blocks = (uint64_t)(a.stride + 255) / 256, block = first_block + blockIdx.x;
    const int type = (int)(block / blocks);
    const int64_t at = (int64_t)(block % blocks) * 256 + lane * 4;
    const int tiles = a.plan.rows ? grad_tiles(a) : 0;  // no rows: no plan
    const int type_first = a.shared || !tiles ? 0 : a.plan.tile_first[type];
    const int type_last = a.shared || !tiles ? tiles : a.plan.tile_first[type + 1];
    int first = 0, count = 0;  // the ranges it lies in
    if (type_last > type_first) {
        const uint32_t ranges = min(a.ranges, (uint32_t)tiles);
        first = range_of(type_first, tiles, ranges);
        count = range_of(type_last - 1, tiles, ranges) - first + 1;
        if (count == 1) return;
    }
    const int share = (count + waves - 1) / waves;
    const int from = first + min(count, wave * share), to = first + min(count, (wave + 1) * share);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (at < a.stride) {
#pragma unroll 8
        for (int r = from; r < to; ++r)  // its first range holds it behind other types
            sum += *reinterpret_cast<const f32x4 *>(a.partial + (int64_t)(2 * r + (r == first)) * a.stride + at);
    }
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < waves; ++w) sum += part[w][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t e = at + i, f = e - a.second_at;
            if (e < a.first)
                ((T *)a.dw)[(int64_t)type * a.first + e] = (T)sum[i];
            else if (f >= 0 && f < a.second && a.db)
                ((T *)a.db)[(int64_t)type * a.second + f] = (T)sum[i];
        }
    }
}

}  // namespace gn2v
