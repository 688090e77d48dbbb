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
constexpr int kSmallPlan = 1024;  // rows one workgroup sorts in LDS

// ------------------------------------------------------------------------------------ the plan
// int32 words: order[rows] (row id at every position), row_types[rows] (type at every position;
// n_types = unknown: any id outside [0, n_types); those rows come last), offsets[n_types + 2]
// (first position of every type, of the unknown rows, rows), tiles[2 * tile_bound] (type, first
// position) with type -1 behind the last one.
struct PlanView {
    int *order, *row_types, *offsets;
    int2 *tiles;
    uint32_t rows, types, tile_bound;
};

template <typename I>
__device__ __forceinline__ int type_at(const I *types, uint32_t row, uint32_t n_types) {
    const I t = types[row];
    return t >= 0 && (uint64_t)t < (uint64_t)n_types ? (int)t : (int)n_types;
}

// Up to 1 024 rows: one workgroup sorts (type << 10 | row) in LDS -- a launch instead of four.
template <typename I>
__global__ __launch_bounds__(kSmallPlan) void plan_small_kernel(const I *__restrict__ types, PlanView p) {
    __shared__ uint32_t key[kSmallPlan];
    __shared__ int wave_sum[kSmallPlan / 64];
    const uint32_t i = threadIdx.x;
    key[i] = i < p.rows ? (uint32_t)type_at(types, i, p.types) << 10 | i : 0xFFFFFFFFu;
    uint32_t n = 64;  // every wave takes part; the sort covers the smallest power of two
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
    uint32_t type = 0;
    if (i < p.rows) {
        type = key[i] >> 10;
        p.order[i] = (int)(key[i] & 1023u);
        p.row_types[i] = (int)type;
        starts = (i - first_of(type)) % kTileRows == 0;
    }
    for (uint32_t t = i; t < p.types + 2; t += kSmallPlan)
        p.offsets[t] = t <= p.types ? (int)first_of(t) : (int)p.rows;
    const unsigned long long ballot = __ballot(starts);
    if ((i & 63) == 0) wave_sum[i >> 6] = __popcll(ballot);
    __syncthreads();
    int at = 0, total = 0;
    for (uint32_t w = 0; w < kSmallPlan / 64; ++w) {
        if (w < i >> 6) at += wave_sum[w];
        total += wave_sum[w];
    }
    at += __popcll(ballot & ((1ull << (i & 63)) - 1));
    if (starts) p.tiles[at] = make_int2((int)type, (int)i);
    for (uint32_t t = i; t < p.tile_bound; t += kSmallPlan)
        if (t >= (uint32_t)total) p.tiles[t] = make_int2(-1, 0);
}

// More rows: one wave per stripe of rows counts its types in LDS, the counts are scanned per type and
// over the types, and the same wave places its rows.  Equal types keep their rows' order (a wave
// ranks its 64 rows by ballots over the bits of their types), so sums over a type's rows have the
// same order in every run.
template <typename I>
__global__ __launch_bounds__(64) void plan_count_kernel(const I *__restrict__ types, uint32_t rows,
                                                        uint32_t n_types, uint32_t stripe,
                                                        uint32_t stripes, int *__restrict__ counts) {
    extern __shared__ int count[];
    for (uint32_t t = threadIdx.x; t <= n_types; t += 64) count[t] = 0;
    __syncthreads();
    const uint64_t first = (uint64_t)blockIdx.x * stripe;
    const uint64_t last = first + stripe < rows ? first + stripe : rows;
    for (uint64_t r = first + threadIdx.x; r < last; r += 64)
        atomicAdd(&count[type_at(types, (uint32_t)r, n_types)], 1);
    __syncthreads();
    for (uint32_t t = threadIdx.x; t <= n_types; t += 64)
        counts[(uint64_t)t * stripes + blockIdx.x] = count[t];
}

// counts[type][stripe] -> exclusive sums over the stripes; totals[type]
__global__ __launch_bounds__(256) void plan_scan_kernel(int *__restrict__ counts, uint32_t stripes,
                                                        int *__restrict__ totals) {
    __shared__ int wave_sum[4];
    int *row = counts + (uint64_t)blockIdx.x * stripes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int carry = 0;
    for (uint32_t first = 0; first < stripes; first += 256) {
        const uint32_t i = first + threadIdx.x;
        const int own = i < stripes ? row[i] : 0;
        int sum = own;
        for (int step = 1; step < 64; step <<= 1) {
            const int other = __shfl_up(sum, step);
            if (lane >= step) sum += other;
        }
        if (lane == 63) wave_sum[wave] = sum;
        __syncthreads();
        int before = carry;
        for (int w = 0; w < wave; ++w) before += wave_sum[w];
        if (i < stripes) row[i] = before + sum - own;
        carry += wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Pieces of at most `piece` consecutive positions of one type, as (type, first position), -1 behind
// the last; first[t] = pieces before type t.  With `totals` the offsets are made from them first.
// One workgroup; `groups` = the types and, for a plan's tiles, the unknown rows.
__global__ __launch_bounds__(1024) void plan_pieces_kernel(const int *__restrict__ totals, int *offsets,
                                                           uint32_t groups, uint32_t piece,
                                                           uint32_t bound, int2 *__restrict__ pieces,
                                                           int *__restrict__ first) {
    __shared__ int sums[2][16];
    __shared__ int carry[2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x < 2) carry[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t base = 0; base < groups; base += 1024) {
        const uint32_t t = base + threadIdx.x;
        const int own = t >= groups ? 0 : totals ? totals[t] : offsets[t + 1] - offsets[t];
        const int own_pieces = (int)(((uint32_t)own + piece - 1) / piece);
        int rows = own, count = own_pieces;
        for (int step = 1; step < 64; step <<= 1) {
            const int a = __shfl_up(rows, step), b = __shfl_up(count, step);
            if (lane >= step) {
                rows += a;
                count += b;
            }
        }
        if (lane == 63) {
            sums[0][wave] = rows;
            sums[1][wave] = count;
        }
        __syncthreads();
        int before = carry[0], before_pieces = carry[1];
        for (int w = 0; w < wave; ++w) {
            before += sums[0][w];
            before_pieces += sums[1][w];
        }
        const int start = before + rows - own, at = before_pieces + count - own_pieces;
        if (t < groups) {
            if (totals) offsets[t] = start;
            if (first) first[t] = at;
        }
        const int from = totals ? start : (t < groups ? offsets[t] : 0);
        // a wave lists its 64 types one after the other: a type may hold all the pieces
        for (int l = 0; l < 64; ++l) {
            const int n = __shfl(own_pieces, l);
            if (n == 0) continue;
            const int type = __shfl((int)t, l), f = __shfl(from, l), a = __shfl(at, l);
            for (int i = lane; i < n; i += 64)
                pieces[a + i] = make_int2(type, f + (int)((uint32_t)i * piece));
        }
        __syncthreads();
        if (threadIdx.x == 0)
            for (int w = 0; w < 16; ++w) {
                carry[0] += sums[0][w];
                carry[1] += sums[1][w];
            }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (totals) offsets[groups] = carry[0];
        if (first) first[groups] = carry[1];
    }
    for (uint32_t i = (uint32_t)carry[1] + threadIdx.x; i < bound; i += 1024)
        pieces[i] = make_int2(-1, 0);
}

template <typename I>
__global__ __launch_bounds__(64) void plan_place_kernel(const I *__restrict__ types, PlanView p,
                                                        uint32_t stripe, uint32_t stripes,
                                                        const int *__restrict__ counts, int bits) {
    extern __shared__ int next[];
    for (uint32_t t = threadIdx.x; t <= p.types; t += 64)
        next[t] = p.offsets[t] + counts[(uint64_t)t * stripes + blockIdx.x];
    __syncthreads();
    const uint64_t first = (uint64_t)blockIdx.x * stripe;
    const uint64_t last = first + stripe < p.rows ? first + stripe : p.rows;
    for (uint64_t base = first; base < last; base += 64) {
        const uint64_t r = base + threadIdx.x;
        const bool live = r < last;
        const int type = live ? type_at(types, (uint32_t)r, p.types) : 0;
        unsigned long long same = __ballot(live);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot(type >> b & 1);
            same &= type >> b & 1 ? set : ~set;
        }
        const unsigned long long below = same & ((1ull << threadIdx.x) - 1);
        if (live) {
            const int at = next[type] + __popcll(below);
            p.order[at] = (int)r;
            p.row_types[at] = type;
        }
        __syncthreads();  // every lane has read its counter
        if (live && below == 0) next[type] += __popcll(same);
        __syncthreads();
    }
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

// 16 bytes of a row, zeros from element `valid` on.  `align`: bytes the row's address is a multiple of.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T *p, int valid, int align) {
    constexpr int E = Tile<T>::kChunk;
    u32x4 v = {0, 0, 0, 0};
    if (valid >= E) {
        if (align == 16) return *reinterpret_cast<const u32x4 *>(p);
        if (align == 8) {
            const uint2 a = reinterpret_cast<const uint2 *>(p)[0];
            const uint2 b = reinterpret_cast<const uint2 *>(p)[1];
            return u32x4{a.x, a.y, b.x, b.y};
        }
        if (align == 4) {
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

__device__ __forceinline__ bf16x4 read_transposed(const __bf16 *p) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(p));
    return __builtin_bit_cast(bf16x4, v);
}
__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
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
    // rows of outer elements: s[inner][outer]
    __device__ __forceinline__ void columns(const float *s, int stride, int outer, int inner, int lane) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = s[(inner + 4 * (lane >> 4) + i) * stride + outer + (lane & 15)];
    }
    __device__ __forceinline__ float sum() const { return (v[0] + v[1]) + (v[2] + v[3]); }
};
template <> struct Frag<__bf16> {
    bf16x8 v;
    __device__ __forceinline__ void rows(const __bf16 *s, int stride, int outer, int inner, int lane) {
        const __bf16 *p = s + (outer + (lane & 15)) * stride + inner + 4 * (lane >> 4);
        v = join(*reinterpret_cast<const bf16x4 *>(p), *reinterpret_cast<const bf16x4 *>(p + 16));
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
    int align;
};

struct ProductArgs {
    const void *x;
    int64_t ldx;
    int x_align;
    WeightView w;
    const void *bias;  // [type][N] or [N] (adapted form), may be NULL
    int64_t bias_type;
    void *y;           // rows at their ids; `sorted`: float32 rows at their positions
    int64_t ldy;
    int y_vec, sorted;
    float scale;       // of the product (before the bias)
    PlanView plan;
    int K, N;
    // adapted form: low[position][rank] float32 times the `up` weights of the row's type
    const float *low;
    int rank;
    WeightView up;
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
template <typename T, int BN, bool WT, bool ADAPT>
__global__ __launch_bounds__(256) void product_kernel(ProductArgs a) {
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
    const uint32_t tiles = ADAPT ? (a.plan.rows + 63) / 64 : a.plan.tile_bound;
    if (!tile_of_block(tiles, (uint32_t)((a.N + BN - 1) / BN), &tile, &column)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = (int)column * BN;
    int type = 0, start, count;
    if (ADAPT) {
        start = (int)(tile * 64);
        count = min(64, (int)(a.plan.rows - tile * 64));
    } else {
        const int2 t = a.plan.tiles[tile];
        type = t.x;
        start = t.y;
        if (type < 0) return;
        count = min(64, a.plan.offsets[type + 1] - start);
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
                xr[i] = row < count
                            ? load_chunk((const T *)a.x + (int64_t)ids[row] * a.ldx + k, a.K - k, a.x_align)
                            : u32x4{0, 0, 0, 0};
            }
        };
        auto fetch_w = [&](const T *p, const WeightView &v, int k0, int depth) {
#pragma unroll
            for (int i = 0; i < WL; ++i) {
                const int c = tid + 256 * i;
                if (WT) {
                    const int n = c / (BK / E), k = k0 + c % (BK / E) * E;
                    wr[i] = n0 + n < a.N ? load_chunk(p + (int64_t)(n0 + n) * v.outer + k, depth - k, v.align)
                                         : u32x4{0, 0, 0, 0};
                } else {
                    const int k = k0 + c / (BN / E), n = n0 + c % (BN / E) * E;
                    wr[i] = k < depth ? load_chunk(p + (int64_t)k * v.inner + n, a.N - n, v.align)
                                      : u32x4{0, 0, 0, 0};
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
            if (__popcll(runs) <= 4) {
                // Few runs: 32 rank columns at a time, rows of other types zero.  In bfloat16 the
                // low-rank rows enter as a high and a low part, 16 bits of them together.
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
                                const __bf16 high = to_bf16(v);
                                xs[row * XS + (i & 31)] = high;
                                xs[row * XS + 32 + (i & 31)] = to_bf16(v - (float)high);
                            }
                        }
                        put_w();
                        __syncthreads();
#pragma unroll
                        for (int slab = 0; slab < 2; ++slab) {
                            if (sizeof(T) == 4 && j0 + slab * 16 >= a.rank) break;
                            Frag<T> xf[MI], wf[NI];
#pragma unroll
                            for (int mi = 0; mi < MI; ++mi)
                                xf[mi].rows(xs, XS, m0 + mi * 16, slab * SLAB, lane);
#pragma unroll
                            for (int ni = 0; ni < NI; ++ni) weights(wf[ni], ni, sizeof(T) == 4 ? slab * SLAB : 0);
#pragma unroll
                            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                                for (int ni = 0; ni < NI; ++ni)
                                    acc[mi][ni] = mma(wf[ni], xf[mi], acc[mi][ni]);
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
                store4((float *)a.y + (int64_t)(start + row) * a.ldy + n, v, a.N - n, a.y_vec);
            else
                store4((T *)a.y + (int64_t)ids[row] * a.ldy + n, v, a.N - n, a.y_vec);
        }
    }
}

// --------------------------------------------------------------------------------- few rows
// One workgroup per row and 64 columns: lanes read 16 bytes of a weight row each, the workgroup's
// 256 / (64 / kChunk) row groups split the inner axis and are joined in LDS.  No plan, one launch.
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
            const u32x4 q = load_chunk(w + (int64_t)k * v.inner + n0 + c, a.N - n0 - c, v.align);
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
        if (a.bias) s += (float)((const T *)a.bias)[(ADAPT ? 0 : (int64_t)type * a.bias_type) + n0 + tid];
        y[n0 + tid] = (T)s;
    }
}

// ------------------------------------------------------------------------- weights' gradients
// dW[t] = sum over the rows of type t of x[r]^T dy[r].  The row axis is cut into chunks; a workgroup
// adds one chunk's outer products of a block of dW in registers, a second launch joins the chunks of
// a type in their order (no atomics: the same bits in every run).  A type of one chunk is written at
// once.  Either operand may be float32 rows at their positions (the low-rank rows), which enter
// bfloat16 products as a high and a low part.
struct GradArgs {
    const void *x, *dy;
    int64_t ldx, ldy;
    int x_align, y_align;
    const int *order;    // NULL: rows at their positions
    const int2 *chunks;  // NULL: one group of all rows
    const int *first, *offsets;
    uint32_t rows, types, chunk_rows, chunk_bound;
    int K, N;
    float *partial;  // [chunk][stride]: K * N products, then N column sums
    int64_t stride;
    void *dw;        // [type][K][N], may be NULL when only the bias is asked for (K = 0)
    void *db;        // [type][N] or NULL
};

template <typename T, int MI, int NI, bool XLOW, bool YLOW>
__global__ __launch_bounds__(256) void grad_kernel(GradArgs a) {
    constexpr int E = Tile<T>::kChunk, R = Tile<T>::kDepth, STEP = Tile<T>::kSlab;
    constexpr int BM = 32 * MI, BN = 32 * NI;
    constexpr bool SPLITX = XLOW && sizeof(T) == 2, SPLITY = YLOW && sizeof(T) == 2;
    // row strides that keep the four lane groups, four rows apart, in different banks: 4 words more
    // than a multiple of 32 (float), 8 words more (bfloat16, read in transposed blocks of 4 rows)
    constexpr int PAD = sizeof(T) == 4 ? 4 : 16;
    constexpr int XW = BM * (SPLITX ? 2 : 1) + PAD, YW = BN * (SPLITY ? 2 : 1) + PAD;
    constexpr int XL = R * BM / E / 256, YL = R * BN / E / 256;
    static_assert(XL >= 1 && YL >= 1, "a block of at least 32 x 32");
    __shared__ __align__(16) T xs[R * XW];
    __shared__ __align__(16) T ys[R * YW];
    __shared__ int ids[2][R];
    const uint32_t kb = a.K > 0 ? (uint32_t)((a.K + BM - 1) / BM) : 1, nb = (uint32_t)((a.N + BN - 1) / BN);
    uint32_t chunk, block;
    if (!tile_of_block(a.chunk_bound, kb * nb, &chunk, &block)) return;
    const int k0 = (int)(block / nb) * BM, n0 = (int)(block % nb) * BN;
    int type = 0, start, last, chunks;
    if (a.chunks) {
        const int2 c = a.chunks[chunk];
        type = c.x;
        if (type < 0) return;
        start = c.y;
        last = a.offsets[type + 1];
        chunks = a.first[type + 1] - a.first[type];
    } else {
        start = (int)(chunk * a.chunk_rows);
        last = (int)a.rows;
        chunks = (int)a.chunk_bound;
    }
    last = last - start < (int)a.chunk_rows ? last : start + (int)a.chunk_rows;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1;
    f32x4 acc[MI][NI] = {};
    float sums[NI] = {};
    const bool want_sums = a.db && k0 == 0 && wm == 0;
    auto fetch_id = [&](int p) { return p < last ? (a.order ? a.order[p] : p) : 0; };
    u32x4 xr[XL], yr[YL], xr2[SPLITX ? XL : 1], yr2[SPLITY ? YL : 1];
    // float32 rows in a bfloat16 product: 8 floats -> 8 high and 8 low parts
    auto fetch_low = [&](const float *p, int valid, int align, u32x4 &high, u32x4 &low) {
        const u32x4 q0 = load_chunk(p, valid, align), q1 = load_chunk(p + 4, valid - 4, align);
        bf16x8 h, l;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = __uint_as_float(i < 4 ? q0[i & 3] : q1[i & 3]);
            h[i] = to_bf16(v);
            l[i] = to_bf16(v - (float)h[i]);
        }
        high = __builtin_bit_cast(u32x4, h);
        low = __builtin_bit_cast(u32x4, l);
    };
    auto fetch = [&](int p0, const int *id) {
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int c = tid + 256 * i, row = c / (BM / E), k = k0 + c % (BM / E) * E;
            const bool live = p0 + row < last && k < a.K;
            xr[i] = u32x4{0, 0, 0, 0};
            if constexpr (SPLITX) {
                xr2[i] = u32x4{0, 0, 0, 0};
                if (live)
                    fetch_low((const float *)a.x + (int64_t)(p0 + row) * a.ldx + k, a.K - k, a.x_align, xr[i], xr2[i]);
            } else if (live) {
                xr[i] = load_chunk((const T *)a.x + (int64_t)(XLOW ? p0 + row : id[row]) * a.ldx + k, a.K - k, a.x_align);
            }
        }
#pragma unroll
        for (int i = 0; i < YL; ++i) {
            const int c = tid + 256 * i, row = c / (BN / E), n = n0 + c % (BN / E) * E;
            const bool live = p0 + row < last && n < a.N;
            yr[i] = u32x4{0, 0, 0, 0};
            if constexpr (SPLITY) {
                yr2[i] = u32x4{0, 0, 0, 0};
                if (live)
                    fetch_low((const float *)a.dy + (int64_t)(p0 + row) * a.ldy + n, a.N - n, a.y_align, yr[i], yr2[i]);
            } else if (live) {
                yr[i] = load_chunk((const T *)a.dy + (int64_t)(YLOW ? p0 + row : id[row]) * a.ldy + n, a.N - n, a.y_align);
            }
        }
    };
    if (tid < R) {
        ids[0][tid] = fetch_id(start + tid);
        ids[1][tid] = fetch_id(start + R + tid);
    }
    __syncthreads();
    fetch(start, ids[0]);
    int next = 1;
    for (int p0 = start; p0 < last; p0 += R) {
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
        int ahead = 0;
        if (p0 + R < last) {
            fetch(p0 + R, ids[next]);
            if (tid < R) ahead = fetch_id(p0 + 2 * R + tid);
        }
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
        __syncthreads();
        next ^= 1;
        if (tid < R) ids[next][tid] = ahead;  // the ids used last are free: `fetch` of the stage after next
    }
    // lane: row k = lane % 16 of the block, four consecutive columns n
    float *part = a.partial + (int64_t)chunk * a.stride;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const int k = k0 + wm * MI * 16 + mi * 16 + (lane & 15);
        if (k >= a.K) continue;
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) {
            const int n = n0 + wn * NI * 16 + ni * 16 + 4 * (lane >> 4);
            const bool vec = (a.N & 3) == 0;
            if (chunks == 1)
                store4((T *)a.dw + ((int64_t)type * a.K + k) * a.N + n, acc[mi][ni], a.N - n, vec);
            else
                store4(part + (int64_t)k * a.N + n, acc[mi][ni], a.N - n, vec);
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
                if (chunks == 1)
                    ((T *)a.db)[(int64_t)type * a.N + n] = (T)s;
                else
                    part[(int64_t)a.K * a.N + n] = s;
            }
        }
    }
}

// Joins the chunks of a type in their order: sixteen waves sum a sixteenth of them each, 256 elements
// at a time.  Types without rows get zeros; types of one chunk are done.
template <typename T>
__global__ __launch_bounds__(1024) void grad_join_kernel(GradArgs a) {
    __shared__ f32x4 part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t blocks = (a.stride + 255) / 256;
    const int type = (int)(blockIdx.x / blocks);
    const int64_t at = (int64_t)(blockIdx.x % blocks) * 256 + lane * 4;
    const int first = a.chunks ? a.first[type] : 0;
    const int count = a.chunks ? a.first[type + 1] - first : (int)a.chunk_bound;
    if (count == 1) return;
    const int share = (count + 15) / 16;
    const int from = first + min(count, wave * share), to = first + min(count, (wave + 1) * share);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (at < a.stride) {
#pragma unroll 8
        for (int c = from; c < to; ++c)
            sum += *reinterpret_cast<const f32x4 *>(a.partial + (int64_t)c * a.stride + at);
    }
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < 16; ++w) sum += part[w][lane];
        const int64_t weights = (int64_t)a.K * a.N;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t e = at + i;
            if (e < weights)
                ((T *)a.dw)[(int64_t)type * weights + e] = (T)sum[i];
            else if (e < weights + a.N && a.db)
                ((T *)a.db)[(int64_t)type * a.N + e - weights] = (T)sum[i];
        }
    }
}

}  // namespace gn2v
