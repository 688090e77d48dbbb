// Embedding tables held in 8 bits: codes u8[rows][stride] (int8 or OCP e4m3) and one float32 scale per
// row and group of `group` consecutive columns.  Written rows are quantised on the way in, rows are
// read back as float32 / bfloat16, and the edge operators read their two rows in this form: a gathered
// row of 128 columns is 128 + 4 * groups bytes instead of 512.
//
//   scale = max(float32(max |x| * float32(1 / largest code value)), 2^-90),   code = x / scale rounded ONCE
//   to the nearest code, ties to even;   value = float32(code * scale).
// The scale is off by a last bit or two from the quotient, and the largest |x| / scale then from the largest
// code value, to which it is rounded all the same.
// A group that holds an infinity or a NaN gets the scale NaN: all of it reads back as NaN.
#pragma once
#include "edge_kernels.h"
#include "typed_kernels.h"

namespace gn2v {

enum CodeType : uint32_t { kInt8 = 0, kE4m3 = 1 };

struct TableView {
    uint8_t *codes;
    float *scales;
    uint64_t rows;
    uint32_t d, stride, group_shift, groups;  // stride: bytes, a multiple of 16
};

// x / scale, rounded to float32 so that a second rounding to fewer bits is that of the exact quotient
// (round to odd: where the division is inexact, the neighbour with an odd last bit that encloses it).
// `inverse` = 1 / scale: the product with it, corrected once, is off by less than its last bit, and the
// remainder then says on which side.  Remainders are exact: the scale is at least 2^-90, so its last bit
// does not underflow where a code's border can lie.
__device__ __forceinline__ float divide_to_odd(float x, float scale, float inverse) {
    const float near = x * inverse;
    const float q = __fmaf_rn(__fmaf_rn(-near, scale, x), inverse, near);
    const float r = __fmaf_rn(-q, scale, x);
    uint32_t bits = __float_as_uint(q);
    // the exact quotient lies above |q| when the remainder has x's sign
    const uint32_t towards = (__float_as_uint(r) ^ __float_as_uint(x)) >> 31 ? 0xFFFFFFFFu : 1u;
    if (r != 0.f && !(bits & 1u) && (bits << 1) != 0) bits += towards;
    return __uint_as_float(bits);
}

// four consecutive codes to a word
template <uint32_t CODE>
__device__ __forceinline__ uint32_t encode4(const float *x, float scale, float inverse) {
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = divide_to_odd(x[i], scale, inverse);
    if constexpr (CODE == kInt8) {
        uint32_t out = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) out |= ((uint32_t)(int)rintf(q[i]) & 255u) << (8 * i);
        return out;
    } else {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    }
}

template <uint32_t CODE>
__device__ __forceinline__ void decode4(uint32_t w, float scale, float *v) {
    // a value is the rounded product wherever it is used: a fused multiply-add behind it would give the
    // difference of a row with itself another value than zero
#pragma clang fp contract(off)
    if constexpr (CODE == kInt8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> (8 * i)) * scale;
    } else {
        v[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * scale;
        v[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * scale;
        v[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * scale;
        v[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * scale;
    }
}

// row id of entry i: -1 where it lies outside the table (such rows are not written, and read as zeros)
__device__ __forceinline__ int64_t table_row(const void *ids, int id_bytes, uint64_t i, uint64_t rows) {
    if (!ids) return i < rows ? (int64_t)i : -1;
    const int64_t r = id_bytes == 8 ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i];
    return r >= 0 && (uint64_t)r < rows ? r : -1;
}

// the rows of entries first, first + step, ... (U of them; -1 behind the last entry): all ids are under
// way before one is looked at
template <int U>
__device__ __forceinline__ void table_rows(const void *ids, int id_bytes, uint64_t first, uint64_t step,
                                           uint64_t n, uint64_t rows, int64_t *r) {
    int64_t id[U];
    if (!ids) {
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = (int64_t)(first + u * step);
    } else if (id_bytes == 8) {
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = ((const int64_t *)ids)[min(first + u * step, n - 1)];
    } else {
        int32_t half[U];
#pragma unroll
        for (int u = 0; u < U; ++u) half[u] = ((const int32_t *)ids)[min(first + u * step, n - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = half[u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        r[u] = first + u * step < n && id[u] >= 0 && (uint64_t)id[u] < rows ? id[u] : -1;
}

// Columns a lane takes: 16 bytes of the float32 / bfloat16 row, so that what the lanes of a row load or
// store at once is contiguous.
template <typename T> constexpr int kColumns = Tile<T>::kChunk;

// elements c .. of a row of d as float32, zeros behind its end
__device__ __forceinline__ void widen(const u32x4 &q, float *v, float) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(q[i]);
}
__device__ __forceinline__ void widen(const u32x4 &q, float *v, __bf16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(i & 1 ? q[i / 2] & 0xFFFF0000u : q[i / 2] << 16);
}

// ---- writing.  The same row twice in one call: the last entry wins, whatever the order the
// workgroups run in.  A few entries: every entry looks at the ones behind it.  More: three launches
// over a scratch word per table row (cleared, the highest entry, the write).  Rows of 128 floats, scratch
// against looking: 256 entries 7.4 / 5.6 us, 1 024 entries 8.0 / 9.7, 8 192 entries 9 / 69.
__global__ __launch_bounds__(256) void table_owner_kernel(const void *ids, int id_bytes, uint64_t n,
                                                          uint64_t rows, int *owner, int clear) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
        const int64_t r = table_row(ids, id_bytes, i, rows);
        if (r < 0) continue;
        if (clear)
            owner[r] = -1;
        else
            atomicMax(&owner[r], (int)i);
    }
}

// Rows and edges are taken kAhead at a time per group of lanes, so that the ids, then the rows of several
// are under way together: what bounds these kernels is how many lines a CU has on order.
constexpr int kAhead = 4;

// `lanes` lanes per row, a power of two up to 64.
template <typename T, uint32_t CODE>
__global__ __launch_bounds__(256) void table_write_kernel(TableView t, const T *__restrict__ values,
                                                          int64_t ldv, int mode, const void *ids,
                                                          int id_bytes, uint64_t n, const int *owner,
                                                          int lanes_shift) {
    constexpr int U = 2, C = kColumns<T>;  // encoding needs the registers that more rows would take
    const int lane = threadIdx.x & ((1 << lanes_shift) - 1);
    const uint64_t entries = ((uint64_t)gridDim.x * 256) >> lanes_shift;
    const uint64_t mine = ((uint64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_shift;
    // every lane of a wave runs the same number of steps: the reductions cross lanes
    const uint64_t steps = (n + entries * U - 1) / (entries * U);
    for (uint64_t s = 0; s < steps; ++s) {
        const uint64_t e0 = mine + s * U * entries;
        int64_t r[U];
        table_rows<U>(ids, id_bytes, e0, entries, n, t.rows, r);
        for (uint32_t c0 = 0; c0 < t.stride; c0 += (uint32_t)C << lanes_shift) {
            const uint32_t c = c0 + C * lane;
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                raw[u] = load_chunk(values + (int64_t)(e0 + u * entries) * ldv, (int)c, (int)t.d, mode,
                                    e0 + u * entries < n);
            if (ids && c0 == 0) {
                // a later entry of the same row takes it
                if (owner) {
                    int last[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) last[u] = r[u] >= 0 ? owner[r[u]] : 0;
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (r[u] >= 0 && last[u] != (int)(e0 + u * entries)) r[u] = -1;
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        int later = 0;
                        if (r[u] >= 0)
                            for (uint64_t j = e0 + u * entries + 1 + lane; j < n; j += 1u << lanes_shift)
                                later |= table_row(ids, id_bytes, j, t.rows) == r[u];
                        for (int step = 1; step < 1 << lanes_shift; step <<= 1) later |= __shfl_xor(later, step);
                        if (later) r[u] = -1;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[C];
                widen(raw[u], x, T());
                uint32_t top = 0;  // as bits: NaN lies above infinity above the numbers
#pragma unroll
                for (int k = 0; k < C; ++k) top = max(top, __float_as_uint(x[k]) & 0x7FFFFFFFu);
                // a group is 2 to 32 consecutive lanes of a row; rows narrower than it have fewer lanes
                for (int step = 1; step < 1 << lanes_shift && (uint32_t)(C * step) < 1u << t.group_shift; step <<= 1)
                    top = max(top, (uint32_t)__shfl_xor((int)top, step));
                if (r[u] < 0 || c >= t.stride) continue;
                const bool finite = top < 0x7F800000u;
                constexpr float largest = CODE == kInt8 ? 127.f : 448.f;
                const float scale = finite ? fmaxf(__uint_as_float(top) * (1.f / largest), 0x1p-90f) : __builtin_nanf("");
#pragma unroll
                for (int w = 0; w < C / 4; ++w)
                    reinterpret_cast<uint32_t *>(t.codes + (uint64_t)r[u] * t.stride + c)[w] =
                        finite ? encode4<CODE>(x + 4 * w, scale, 1.f / scale) : 0;
                if (c < t.d && (c & ((1u << t.group_shift) - 1)) == 0)
                    t.scales[(uint64_t)r[u] * t.groups + (c >> t.group_shift)] = scale;
            }
        }
    }
}

// codes c .. c + C - 1 of a row and their scale; zeros where there is no such row
template <int C>
struct Codes {
    uint32_t w[C / 4];
    float scale;
};
template <int C>
__device__ __forceinline__ Codes<C> load_codes(const TableView &t, int64_t r, uint32_t c) {
    Codes<C> q = {};
    if (r >= 0 && c < t.d) {
        const uint8_t *p = t.codes + (uint64_t)r * t.stride + c;
        if constexpr (C == 4) {
            q.w[0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            q.w[0] = v.x;
            q.w[C / 4 - 1] = v.y;
        }
        q.scale = t.scales[(uint64_t)r * t.groups + (c >> t.group_shift)];
    }
    return q;
}

// C consecutive output elements, `valid` of them inside the row
// (past the caches: nobody reads them here, the table's rows are read again; 1.2 M edges of 100 columns
// 161 -> 154 us)
__device__ __forceinline__ void store_columns(float *p, const float *v, int valid, int align) {
    if (align == 16 && valid >= 4) {
        __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4 *>(p));
        return;
    }
    store4(p, f32x4{v[0], v[1], v[2], v[3]}, valid, align == 16);
}
__device__ __forceinline__ void store_columns(__bf16 *p, const float *v, int valid, int align) {
    store8(p, v, valid, align);
}

template <typename T, uint32_t CODE>
__global__ __launch_bounds__(256) void table_read_kernel(TableView t, const void *ids, int id_bytes,
                                                         uint64_t n, T *__restrict__ out, int64_t ldo,
                                                         int align, int lanes_shift) {
    constexpr int U = kAhead, C = kColumns<T>;
    const int lane = threadIdx.x & ((1 << lanes_shift) - 1);
    const uint64_t entries = ((uint64_t)gridDim.x * 256) >> lanes_shift;
    for (uint64_t e0 = ((uint64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_shift; e0 < n; e0 += entries * U) {
        int64_t r[U];
        table_rows<U>(ids, id_bytes, e0, entries, n, t.rows, r);
        for (uint32_t c = C * lane; c < t.d; c += (uint32_t)C << lanes_shift) {
            Codes<C> q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = load_codes<C>(t, r[u], c);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (e0 + u * entries >= n) break;
                float v[C];
#pragma unroll
                for (int w = 0; w < C / 4; ++w) decode4<CODE>(q[u].w[w], q[u].scale, v + 4 * w);
                store_columns(out + (int64_t)(e0 + u * entries) * ldo + c, v, (int)(t.d - c), align);
            }
        }
    }
}

// ---- edges, both rows in 8 bits, the operator in float32
template <uint32_t METHOD>
__device__ __forceinline__ float edge_value(float a, float b) {
    if constexpr (METHOD == kHadamard) return a * b;
    if constexpr (METHOD == kSum) return a + b;
    if constexpr (METHOD == kAverage) return (a + b) / 2.f;
    if constexpr (METHOD == kL1) return a - b;
    if constexpr (METHOD == kAbsoluteL1) return fabsf(a - b);
    if constexpr (METHOD == kSquaredL2) return (a - b) * (a - b);
    if constexpr (METHOD == kL2) return sqrtf((a - b) * (a - b));
    if constexpr (METHOD == kMin) return fminf(a, b);
    if constexpr (METHOD == kMax) return fmaxf(a, b);
    return a;  // Concatenate: the source's half
}

template <uint32_t METHOD, uint32_t CODE>
__global__ __launch_bounds__(256) void table_edges_kernel(TableView src, TableView dst,
                                                          const void *src_ids, const void *dst_ids,
                                                          int id_bytes, uint64_t n,
                                                          float *__restrict__ out, int64_t ldo, int align,
                                                          int lanes_shift) {
    constexpr int U = kAhead;
    const int lane = threadIdx.x & ((1 << lanes_shift) - 1);
    const uint64_t edges = ((uint64_t)gridDim.x * 256) >> lanes_shift;
    for (uint64_t e0 = ((uint64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_shift; e0 < n; e0 += edges * U) {
        int64_t a[U], b[U];
        table_rows<U>(src_ids, id_bytes, e0, edges, n, src.rows, a);
        table_rows<U>(dst_ids, id_bytes, e0, edges, n, dst.rows, b);
        for (uint32_t c = 4 * lane; c < src.d; c += 4u << lanes_shift) {
            Codes<4> p[U], q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                p[u] = load_codes<4>(src, a[u], c);
                q[u] = load_codes<4>(dst, b[u], c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (e0 + u * edges >= n) break;
                float x[4], y[4], v[4];
                decode4<CODE>(p[u].w[0], p[u].scale, x);
                decode4<CODE>(q[u].w[0], q[u].scale, y);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = edge_value<METHOD>(x[i], y[i]);
                float *o = out + (int64_t)(e0 + u * edges) * ldo + c;
                store_columns(o, v, (int)(src.d - c), align);
                if constexpr (METHOD == kConcatenate) store_columns(o + src.d, y, (int)(src.d - c), align);
            }
        }
    }
}

// L2Distance and CosineSimilarity: sixteen columns per lane and step.  A lane's columns lie in one group
// of each row, so the cosine's sums are of codes -- whole numbers for int8, four products an
// instruction -- and scaled afterwards; distances need the values themselves.
template <uint32_t CODE>
__device__ __forceinline__ void dot16(const u32x4 &a, const u32x4 &b, float &ab, float &aa, float &bb) {
    if constexpr (CODE == kInt8) {
        int s = 0, p = 0, q = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s = __builtin_amdgcn_sdot4((int)a[i], (int)b[i], s, false);
            p = __builtin_amdgcn_sdot4((int)a[i], (int)a[i], p, false);
            q = __builtin_amdgcn_sdot4((int)b[i], (int)b[i], q, false);
        }
        ab = (float)s;
        aa = (float)p;
        bb = (float)q;
    } else {
        ab = aa = bb = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x2 x = h ? __builtin_amdgcn_cvt_pk_f32_fp8((int)a[i], true)
                                  : __builtin_amdgcn_cvt_pk_f32_fp8((int)a[i], false);
                const f32x2 y = h ? __builtin_amdgcn_cvt_pk_f32_fp8((int)b[i], true)
                                  : __builtin_amdgcn_cvt_pk_f32_fp8((int)b[i], false);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    ab = fmaf(x[k], y[k], ab);
                    aa = fmaf(x[k], x[k], aa);
                    bb = fmaf(y[k], y[k], bb);
                }
            }
        }
    }
}

struct Codes16 {
    u32x4 code;
    float scale;
};
__device__ __forceinline__ Codes16 load_codes16(const TableView &t, int64_t r, uint32_t c) {
    Codes16 q = {{0, 0, 0, 0}, 0.f};
    if (r >= 0 && c < t.d) {
        q.code = *reinterpret_cast<const u32x4 *>(t.codes + (uint64_t)r * t.stride + c);
        q.scale = t.scales[(uint64_t)r * t.groups + (c >> t.group_shift)];
    }
    return q;
}
// columns behind the last one count as zeros, whatever the row's padding holds
__device__ __forceinline__ void mask_codes16(Codes16 &q, int valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int v = min(max(valid - 4 * i, 0), 4);
        q.code[i] &= (uint32_t)((1ull << (8 * v)) - 1);
    }
}

template <uint32_t METHOD, uint32_t CODE>
__global__ __launch_bounds__(256) void table_scores_kernel(TableView src, TableView dst,
                                                           const void *src_ids, const void *dst_ids,
                                                           int id_bytes, uint64_t n,
                                                           float *__restrict__ out, int64_t ldo,
                                                           int lanes_shift) {
    constexpr int U = kAhead;
    const int lane = threadIdx.x & ((1 << lanes_shift) - 1);
    const uint64_t edges = ((uint64_t)gridDim.x * 256) >> lanes_shift;
    const uint64_t mine = ((uint64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_shift;
    // every lane of a wave runs the same number of steps: the reductions cross lanes
    const uint64_t steps = (n + edges * U - 1) / (edges * U);
    for (uint64_t s = 0; s < steps; ++s) {
        int64_t a[U], b[U];
        float ab[U] = {}, aa[U] = {}, bb[U] = {};
        table_rows<U>(src_ids, id_bytes, mine + s * U * edges, edges, n, src.rows, a);
        table_rows<U>(dst_ids, id_bytes, mine + s * U * edges, edges, n, dst.rows, b);
        for (uint32_t c = 16 * lane; c < src.d; c += 16u << lanes_shift) {
            Codes16 p[U], q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                p[u] = load_codes16(src, a[u], c);
                q[u] = load_codes16(dst, b[u], c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (src.d & 15u) {
                    mask_codes16(p[u], (int)(src.d - c));
                    mask_codes16(q[u], (int)(src.d - c));
                }
                if constexpr (METHOD == kCosineSimilarity) {
                    float x, y, z;
                    dot16<CODE>(p[u].code, q[u].code, x, y, z);
                    // one scale after the other, the smaller one first: the product of two may pass float32's
                    // largest number where the codes are zero (a NaN scale still reaches aa or bb)
                    ab[u] = fmaf(x * fminf(p[u].scale, q[u].scale), fmaxf(p[u].scale, q[u].scale), ab[u]);
                    aa[u] = fmaf(y * p[u].scale, p[u].scale, aa[u]);
                    bb[u] = fmaf(z * q[u].scale, q[u].scale, bb[u]);
                } else {
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        float x[4], y[4];
                        decode4<CODE>(p[u].code[h], p[u].scale, x);
                        decode4<CODE>(q[u].code[h], q[u].scale, y);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float d = x[i] - y[i];
                            ab[u] = fmaf(d, d, ab[u]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            for (int step = 1; step < 1 << lanes_shift; step <<= 1) {
                ab[u] += __shfl_xor(ab[u], step);
                if constexpr (METHOD == kCosineSimilarity) {
                    aa[u] += __shfl_xor(aa[u], step);
                    bb[u] += __shfl_xor(bb[u], step);
                }
            }
            const uint64_t e = mine + (s * U + u) * edges;
            if (e < n && lane == 0) {
                if constexpr (METHOD == kL2Distance) {
                    out[e * ldo] = sqrtf(ab[u]);
                } else {
                    const float norm = sqrtf(aa[u]) * sqrtf(bb[u]);
                    out[e * ldo] = ab[u] / (norm < 1e-6f ? 1e-6f : norm);  // NaN norms stay NaN
                }
            }
        }
    }
}

}  // namespace gn2v
