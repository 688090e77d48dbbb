// Embedding tables held in 8 bits: codes u8[rows][stride] (int8 or OCP e4m3) and one float32 scale per
// row and group of `group` consecutive columns.  Written rows are quantised on the way in, rows are
// read back as float32 / bfloat16, and the edge operators read their two rows in this form: a gathered
// row of 128 columns is 128 + 4 * groups bytes instead of 512.
//
//   scale = max(float32(max |x| / largest code value), 2^-90),   code = x / scale rounded ONCE to the
//   nearest code, ties to even;   value = float32(code * scale).
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
// (round to odd: where the division was inexact, the neighbour with an odd last bit that encloses it).
// The remainder is exact: the scale is at least 2^-90, so its last bit does not underflow where a
// code's border can lie.
__device__ __forceinline__ float divide_to_odd(float x, float scale) {
    const float q = x / scale;
    const float r = __fmaf_rn(-q, scale, x);
    uint32_t bits = __float_as_uint(q);
    if (r != 0.f && !(bits & 1u)) {
        // the exact quotient lies above |q| when the remainder has q's sign
        const bool larger = (r > 0.f) == (x > 0.f);
        if ((bits & 0x7FFFFFFFu) != 0) bits += larger ? 1u : -1u;
    }
    return __uint_as_float(bits);
}

template <uint32_t CODE>
__device__ __forceinline__ uint2 encode8(const float *x, float scale) {
    uint2 out = {0, 0};
    if constexpr (CODE == kInt8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = (int)rintf(divide_to_odd(x[i], scale));
            (i < 4 ? out.x : out.y) |= ((uint32_t)c & 255u) << (8 * (i & 3));
        }
    } else {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = divide_to_odd(x[i], scale);
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
        out.x = (uint32_t)lo;
        out.y = (uint32_t)hi;
    }
    return out;
}

template <uint32_t CODE>
__device__ __forceinline__ void decode8(uint2 c, float scale, float *v) {
    // a value is the rounded product wherever it is used: a fused multiply-add behind it would give the
    // difference of a row with itself another value than zero
#pragma clang fp contract(off)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t w = h ? c.y : c.x;
        float *o = v + 4 * h;
        if constexpr (CODE == kInt8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = (float)(int8_t)(w >> (8 * i)) * scale;
        } else {
            o[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * scale;
            o[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * scale;
            o[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * scale;
            o[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * scale;
        }
    }
}

// row id of entry i: -1 where it lies outside the table (such rows are not written, and read as zeros)
__device__ __forceinline__ int64_t table_row(const void *ids, int id_bytes, uint64_t i, uint64_t rows) {
    if (!ids) return i < rows ? (int64_t)i : -1;
    const int64_t r = id_bytes == 8 ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i];
    return r >= 0 && (uint64_t)r < rows ? r : -1;
}

// elements c .. c + 7 of a row of d as float32, zeros behind its end
template <typename T>
__device__ __forceinline__ void load8(const T *row, int c, int d, int mode, float *v) {
    if constexpr (sizeof(T) == 4) {
        const u32x4 a = load_chunk(row, c, d, mode), b = load_chunk(row, c + 4, d, mode);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float(a[i]);
            v[4 + i] = __uint_as_float(b[i]);
        }
    } else {
        const u32x4 a = load_chunk(row, c, d, mode);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = __uint_as_float(i & 1 ? a[i / 2] & 0xFFFF0000u : a[i / 2] << 16);
    }
}

// ---- writing.  The same row twice in one call: the last entry wins, whatever the order the
// workgroups run in.  A few entries: every entry looks at the ones behind it.  More: three launches
// over a scratch word per table row (cleared, the highest entry, the write).
constexpr uint32_t kFewEntries = 1024;

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

// `lanes` lanes per row (a power of two up to 64), eight columns per lane and step.
template <typename T, uint32_t CODE>
__global__ __launch_bounds__(256) void table_write_kernel(TableView t, const T *__restrict__ values,
                                                          int64_t ldv, int mode, const void *ids,
                                                          int id_bytes, uint64_t n, const int *owner,
                                                          int lanes_shift) {
    const int lane = threadIdx.x & ((1 << lanes_shift) - 1);
    const uint64_t entries = ((uint64_t)gridDim.x * 256) >> lanes_shift;
    const uint64_t mine = ((uint64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_shift;
    // every lane of a wave runs the same number of steps: the reductions cross lanes
    const uint64_t steps = (n + entries - 1) / entries;
    for (uint64_t s = 0; s < steps; ++s) {
        const uint64_t i = mine + s * entries;
        int64_t r = i < n ? table_row(ids, id_bytes, i, t.rows) : -1;
        if (ids && r >= 0) {
            if (owner) {
                if (owner[r] != (int)i) r = -1;
            } else {
                int later = 0;
                for (uint64_t j = i + 1 + lane; j < n; j += 1u << lanes_shift)
                    later |= table_row(ids, id_bytes, j, t.rows) == r;
                // lanes of one row agree: any later entry takes the row
                for (int step = 1; step < 1 << lanes_shift; step <<= 1) later |= __shfl_xor(later, step);
                if (later) r = -1;
            }
        }
        for (uint32_t c0 = 0; c0 < t.stride; c0 += 8u << lanes_shift) {
            const uint32_t c = c0 + 8 * lane;
            float x[8] = {};
            if (r >= 0 && c < t.d) load8(values + (int64_t)i * ldv, (int)c, (int)t.d, mode, x);
            uint32_t top = 0;  // as bits: NaN lies above infinity above the numbers
#pragma unroll
            for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7FFFFFFFu);
            // a group is 2 to 16 consecutive lanes of a row; rows narrower than it have fewer lanes
            for (int step = 1; step < 1 << lanes_shift && 8u * step < 1u << t.group_shift; step <<= 1)
                top = max(top, (uint32_t)__shfl_xor((int)top, step));
            if (r < 0 || c >= t.stride) continue;
            const bool finite = top < 0x7F800000u;
            constexpr float largest = CODE == kInt8 ? 127.f : 448.f;
            const float scale = finite ? fmaxf(__uint_as_float(top) / largest, 0x1p-90f) : __builtin_nanf("");
            uint2 code = {0, 0};
            if (finite) code = encode8<CODE>(x, scale);
            *reinterpret_cast<uint2 *>(t.codes + (uint64_t)r * t.stride + c) = code;
            if (c < t.d && (c & ((1u << t.group_shift) - 1)) == 0)
                t.scales[(uint64_t)r * t.groups + (c >> t.group_shift)] = scale;
        }
    }
}

template <uint32_t CODE>
__device__ __forceinline__ void table_chunk(const TableView &t, int64_t r, uint32_t c, float *v) {
    if (r >= 0 && c < t.d) {
        const uint2 code = *reinterpret_cast<const uint2 *>(t.codes + (uint64_t)r * t.stride + c);
        decode8<CODE>(code, t.scales[(uint64_t)r * t.groups + (c >> t.group_shift)], v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
}

template <typename T, uint32_t CODE>
__global__ __launch_bounds__(256) void table_read_kernel(TableView t, const void *ids, int id_bytes,
                                                         uint64_t n, T *__restrict__ out, int64_t ldo,
                                                         int align, int lanes_shift) {
    const int lane = threadIdx.x & ((1 << lanes_shift) - 1);
    const uint64_t entries = ((uint64_t)gridDim.x * 256) >> lanes_shift;
    for (uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_shift; i < n; i += entries) {
        const int64_t r = table_row(ids, id_bytes, i, t.rows);
        for (uint32_t c = 8 * lane; c < t.d; c += 8u << lanes_shift) {
            float v[8];
            table_chunk<CODE>(t, r, c, v);
            store8(out + (int64_t)i * ldo + c, v, (int)(t.d - c), align);
        }
    }
}

// One edge per `lanes` lanes: both rows in 8 bits, the operator in float32.
template <uint32_t METHOD, uint32_t CODE>
__global__ __launch_bounds__(256) void table_edges_kernel(TableView src, TableView dst,
                                                          const void *src_ids, const void *dst_ids,
                                                          int id_bytes, uint64_t n,
                                                          float *__restrict__ out, int64_t ldo, int align,
                                                          int lanes_shift) {
    constexpr bool kReduce = METHOD == kL2Distance || METHOD == kCosineSimilarity;
    const int lane = threadIdx.x & ((1 << lanes_shift) - 1);
    const uint64_t edges = ((uint64_t)gridDim.x * 256) >> lanes_shift;
    const uint64_t mine = ((uint64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_shift;
    const uint64_t steps = (n + edges - 1) / edges;  // the reductions cross lanes: all take every step
    for (uint64_t s = 0; s < steps; ++s) {
        const uint64_t e = mine + s * edges;
        const bool live = e < n;
        const int64_t u = live ? table_row(src_ids, id_bytes, e, src.rows) : -1;
        const int64_t w = live ? table_row(dst_ids, id_bytes, e, dst.rows) : -1;
        float *o = out + (int64_t)e * ldo;
        float ab = 0.f, aa = 0.f, bb = 0.f;
        for (uint32_t c = 8 * lane; c < src.d; c += 8u << lanes_shift) {
            float a[8], b[8], v[8];
            table_chunk<CODE>(src, u, c, a);
            table_chunk<CODE>(dst, w, c, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (METHOD == kL2Distance) {
                    const float x = a[i] - b[i];
                    ab = fmaf(x, x, ab);
                } else if constexpr (METHOD == kCosineSimilarity) {
                    ab = fmaf(a[i], b[i], ab);
                    aa = fmaf(a[i], a[i], aa);
                    bb = fmaf(b[i], b[i], bb);
                } else if constexpr (METHOD == kHadamard) {
                    v[i] = a[i] * b[i];
                } else if constexpr (METHOD == kSum) {
                    v[i] = a[i] + b[i];
                } else if constexpr (METHOD == kAverage) {
                    v[i] = (a[i] + b[i]) / 2.f;
                } else if constexpr (METHOD == kL1) {
                    v[i] = a[i] - b[i];
                } else if constexpr (METHOD == kAbsoluteL1) {
                    v[i] = fabsf(a[i] - b[i]);
                } else if constexpr (METHOD == kSquaredL2) {
                    v[i] = (a[i] - b[i]) * (a[i] - b[i]);
                } else if constexpr (METHOD == kL2) {
                    v[i] = sqrtf((a[i] - b[i]) * (a[i] - b[i]));
                } else if constexpr (METHOD == kMin) {
                    v[i] = fminf(a[i], b[i]);
                } else if constexpr (METHOD == kMax) {
                    v[i] = fmaxf(a[i], b[i]);
                } else {
                    v[i] = a[i];  // Concatenate: the source's half
                }
            }
            if constexpr (!kReduce) {
                if (live) {
                    store8(o + c, v, (int)(src.d - c), align);
                    if constexpr (METHOD == kConcatenate) store8(o + src.d + c, b, (int)(src.d - c), align);
                }
            }
        }
        if constexpr (kReduce) {
            for (int step = 1; step < 1 << lanes_shift; step <<= 1) {
                ab += __shfl_xor(ab, step);
                if constexpr (METHOD == kCosineSimilarity) {
                    aa += __shfl_xor(aa, step);
                    bb += __shfl_xor(bb, step);
                }
            }
            if (live && lane == 0) {
                if constexpr (METHOD == kL2Distance) {
                    o[0] = sqrtf(ab);
                } else {
                    const float norm = sqrtf(aa) * sqrtf(bb);
                    o[0] = ab / (norm < 1e-6f ? 1e-6f : norm);  // NaN norms stay NaN
                }
            }
        }
    }
}

}  // namespace gn2v
