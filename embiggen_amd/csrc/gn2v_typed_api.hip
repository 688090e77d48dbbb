// libgn2v.so -- the operators on rows of embedding tables declared at the end of gn2v_internal.h:
// typed and adapted products, their gradients, tables in 8 bits.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../../include/gn2v_internal.h"
#include "handle.h"
#include "quantized_kernels.h"
#include "typed_kernels.h"

using namespace gn2v_host;

namespace {

constexpr uint64_t kMaxRows = (1ull << 31) - (1ull << 20);  // positions are int32

// A launch holds fewer than 2^32 threads along an axis.
constexpr uint64_t max_blocks(uint64_t threads) { return 0xFFFFFFFFull / threads; }

// the plan's words, and the stripes its rows are counted in
struct PlanSizes {
    uint64_t words, temp;
    uint32_t stripes, stripe;
};

PlanSizes plan_sizes(uint64_t rows, uint32_t types) {
    PlanSizes s;
    s.words = 2 * rows + 2 * (types + 2ull);
    // Stripes that are not much shorter than the list of counts that each of them has: of 1 M rows of 4 095
    // types 71 us instead of 116 with stripes of 1 024 rows, of 32 768 types 288 instead of 1 990 (where
    // one wave places a stripe's rows, and half as many types per row cost 479).
    const uint64_t groups = types + 1ull, least = groups <= 4096 ? groups / 2 : groups / 8;
    const uint64_t stripe = std::max({(uint64_t)1024, least, (rows + gn2v::kStripes - 1) / gn2v::kStripes});
    s.stripe = (uint32_t)((stripe + 255) / 256 * 256);
    s.stripes = (uint32_t)((rows + s.stripe - 1) / s.stripe);
    s.temp = rows <= gn2v::kSmallPlan ? 0 : (s.stripes + 1ull) * (types + 1ull);
    return s;
}

// tiles of at most 64 rows of one type, unknown rows among the types
uint64_t tile_bound(uint64_t rows, uint64_t groups) {
    return std::min<uint64_t>(rows, (rows + gn2v::kTileRows - 1) / gn2v::kTileRows + std::min(groups, rows));
}

gn2v::PlanView plan_view(const int32_t *d_plan, uint64_t rows, uint32_t types) {
    gn2v::PlanView v{};
    v.rows = (uint32_t)rows;
    v.types = types;
    if (!d_plan) return v;
    int *p = const_cast<int32_t *>(d_plan);
    v.order = p;
    v.row_types = p + rows;
    v.offsets = p + 2 * rows;
    v.tile_first = v.offsets + types + 2;
    return v;
}

int check_plan(uint64_t rows, uint32_t types) {
    if (rows > kMaxRows) return fail("too many rows: at most 2^31 - 2^20");
    if (types < 1 || types > GN2V_MAX_TYPES) return fail("need 1 <= n_types <= 32768");
    return 0;
}

uint32_t size_of(uint32_t dtype) { return dtype == GN2V_F32 ? 4 : 2; }

// the largest power of two up to 16 bytes that divides a row's address, whichever row
int alignment(const void *base, int64_t stride_elements, uint32_t size) {
    const uint64_t bits = (uint64_t)(uintptr_t)base | (uint64_t)(stride_elements * (int64_t)size) | 16u;
    return (int)(bits & (~bits + 1));
}

// how the chunks of rows of `length` elements are loaded (ChunkMode)
int mode_of(const void *base, int64_t stride, uint32_t length, uint32_t size, int64_t type_stride = 0) {
    const int align = std::min(alignment(base, stride, size), alignment(nullptr, type_stride, size));
    if (align == 16 && length % (16 / size) == 0) return gn2v::kWhole;
    return size == 4 || (align >= 4 && length % 2 == 0) ? gn2v::kWords : gn2v::kElements;
}

template <typename I>
void launch_plan(const I *types, const gn2v::PlanView &v, int32_t *temp, hipStream_t s) {
    if (v.rows <= gn2v::kSmallPlan) {
        hipLaunchKernelGGL((gn2v::plan_small_kernel<I>), dim3(1), dim3(gn2v::kSmallPlan), 0, s, types, v);
        return;
    }
    const PlanSizes z = plan_sizes(v.rows, v.types);
    const uint32_t groups = v.types + 1;
    // four placing waves a workgroup while their counters fit 64 KB, one with up to 128 KB of them else;
    // more waves sum over many types (of 32 768 types, 3 000 rows: 155 us; 420 with 64 threads)
    const unsigned parts = groups <= 4096 ? 4 : 1, threads = groups <= 256 ? 256 : 1024;
    const size_t lds = groups * sizeof(int);
    if (lds * parts > 65536 - 128) {  // more than the default limit, beside the kernel's own 128 bytes
        (void)hipFuncSetAttribute((const void *)gn2v::plan_count_kernel<I>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        (void)hipFuncSetAttribute((const void *)gn2v::plan_place_kernel<I>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)(lds * parts));
    }
    int *counts = temp, *totals = temp + (uint64_t)z.stripes * groups;
    hipLaunchKernelGGL((gn2v::plan_count_kernel<I>), dim3(z.stripes), dim3(256), lds, s, types, v.rows,
                       v.types, z.stripe, counts);
    hipLaunchKernelGGL(gn2v::plan_scan_kernel, dim3((groups + 3) / 4), dim3(256), 0, s, counts, z.stripes,
                       groups, totals);
    int bits = 0;
    while (v.types >> bits) ++bits;
    hipLaunchKernelGGL((gn2v::plan_place_kernel<I>), dim3(z.stripes), dim3(threads), lds * parts, s, types,
                       v, z.stripe, z.stripes, counts, bits, totals, parts);
}

int check_product(const gn2v_product_io *io) {
    if (!io) return fail("NULL io");
    if (io->dtype != GN2V_F32 && io->dtype != GN2V_BF16) return fail("unknown dtype");
    if (check_plan(io->rows, io->n_types)) return 1;
    if (io->inputs == 0 || io->outputs == 0 || io->inputs > (1u << 20) || io->outputs > (1u << 20))
        return fail("need 1 <= inputs, outputs <= 2^20");
    if (io->rank > GN2V_MAX_RANK) return fail("rank must be at most 64");
    if (io->ldx < (int64_t)io->inputs || io->ldy < (int64_t)io->outputs)
        return fail("row strides must hold a row");
    if (io->rows && (!io->d_x || !io->weight.d_data || !io->d_y)) return fail("NULL pointer");
    if (io->weight.inner != 1 && io->weight.outer != 1)
        return fail("one of the weights' two strides must be 1");
    return 0;
}

// Weights of `inputs` x `outputs` whose inner elements (`wt`) or outer elements are contiguous.  Where
// an axis has one element its stride says nothing, and both may hold.
gn2v::WeightView view_of(const gn2v_weights &w, uint32_t inputs, uint32_t outputs, uint32_t size, bool wt) {
    gn2v::WeightView v{w.d_data, w.type_stride, w.inner, w.outer, 0};
    v.mode = mode_of(w.d_data, wt ? w.outer : w.inner, wt ? inputs : outputs, size, w.type_stride);
    return v;
}
bool is_wt(const gn2v_weights &w) { return w.outer != 1; }

gn2v::ProductArgs product_args(const gn2v_product_io *io, bool wt) {
    const uint32_t size = size_of(io->dtype);
    gn2v::ProductArgs a{};
    a.x = io->d_x;
    a.ldx = io->ldx;
    a.x_mode = mode_of(io->d_x, io->ldx, io->inputs, size);
    a.w = view_of(io->weight, io->inputs, io->outputs, size, wt);
    a.bias = io->d_bias;
    a.bias_type = io->bias_stride;
    a.y = io->d_y;
    a.ldy = io->ldy;
    a.sorted = io->low_rank_rows != 0;
    a.y_align = alignment(io->d_y, io->ldy, a.sorted ? 4 : size);
    a.scale = io->scale;
    a.plan = plan_view(io->d_plan, io->rows, io->n_types);
    a.K = (int)io->inputs;
    a.N = (int)io->outputs;
    return a;
}

uint64_t product_tiles(const gn2v::ProductArgs &a, bool any_type) {
    return any_type ? (a.plan.rows + 63) / 64 : tile_bound(a.plan.rows, a.plan.types + 1ull);
}

template <typename T, int BN, bool WT, bool ADAPT>
void launch_product_kernel(const gn2v::ProductArgs &a, hipStream_t s) {
    const unsigned blocks = (unsigned)((product_tiles(a, ADAPT) + 7) / 8 * 8 * ((a.N + BN - 1) / BN));
    hipLaunchKernelGGL((gn2v::product_kernel<T, BN, WT, ADAPT>), dim3(blocks), dim3(256), 0, s, a);
}

template <typename T, bool WT, bool ADAPT>
void launch_product_bn(const gn2v::ProductArgs &a, hipStream_t s) {
    if (a.N <= 32)
        launch_product_kernel<T, 32, WT, ADAPT>(a, s);
    else if (a.N <= 64)
        launch_product_kernel<T, 64, WT, ADAPT>(a, s);
    else
        launch_product_kernel<T, 128, WT, ADAPT>(a, s);
}

template <typename T, int SLABS, int BN, bool WT, bool ADAPT>
void launch_narrow_kernel(gn2v::ProductArgs a, hipStream_t s) {
    // as many workgroups as are resident at once: two per CU
    const unsigned columns = (unsigned)((a.N + BN - 1) / BN);
    a.ranges = (uint32_t)std::min<uint64_t>(product_tiles(a, false), std::max(512u / columns, 64u));
    hipLaunchKernelGGL((gn2v::narrow_product_kernel<T, SLABS, BN, WT, ADAPT>),
                       dim3((a.ranges + 7) / 8 * 8 * columns), dim3(gn2v::kNarrowThreads), 0, s, a);
}

template <typename T, int SLABS, bool WT, bool ADAPT>
void launch_narrow_bn(const gn2v::ProductArgs &a, hipStream_t s) {
    if (a.N <= 64)
        launch_narrow_kernel<T, SLABS, 64, WT, ADAPT>(a, s);
    else
        launch_narrow_kernel<T, SLABS, 128, WT, ADAPT>(a, s);
}

// The least number of slabs that hold a row: 200 000 float32 rows of 72 and of 96 elements take 66 and 61 us with
// six of them, 81 and 77 with eight, bfloat16 rows of 144 and of 192 elements 60 and 41 instead of 73 and 47.
template <typename T, bool WT, bool ADAPT>
void launch_narrow(const gn2v::ProductArgs &a, hipStream_t s) {
    constexpr int slab = gn2v::Tile<T>::kSlab;
    if (a.K <= 2 * slab)
        launch_narrow_bn<T, 2, WT, ADAPT>(a, s);
    else if (a.K <= 4 * slab)
        launch_narrow_bn<T, 4, WT, ADAPT>(a, s);
    else if (a.K <= 6 * slab)
        launch_narrow_bn<T, 6, WT, ADAPT>(a, s);
    else
        launch_narrow_bn<T, 8, WT, ADAPT>(a, s);
}

// rows whose inner elements fit the narrow kernel's LDS tile
bool is_narrow(uint32_t dtype, uint32_t inputs) { return inputs <= (dtype == GN2V_F32 ? 128u : 256u); }

template <bool ADAPT>
int launch_product(uint32_t dtype, const gn2v::ProductArgs &a, bool wt, bool narrow, hipStream_t s) {
    // one workgroup per tile and block of columns, as launch_product_bn chooses it; narrow rows: resident ones
    const uint64_t bn = a.N <= 32 ? 32 : a.N <= 64 ? 64 : 128;
    if (!narrow && (product_tiles(a, ADAPT) + 7) / 8 * 8 * ((a.N + bn - 1) / bn) > max_blocks(256))
        return fail("too many rows and columns for one launch: at most 2^24 tiles of 64 rows x 128 columns");
    if (narrow) {
        if (dtype == GN2V_F32)
            wt ? launch_narrow<float, true, ADAPT>(a, s) : launch_narrow<float, false, ADAPT>(a, s);
        else
            wt ? launch_narrow<__bf16, true, ADAPT>(a, s) : launch_narrow<__bf16, false, ADAPT>(a, s);
    } else if (dtype == GN2V_F32) {
        wt ? launch_product_bn<float, true, ADAPT>(a, s) : launch_product_bn<float, false, ADAPT>(a, s);
    } else {
        wt ? launch_product_bn<__bf16, true, ADAPT>(a, s) : launch_product_bn<__bf16, false, ADAPT>(a, s);
    }
    HIP_TRY(hipGetLastError());
    return 0;
}

// How a gradient's tiles are dealt out: to as many workgroups as are resident at once over the blocks
// of dw, with no more than 256 MB of partial sums.
struct GradSizes {
    uint32_t bm, bn, ranges;
    uint64_t first, second, second_at, stride, bytes;
};

uint32_t block_of(uint32_t n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }

// sums of `first` and `second` elements per range and slot
void set_sums(GradSizes &g, uint64_t first, uint64_t second, uint64_t tiles, uint64_t ranges) {
    g.first = first;
    g.second = second;
    g.second_at = (first + 3) / 4 * 4;
    g.stride = (g.second_at + second + 3) / 4 * 4;
    ranges = std::min<uint64_t>(ranges, (32ull << 20) / g.stride);
    g.ranges = (uint32_t)std::max<uint64_t>(1, std::min(ranges, tiles));
    g.bytes = tiles ? 2ull * g.ranges * g.stride * 4 : 0;
}

GradSizes grad_sizes(const gn2v_gradient_io *io) {
    GradSizes g;
    g.bm = block_of(io->inputs);
    g.bn = block_of(io->outputs);
    const uint64_t blocks = std::max<uint64_t>(1, (io->inputs + g.bm - 1) / g.bm) * ((io->outputs + g.bn - 1) / g.bn);
    const uint64_t resident = 256u * gn2v::grad_waves(g.bm / 32, g.bn / 32);
    set_sums(g, (uint64_t)io->inputs * io->outputs, io->outputs,
             tile_bound(io->rows, io->shared ? 0 : io->n_types), std::max<uint64_t>(1, resident / blocks));
    return g;
}

void set_sums(gn2v::GradArgs &a, const GradSizes &g, void *partial, void *dw, void *db) {
    a.ranges = g.ranges;
    a.stride = (int64_t)g.stride;
    a.first = (int64_t)g.first;
    a.second = (int64_t)g.second;
    a.second_at = (int64_t)g.second_at;
    a.partial = (float *)partial;
    a.dw = dw;
    a.db = db;
}

template <typename T>
void launch_join(const gn2v::GradArgs &a, uint32_t types, hipStream_t s) {
    // few types lie in many ranges each: sixteen waves share them, four where there are many types
    const uint64_t blocks = types * (uint64_t)((a.stride + 255) / 256);
    const unsigned threads = types >= 64 ? 256 : 1024;
    // 2^30 sums with sixteen waves, 2^32 with four fill a launch
    for (uint64_t first = 0; first < blocks; first += max_blocks(threads))
        hipLaunchKernelGGL((gn2v::grad_join_kernel<T>), dim3((unsigned)std::min(blocks - first, max_blocks(threads))),
                           dim3(threads), 0, s, a, first);
}

// The adapted form's gradients in one pass over the rows: small enough for one block of sums.  The
// types' sums and those of the shared weight lie behind one another in d_temp.
struct FusedSizes {
    bool fused;
    GradSizes types, all;
};

FusedSizes fused_sizes(const gn2v_adapted_gradient_io *io) {
    FusedSizes f{};
    f.fused = io->d_down && io->d_up && io->rank <= gn2v::kFusedRank && io->inputs <= 128 && io->outputs <= 128;
    if (!f.fused) return f;
    const bool want = io->d_dw || io->d_db;
    const uint64_t tiles = tile_bound(io->rows, io->n_types + (want ? 1ull : 0ull));
    f.types.bm = f.all.bm = io->inputs <= 64 ? 64 : 128;
    f.types.bn = f.all.bn = io->outputs <= 64 ? 64 : 128;
    set_sums(f.types, (uint64_t)io->inputs * io->rank, (uint64_t)io->rank * io->outputs, tiles,
             256u * gn2v::adapted_grad_groups((int)size_of(io->dtype)));
    if (want) set_sums(f.all, io->d_dw ? (uint64_t)io->inputs * io->outputs : 0, io->outputs, tiles, f.types.ranges);
    return f;
}

int check_gradient(const gn2v_gradient_io *io) {
    if (!io) return fail("NULL io");
    if (io->dtype != GN2V_F32 && io->dtype != GN2V_BF16) return fail("unknown dtype");
    if (check_plan(io->rows, io->n_types)) return 1;
    if (io->outputs == 0 || io->inputs > (1u << 20) || io->outputs > (1u << 20))
        return fail("need inputs <= 2^20, 1 <= outputs <= 2^20");
    if (io->x_low && io->y_low) return fail("at most one operand is low-rank rows");
    if ((io->x_low && io->inputs > GN2V_MAX_RANK) || (io->y_low && io->outputs > GN2V_MAX_RANK))
        return fail("low-rank rows are at most 64 wide");
    return 0;
}

int check_adapted_gradient(const gn2v_adapted_gradient_io *io) {
    if (!io) return fail("NULL io");
    if (io->dtype != GN2V_F32 && io->dtype != GN2V_BF16) return fail("unknown dtype");
    if (check_plan(io->rows, io->n_types)) return 1;
    if (io->inputs == 0 || io->outputs == 0 || io->inputs > (1u << 20) || io->outputs > (1u << 20))
        return fail("need 1 <= inputs, outputs <= 2^20");
    if (io->rank == 0 || io->rank > GN2V_MAX_RANK) return fail("need a rank of 1 to 64");
    return 0;
}

// the single gradients an adapted form's are made of where they are not fused: 0 down, 1 up, 2 shared
gn2v_gradient_io part_of(const gn2v_adapted_gradient_io *io, int which) {
    gn2v_gradient_io g{};
    g.dtype = io->dtype;
    g.n_types = io->n_types;
    g.rows = io->rows;
    g.inputs = which == 1 ? io->rank : which == 2 && !io->d_dw ? 0 : io->inputs;
    g.outputs = which == 0 ? io->rank : io->outputs;
    g.d_x = which == 1 ? (const void *)io->d_low : io->d_x;
    g.ldx = which == 1 ? (int64_t)io->rank : io->ldx;
    g.d_dy = which == 0 ? (const void *)io->d_back : io->d_dy;
    g.ldy = which == 0 ? (int64_t)io->rank : io->ldy;
    g.x_low = which == 1;
    g.y_low = which == 0;
    g.shared = which == 2;
    g.d_plan = io->d_plan;
    g.d_dw = which == 0 ? io->d_down : which == 1 ? io->d_up : io->d_dw;
    g.d_db = which == 2 ? io->d_db : nullptr;
    g.d_temp = io->d_temp;
    g.temp_bytes = io->temp_bytes;
    return g;
}

bool has_part(const gn2v_adapted_gradient_io *io, int which) {
    return which == 0 ? io->d_down != nullptr : which == 1 ? io->d_up != nullptr : io->d_dw || io->d_db;
}

template <typename T, int MI, int NI>
void launch_fused(const gn2v::AdaptedGradArgs &a, bool want, hipStream_t s) {
    if (want)
        hipLaunchKernelGGL((gn2v::adapted_grad_kernel<T, MI, NI, true>), dim3(a.types.ranges), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((gn2v::adapted_grad_kernel<T, MI, NI, false>), dim3(a.types.ranges), dim3(256), 0, s, a);
}

template <typename T>
void launch_fused_grad(const gn2v_adapted_gradient_io *io, const FusedSizes &f, const gn2v::AdaptedGradArgs &a,
                       hipStream_t s) {
    const bool want = io->d_dw || io->d_db;
    if (io->rows) {
        if (f.types.bm == 64)
            f.types.bn == 64 ? launch_fused<T, 2, 2>(a, want, s) : launch_fused<T, 2, 4>(a, want, s);
        else
            f.types.bn == 64 ? launch_fused<T, 4, 2>(a, want, s) : launch_fused<T, 4, 4>(a, want, s);
    }
    launch_join<T>(a.types, io->n_types, s);
    if (want) launch_join<T>(a.all, 1, s);
}

template <typename T, int MI, int NI>
void launch_grad_low(const gn2v_gradient_io *io, const gn2v::GradArgs &a, unsigned blocks, hipStream_t s) {
    // low-rank rows are at most 64 wide (check_gradient)
    if constexpr (MI <= 2)
        if (io->x_low) {
            hipLaunchKernelGGL((gn2v::grad_kernel<T, MI, NI, true, false>), dim3(blocks), dim3(256), 0, s, a);
            return;
        }
    if constexpr (NI <= 2)
        if (io->y_low) {
            hipLaunchKernelGGL((gn2v::grad_kernel<T, MI, NI, false, true>), dim3(blocks), dim3(256), 0, s, a);
            return;
        }
    hipLaunchKernelGGL((gn2v::grad_kernel<T, MI, NI, false, false>), dim3(blocks), dim3(256), 0, s, a);
}

template <typename T>
void launch_grad(const gn2v_gradient_io *io, const GradSizes &g, const gn2v::GradArgs &a, unsigned blocks,
                 hipStream_t s) {
#define GN2V_GRAD(BM, BN) \
    if (g.bm == BM && g.bn == BN) launch_grad_low<T, BM / 32, BN / 32>(io, a, blocks, s)
    GN2V_GRAD(32, 32);
    GN2V_GRAD(32, 64);
    GN2V_GRAD(32, 128);
    GN2V_GRAD(64, 32);
    GN2V_GRAD(64, 64);
    GN2V_GRAD(64, 128);
    GN2V_GRAD(128, 32);
    GN2V_GRAD(128, 64);
    GN2V_GRAD(128, 128);
#undef GN2V_GRAD
}

int check_table(const gn2v_table8 *t) {
    if (!t) return fail("NULL table");
    if (t->code != GN2V_INT8 && t->code != GN2V_E4M3) return fail("unknown code type");
    if (t->group != 16 && t->group != 32 && t->group != 64 && t->group != 128)
        return fail("group must be 16, 32, 64 or 128");
    if (t->d == 0 || t->d > (1u << 20) || t->stride < t->d || (t->stride & 15))
        return fail("need 0 < d <= stride, stride % 16 == 0, d <= 2^20");
    if (t->rows && (!t->d_codes || !t->d_scales)) return fail("NULL pointer");
    if ((uintptr_t)t->d_codes & 15) return fail("codes must be 16-byte aligned");
    return 0;
}

gn2v::TableView table_view(const gn2v_table8 *t) {
    gn2v::TableView v;
    v.codes = (uint8_t *)t->d_codes;
    v.scales = t->d_scales;
    v.rows = t->rows;
    v.d = t->d;
    v.stride = t->stride;
    v.group_shift = t->group == 16 ? 4 : t->group == 32 ? 5 : t->group == 64 ? 6 : 7;
    v.groups = (t->d + t->group - 1) / t->group;
    return v;
}

// lanes per row: `columns` columns each, a power of two, a wave at most
int lanes_shift(uint32_t d, uint32_t columns) {
    int shift = 0;
    while (shift < 6 && (columns << shift) < d) ++shift;
    return shift;
}

// Workgroups of 256 threads for n rows of 1 << shift lanes, `ahead` rows at a time: a step each, but for
// few rows, which are spread over the CUs (a grid-stride loop over resident workgroups left the last
// step's waves idle: 333 333 written rows 88 us instead of 62).
unsigned row_blocks(uint64_t n, int shift, uint64_t ahead) {
    const uint64_t per = 256u >> shift, all = (n + per - 1) / per;
    return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>(std::min<uint64_t>(all, 1u << 22), std::max<uint64_t>(512, (all + ahead - 1) / ahead)));
}

int check_ids(const void *ids, uint32_t id_bytes) {
    if (ids && id_bytes != 4 && id_bytes != 8) return fail("id_bytes must be 4 or 8");
    return 0;
}

template <typename T>
void launch_write(const gn2v_table8 *t, const gn2v::TableView &v, const void *values, int64_t ldv,
                  const void *ids, uint32_t id_bytes, uint64_t n, const int32_t *owner, hipStream_t s) {
    const int shift = lanes_shift(t->d, gn2v::kColumns<T>), mode = mode_of(values, ldv, t->d, sizeof(T));
    const unsigned blocks = row_blocks(n, shift, 2);
    if (t->code == GN2V_INT8)
        hipLaunchKernelGGL((gn2v::table_write_kernel<T, gn2v::kInt8>), dim3(blocks), dim3(256), 0, s, v,
                           (const T *)values, ldv, mode, ids, (int)id_bytes, n, owner, shift);
    else
        hipLaunchKernelGGL((gn2v::table_write_kernel<T, gn2v::kE4m3>), dim3(blocks), dim3(256), 0, s, v,
                           (const T *)values, ldv, mode, ids, (int)id_bytes, n, owner, shift);
}

template <typename T>
void launch_read(const gn2v_table8 *t, const gn2v::TableView &v, const void *ids, uint32_t id_bytes,
                 uint64_t n, void *out, int64_t ldo, hipStream_t s) {
    const int shift = lanes_shift(t->d, gn2v::kColumns<T>), align = alignment(out, ldo, sizeof(T));
    const unsigned blocks = row_blocks(n, shift, gn2v::kAhead);
    if (t->code == GN2V_INT8)
        hipLaunchKernelGGL((gn2v::table_read_kernel<T, gn2v::kInt8>), dim3(blocks), dim3(256), 0, s, v, ids,
                           (int)id_bytes, n, (T *)out, ldo, align, shift);
    else
        hipLaunchKernelGGL((gn2v::table_read_kernel<T, gn2v::kE4m3>), dim3(blocks), dim3(256), 0, s, v, ids,
                           (int)id_bytes, n, (T *)out, ldo, align, shift);
}

template <uint32_t METHOD, uint32_t CODE>
void launch_edges(const gn2v::TableView &a, const gn2v::TableView &b, const void *u, const void *w,
                  uint32_t id_bytes, uint64_t n, float *out, int64_t ldo, hipStream_t s) {
    if constexpr (METHOD == gn2v::kL2Distance || METHOD == gn2v::kCosineSimilarity) {
        const int shift = lanes_shift(a.d, 16);
        hipLaunchKernelGGL((gn2v::table_scores_kernel<METHOD, CODE>), dim3(row_blocks(n, shift, gn2v::kAhead)),
                           dim3(256), 0, s, a, b, u, w, (int)id_bytes, n, out, ldo, shift);
    } else {
        // Concatenate's second half starts behind the first
        const int shift = lanes_shift(a.d, 4),
                  align = std::min(alignment(out, ldo, 4), METHOD == gn2v::kConcatenate ? alignment(out, a.d, 4) : 16);
        hipLaunchKernelGGL((gn2v::table_edges_kernel<METHOD, CODE>), dim3(row_blocks(n, shift, gn2v::kAhead)),
                           dim3(256), 0, s, a, b, u, w, (int)id_bytes, n, out, ldo, align, shift);
    }
}

}  // namespace

extern "C" {

int gn2v_type_plan_words(uint64_t rows, uint32_t n_types, uint64_t *plan_words, uint64_t *temp_words) {
    if (!plan_words || !temp_words) return fail("NULL pointer");
    if (check_plan(rows, n_types)) return 1;
    const PlanSizes s = plan_sizes(rows, n_types);
    *plan_words = s.words;
    *temp_words = s.temp;
    return 0;
}

int gn2v_type_plan(const void *d_types, uint32_t type_bytes, uint64_t rows, uint32_t n_types,
                   int32_t *d_plan, int32_t *d_temp, void *stream) {
    if (check_plan(rows, n_types)) return 1;
    if (type_bytes != 4 && type_bytes != 8) return fail("type_bytes must be 4 or 8");
    if (!d_plan || (rows && !d_types) || (plan_sizes(rows, n_types).temp && !d_temp))
        return fail("NULL pointer");
    DeviceGuard guard(DeviceGuard::of_pointer(d_plan));
    const gn2v::PlanView v = plan_view(d_plan, rows, n_types);
    if (type_bytes == 8)
        launch_plan((const int64_t *)d_types, v, d_temp, (hipStream_t)stream);
    else
        launch_plan((const int32_t *)d_types, v, d_temp, (hipStream_t)stream);
    HIP_TRY(hipGetLastError());
    return 0;
}

int gn2v_typed_product(const gn2v_product_io *io, void *stream) {
    if (check_product(io)) return 1;
    if (io->rows == 0) return 0;
    if (!io->d_plan) return fail("NULL plan");
    DeviceGuard guard(DeviceGuard::of_pointer(io->d_y));
    const bool wt = is_wt(io->weight);
    return launch_product<false>(io->dtype, product_args(io, wt), wt,
                                 !io->low_rank_rows && is_narrow(io->dtype, io->inputs), (hipStream_t)stream);
}

int gn2v_adapted_product(const gn2v_product_io *io, void *stream) {
    if (check_product(io)) return 1;
    if (io->rank == 0) return fail("need a rank of at least 1");
    if (io->low_rank_rows) return fail("low_rank_rows belongs to gn2v_typed_product");
    if (io->rows == 0) return 0;
    if (!io->d_plan || !io->down.d_data || !io->up.d_data) return fail("NULL pointer");
    const bool narrow = io->rank <= gn2v::kFusedRank && is_narrow(io->dtype, io->inputs);
    if (!narrow && !io->d_low) return fail("NULL low-rank rows");
    // the kernel of wide rows takes both weights through one path
    const auto fits = [](const gn2v_weights &w, bool wt, uint32_t inputs, uint32_t outputs) {
        return wt ? w.inner == 1 || inputs == 1 : w.outer == 1 || outputs == 1;
    };
    bool wt = is_wt(io->weight);
    if (!narrow && !fits(io->up, wt, io->rank, io->outputs)) wt = !wt;
    if (!narrow && (!fits(io->up, wt, io->rank, io->outputs) || !fits(io->weight, wt, io->inputs, io->outputs)))
        return fail("weight and up must be laid out alike");
    DeviceGuard guard(DeviceGuard::of_pointer(io->d_y));
    const uint32_t size = size_of(io->dtype);
    gn2v::ProductArgs a = product_args(io, wt);
    a.bias_type = 0;
    a.rank = (int)io->rank;
    a.down = view_of(io->down, io->inputs, io->rank, size, is_wt(io->down));
    a.up = view_of(io->up, io->rank, io->outputs, size, wt);
    a.low_out = io->d_low;
    hipStream_t s = (hipStream_t)stream;
    if (!narrow) {
        // the low-rank rows first, by the typed product
        gn2v::ProductArgs low = a;
        low.w = a.down;
        low.bias = nullptr;
        low.y = io->d_low;
        low.ldy = (int64_t)io->rank;
        low.y_align = alignment(io->d_low, (int64_t)io->rank, 4);
        low.sorted = 1;
        low.N = (int)io->rank;
        if (launch_product<false>(io->dtype, low, is_wt(io->down), false, s)) return 1;
        a.low = io->d_low;
        a.scale = 1.f;  // the low-rank rows hold it
    }
    return launch_product<true>(io->dtype, a, wt, narrow, s);
}

int gn2v_few_rows_product(const gn2v_product_io *io, void *stream) {
    if (check_product(io)) return 1;
    if (io->inputs > GN2V_FEW_ROWS_DEPTH || io->rows > 65535)
        return fail("need inputs <= 4096 and rows <= 65535");
    if (io->low_rank_rows) return fail("low_rank_rows belongs to gn2v_typed_product");
    if (io->weight.outer != 1 || (io->rank && (io->down.outer != 1 || io->up.outer != 1)))
        return fail("weights must have contiguous rows");
    if (io->rows == 0) return 0;
    if (!io->d_plan && (!io->d_types || (io->type_bytes != 4 && io->type_bytes != 8)))
        return fail("need a plan, or int32 / int64 types");
    if (io->rank && (!io->down.d_data || !io->up.d_data)) return fail("NULL pointer");
    DeviceGuard guard(DeviceGuard::of_pointer(io->d_y));
    const uint32_t size = size_of(io->dtype);
    gn2v::FewArgs a{};
    a.x = io->d_x;
    a.ldx = io->ldx;
    a.w = view_of(io->weight, io->inputs, io->outputs, size, false);
    a.bias = io->d_bias;
    a.bias_type = io->bias_stride;
    a.y = io->d_y;
    a.ldy = io->ldy;
    a.types = io->d_plan ? nullptr : io->d_types;
    a.type_bytes = (int)io->type_bytes;
    a.plan = plan_view(io->d_plan, io->rows, io->n_types);
    a.K = (int)io->inputs;
    a.N = (int)io->outputs;
    a.rank = (int)io->rank;
    a.scale = io->scale;
    const dim3 grid((io->outputs + 63) / 64, (unsigned)io->rows);
    hipStream_t s = (hipStream_t)stream;
    if (io->rank) {
        a.down = view_of(io->down, io->inputs, io->rank, size, false);
        a.up = view_of(io->up, io->rank, io->outputs, size, false);
        if (io->dtype == GN2V_F32)
            hipLaunchKernelGGL((gn2v::few_rows_kernel<float, true>), grid, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL((gn2v::few_rows_kernel<__bf16, true>), grid, dim3(256), 0, s, a);
    } else if (io->dtype == GN2V_F32) {
        hipLaunchKernelGGL((gn2v::few_rows_kernel<float, false>), grid, dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL((gn2v::few_rows_kernel<__bf16, false>), grid, dim3(256), 0, s, a);
    }
    HIP_TRY(hipGetLastError());
    return 0;
}

int gn2v_typed_gradient_temp(const gn2v_gradient_io *io, uint64_t *temp_bytes) {
    if (!temp_bytes) return fail("NULL pointer");
    if (check_gradient(io)) return 1;
    *temp_bytes = grad_sizes(io).bytes;
    return 0;
}

int gn2v_typed_gradient(const gn2v_gradient_io *io, void *stream) {
    if (check_gradient(io)) return 1;
    if ((io->inputs && !io->d_dw) || (!io->inputs && !io->d_db)) return fail("NULL gradient");
    if (io->rows && (!io->d_dy || (io->inputs && !io->d_x))) return fail("NULL pointer");
    if (io->rows && !io->d_plan && (!io->shared || io->x_low || io->y_low)) return fail("NULL plan");
    if (io->ldx < (int64_t)io->inputs || io->ldy < (int64_t)io->outputs)
        return fail("row strides must hold a row");
    const GradSizes g = grad_sizes(io);
    if (io->temp_bytes < g.bytes || (g.bytes && !io->d_temp)) return fail("d_temp is too small");
    const uint64_t kb = std::max<uint64_t>(1, (io->inputs + g.bm - 1) / g.bm), nb = (io->outputs + g.bn - 1) / g.bn;
    const uint64_t blocks = (g.ranges + 7ull) / 8 * 8 * kb * nb;
    const uint32_t types = io->shared ? 1 : io->n_types;
    if (blocks > max_blocks(256)) return fail("too many inputs and outputs for one launch");
    DeviceGuard guard(DeviceGuard::of_pointer(io->d_dw ? io->d_dw : io->d_db));
    hipStream_t s = (hipStream_t)stream;
    const uint32_t size = size_of(io->dtype);
    gn2v::GradArgs a{};
    a.x = io->d_x;
    a.dy = io->d_dy;
    a.ldx = io->ldx;
    a.ldy = io->ldy;
    a.x_mode = mode_of(io->d_x, io->ldx, io->inputs, io->x_low ? 4 : size);
    a.y_mode = mode_of(io->d_dy, io->ldy, io->outputs, io->y_low ? 4 : size);
    a.plan = plan_view(io->d_plan, io->rows, io->n_types);
    a.span = io->shared ? gn2v::kRowBlocks : gn2v::kKnownTiles;
    a.shared = io->shared != 0;
    a.K = (int)io->inputs;
    a.N = (int)io->outputs;
    set_sums(a, g, io->d_temp, io->d_dw, io->d_db);
    if (io->rows) {
        if (io->dtype == GN2V_F32)
            launch_grad<float>(io, g, a, (unsigned)blocks, s);
        else
            launch_grad<__bf16>(io, g, a, (unsigned)blocks, s);
        HIP_TRY(hipGetLastError());
    }
    if (io->dtype == GN2V_F32)
        launch_join<float>(a, types, s);
    else
        launch_join<__bf16>(a, types, s);
    HIP_TRY(hipGetLastError());
    return 0;
}

int gn2v_adapted_gradient_temp(const gn2v_adapted_gradient_io *io, uint64_t *temp_bytes) {
    if (!temp_bytes) return fail("NULL pointer");
    if (check_adapted_gradient(io)) return 1;
    const FusedSizes f = fused_sizes(io);
    *temp_bytes = f.types.bytes + f.all.bytes;
    if (!f.fused)
        for (int which = 0; which < 3; ++which)
            if (has_part(io, which)) {
                const gn2v_gradient_io g = part_of(io, which);
                *temp_bytes = std::max<uint64_t>(*temp_bytes, grad_sizes(&g).bytes);
            }
    return 0;
}

int gn2v_adapted_gradient(const gn2v_adapted_gradient_io *io, void *stream) {
    if (check_adapted_gradient(io)) return 1;
    if (io->ldx < (int64_t)io->inputs || io->ldy < (int64_t)io->outputs)
        return fail("row strides must hold a row");
    if (io->rows && (!io->d_plan || !io->d_x || !io->d_dy || (io->d_down && !io->d_back) || (io->d_up && !io->d_low)))
        return fail("NULL pointer");
    uint64_t need = 0;
    if (gn2v_adapted_gradient_temp(io, &need)) return 1;
    if (io->temp_bytes < need || (need && !io->d_temp)) return fail("d_temp is too small");
    const FusedSizes f = fused_sizes(io);
    if (!f.fused) {
        for (int which = 0; which < 3; ++which)
            if (has_part(io, which)) {
                const gn2v_gradient_io g = part_of(io, which);
                if (gn2v_typed_gradient(&g, stream)) return 1;
            }
        return 0;
    }
    DeviceGuard guard(DeviceGuard::of_pointer(io->d_down));
    const uint32_t size = size_of(io->dtype);
    const bool want = io->d_dw || io->d_db;
    gn2v::AdaptedGradArgs a{};
    gn2v::GradArgs &t = a.types;
    t.x = io->d_x;
    t.dy = io->d_dy;
    t.ldx = io->ldx;
    t.ldy = io->ldy;
    t.x_mode = mode_of(io->d_x, io->ldx, io->inputs, size);
    t.y_mode = mode_of(io->d_dy, io->ldy, io->outputs, size);
    t.plan = plan_view(io->d_plan, io->rows, io->n_types);
    t.span = want ? gn2v::kAllTiles : gn2v::kKnownTiles;
    t.K = (int)io->inputs;
    t.N = (int)io->outputs;
    a.all = t;
    a.all.shared = 1;
    set_sums(t, f.types, io->d_temp, io->d_down, io->d_up);
    if (want) set_sums(a.all, f.all, (char *)io->d_temp + f.types.bytes, io->d_dw, io->d_db);
    a.low = io->d_low;
    a.back = io->d_back;
    a.rank = (int)io->rank;
    a.low_mode = std::max(mode_of(io->d_low, io->rank, io->rank, 4), mode_of(io->d_back, io->rank, io->rank, 4));
    if (io->dtype == GN2V_F32)
        launch_fused_grad<float>(io, f, a, (hipStream_t)stream);
    else
        launch_fused_grad<__bf16>(io, f, a, (hipStream_t)stream);
    HIP_TRY(hipGetLastError());
    return 0;
}

int gn2v_table_write(const gn2v_table8 *table, const void *d_values, uint32_t dtype, int64_t ldv,
                     const void *d_ids, uint32_t id_bytes, uint64_t n, int32_t *d_owner, void *stream) {
    if (check_table(table) || check_ids(d_ids, id_bytes)) return 1;
    if (dtype != GN2V_F32 && dtype != GN2V_BF16) return fail("unknown dtype");
    if (n > 0x7FFFFFFFull) return fail("at most 2^31 - 1 entries");
    if (!d_ids && n > table->rows) return fail("more rows than the table has");
    if (ldv < (int64_t)table->d) return fail("the row stride must hold a row");
    if (n == 0 || table->rows == 0) return 0;
    const bool many = d_ids && n > GN2V_TABLE_FEW_ENTRIES;
    if (!d_values || (many && !d_owner)) return fail("NULL pointer");
    DeviceGuard guard(DeviceGuard::of_pointer(table->d_codes));
    const gn2v::TableView v = table_view(table);
    hipStream_t s = (hipStream_t)stream;
    if (many) {
        const unsigned blocks = (unsigned)std::min<uint64_t>((n + 255) / 256, 256 * 16);
        for (int clear = 1; clear >= 0; --clear)
            hipLaunchKernelGGL(gn2v::table_owner_kernel, dim3(blocks), dim3(256), 0, s, d_ids, (int)id_bytes,
                               n, v.rows, (int *)d_owner, clear);
    }
    if (dtype == GN2V_F32)
        launch_write<float>(table, v, d_values, ldv, d_ids, id_bytes, n, many ? d_owner : nullptr, s);
    else
        launch_write<__bf16>(table, v, d_values, ldv, d_ids, id_bytes, n, many ? d_owner : nullptr, s);
    HIP_TRY(hipGetLastError());
    return 0;
}

int gn2v_table_read(const gn2v_table8 *table, const void *d_ids, uint32_t id_bytes, uint64_t n,
                    void *d_out, uint32_t dtype, int64_t ldo, void *stream) {
    if (check_table(table) || check_ids(d_ids, id_bytes)) return 1;
    if (dtype != GN2V_F32 && dtype != GN2V_BF16) return fail("unknown dtype");
    if (ldo < (int64_t)table->d) return fail("the row stride must hold a row");
    if (n == 0) return 0;
    if (!d_out) return fail("NULL pointer");
    DeviceGuard guard(DeviceGuard::of_pointer(d_out));
    const gn2v::TableView v = table_view(table);
    if (dtype == GN2V_F32)
        launch_read<float>(table, v, d_ids, id_bytes, n, d_out, ldo, (hipStream_t)stream);
    else
        launch_read<__bf16>(table, v, d_ids, id_bytes, n, d_out, ldo, (hipStream_t)stream);
    HIP_TRY(hipGetLastError());
    return 0;
}

int gn2v_table_edge_embedding(const gn2v_table8 *src, const gn2v_table8 *dst, const void *d_src_ids,
                              const void *d_dst_ids, uint32_t id_bytes, uint64_t n_edges,
                              uint32_t method, float *d_out, int64_t ldo, void *stream) {
    if (check_table(src) || check_table(dst)) return 1;
    if (id_bytes != 4 && id_bytes != 8) return fail("id_bytes must be 4 or 8");
    if (src->d != dst->d || src->code != dst->code) return fail("both tables need the same width and codes");
    if (method >= gn2v::kEdgeMethodCount) return fail("unknown edge embedding method");
    const int64_t need = method == gn2v::kConcatenate ? 2 * (int64_t)src->d
                         : (method == gn2v::kL2Distance || method == gn2v::kCosineSimilarity) ? 1
                                                                                             : src->d;
    if (ldo < need) return fail("out row stride is too small for this method");
    if (n_edges == 0) return 0;
    if (!d_src_ids || !d_dst_ids || !d_out) return fail("NULL pointer");
    DeviceGuard guard(DeviceGuard::of_pointer(d_out));
    const gn2v::TableView a = table_view(src), b = table_view(dst);
    hipStream_t s = (hipStream_t)stream;
    switch (method) {
#define GN2V_EDGES(M)                                                                             \
    case gn2v::M:                                                                                 \
        src->code == GN2V_INT8                                                                    \
            ? launch_edges<gn2v::M, gn2v::kInt8>(a, b, d_src_ids, d_dst_ids, id_bytes, n_edges, d_out, ldo, s) \
            : launch_edges<gn2v::M, gn2v::kE4m3>(a, b, d_src_ids, d_dst_ids, id_bytes, n_edges, d_out, ldo, s); \
        break
        GN2V_EDGES(kHadamard);
        GN2V_EDGES(kSum);
        GN2V_EDGES(kAverage);
        GN2V_EDGES(kL1);
        GN2V_EDGES(kAbsoluteL1);
        GN2V_EDGES(kSquaredL2);
        GN2V_EDGES(kL2);
        GN2V_EDGES(kConcatenate);
        GN2V_EDGES(kMin);
        GN2V_EDGES(kMax);
        GN2V_EDGES(kL2Distance);
        GN2V_EDGES(kCosineSimilarity);
#undef GN2V_EDGES
    }
    HIP_TRY(hipGetLastError());
    return 0;
}

}  // extern "C"
