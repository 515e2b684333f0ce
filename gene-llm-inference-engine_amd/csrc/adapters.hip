// Low-rank adapters of many requests beside a product that all rows share.
//
// Row t of a batch belongs to a request whose adapter is e = ids[t], and gets out[t] = base[t] + scale_e * B_e (A_e x_t): A_e is [rank, width], B_e is
// [columns, rank].  Where the product is several projections packed into one (queries, keys and values), A_e holds a block of `rank` rows for
// each and the columns of projection s read block s.  A number outside 0 .. adapters-1 is no adapter: out[t] = base[t].
//
// Two launches: t = A_e x_t in 32 bits, [rows, ranks], and the way up with the sum onto base in its epilogue.  Every sum's order depends on the
// sizes of its own row alone, so a row's result has the same bits in every batch.
#include "common.h"

namespace {

constexpr int MAX_SLICES = 4;

struct Slices {                             // of the columns: slice s begins at begin[s] and reads block s of the ranks
    int n;
    int begin[MAX_SLICES + 1];
};

// One wave for a row and a rank.
template <typename X, typename W>
__global__ __launch_bounds__(256) void adapters_down_kernel(const X* __restrict__ x, long ldx, const W* __restrict__ a, const int* __restrict__ ids, float* __restrict__ t,
                                                            int n_rows, int width, int ranks, int n_adapters) {
    const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (item >= (long)n_rows * ranks) return;
    const int row = (int)(item / ranks), rank = (int)(item % ranks);
    const int e = ids[row];
    if (e < 0 || e >= n_adapters) return;
    const X* xr = x + (size_t)row * ldx;
    const W* ar = a + ((size_t)e * ranks + rank) * width;
    float sum = 0.f;
    for (int k = lane; k < width; k += 64) sum = fmaf(load_f32(xr, k), load_f32(ar, k), sum);
    sum = wave_sum(sum);
    if (lane == 0) t[(size_t)row * ranks + rank] = sum;
}

// One thread for a row and a column.
template <typename W, typename S, typename O>
__global__ __launch_bounds__(256) void adapters_up_kernel(const float* __restrict__ t, const W* __restrict__ b, const float* __restrict__ scales, const int* __restrict__ ids,
                                                          const S* base, long ldb, O* out, long ldo, int columns, int rank, Slices slices, int n_adapters) {
    const int row = blockIdx.y, col = blockIdx.x * 256 + threadIdx.x;
    if (col >= columns) return;
    const int e = ids[row];
    float y = load_f32(base, (size_t)row * ldb + col);
    if (e >= 0 && e < n_adapters) {
        int s = 0;
        while (s + 1 < slices.n && col >= slices.begin[s + 1]) ++s;
        const float* tr = t + (size_t)row * slices.n * rank + s * rank;
        const W* br = b + ((size_t)e * columns + col) * rank;
        float sum = 0.f;
        for (int k = 0; k < rank; ++k) sum = fmaf(tr[k], load_f32(br, k), sum);
        y = fmaf(scales != nullptr ? scales[e] : 1.f, sum, y);
    }
    store_f32(out, (size_t)row * ldo + col, y);
}

template <typename W, typename S, typename O>
void up(const float* t, const void* b, const float* scales, const int* ids, const void* base, long ldb, void* out, long ldo, int n_rows, int columns, int rank,
        const Slices& slices, int n_adapters, hipStream_t stream) {
    for (int first = 0; first < n_rows; first += 65535) {
        const int rows = min(65535, n_rows - first);
        adapters_up_kernel<<<dim3((columns + 255) / 256, rows), 256, 0, stream>>>(t + (size_t)first * slices.n * rank, (const W*)b, scales, ids + first, (const S*)base + (size_t)first * ldb, ldb,
                                                                                   (O*)out + (size_t)first * ldo, ldo, columns, rank, slices, n_adapters);
    }
}

}  // namespace

// Floats of scratch that gi_adapters_add needs.
GI_API long gi_adapters_scratch_floats(int n_rows, int width, int ranks) { return (long)n_rows * ranks; }

GI_API int gi_adapters_add(const void* x, int x_type, long ldx, const void* a, const void* b, int w_type, const int* ids, const float* scales, const void* base, int base_type, long ldb,
                           void* out, int out_type, long ldo, float* t, int n_rows, int width, int columns, int rank, int n_slices, const int* slice_columns, int n_adapters,
                           hipStream_t stream) {
    GI_REQUIRE(n_rows > 0 && width > 0 && columns > 0 && rank > 0 && n_adapters > 0 && ldx >= width && ldb >= columns && ldo >= columns,
               "adapters_add: bad sizes (rows %d, width %d, columns %d, rank %d, adapters %d, strides %ld %ld %ld)", n_rows, width, columns, rank, n_adapters, ldx, ldb, ldo);
    GI_REQUIRE(n_slices >= 1 && n_slices <= MAX_SLICES, "adapters_add: %d packed projections, 1 to %d are taken", n_slices, MAX_SLICES);
    GI_REQUIRE(t != nullptr, "adapters_add: scratch is missing");
    Slices slices{n_slices, {0}};
    for (int s = 0; s < n_slices; ++s) {
        GI_REQUIRE(slice_columns[s] > 0, "adapters_add: a packed projection of %d columns", slice_columns[s]);
        slices.begin[s + 1] = slices.begin[s] + slice_columns[s];
    }
    GI_REQUIRE(slices.begin[n_slices] == columns, "adapters_add: the packed projections have %d columns, out has %d", slices.begin[n_slices], columns);
    const int ranks = rank * n_slices;
    const long items = (long)n_rows * ranks, blocks = (items + 3) / 4;
    GI_REQUIRE(blocks < (1l << 31), "adapters_add: %d rows of %d ranks are too many for one launch", n_rows, ranks);
    const dim3 grid((unsigned)blocks);
#define DOWN(X, W) adapters_down_kernel<<<grid, 256, 0, stream>>>((const X*)x, ldx, (const W*)a, ids, t, n_rows, width, ranks, n_adapters)
    if (x_type == GI_BF16 && w_type == GI_BF16) DOWN(bf16_t, bf16_t);
    else if (x_type == GI_BF16) DOWN(bf16_t, float);
    else if (w_type == GI_BF16) DOWN(float, bf16_t);
    else DOWN(float, float);
#undef DOWN
    GI_CHECK_LAUNCH("adapters_add (down)");
#define UP(W, S, O) up<W, S, O>(t, b, scales, ids, base, ldb, out, ldo, n_rows, columns, rank, slices, n_adapters, stream)
#define UP_S(W, S) (out_type == GI_BF16 ? UP(W, S, bf16_t) : UP(W, S, float))
#define UP_W(W) (base_type == GI_BF16 ? UP_S(W, bf16_t) : UP_S(W, float))
    w_type == GI_BF16 ? UP_W(bf16_t) : UP_W(float);
#undef UP_W
#undef UP_S
#undef UP
    GI_CHECK_LAUNCH("adapters_add (up)");
    return 0;
}
