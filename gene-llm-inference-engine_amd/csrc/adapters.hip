// Low-rank adapters of many requests beside a product that all rows share.
//
// Row t of a batch belongs to a request whose adapter is e = ids[t], and gets out[t] = base[t] + scale_e * B_e (A_e x_t): A_e is [rank, width], B_e is
// [columns, rank].  Where the product is several projections packed into one (queries, keys and values), A_e holds a block of `rank` rows for
// each and the columns of projection s read block s.  A number outside 0 .. adapters-1 is no adapter: out[t] = base[t].
//
// Both ways are matrix products of few ranks (8 to 64 as a rule), far below the matrix cores' rate: what bounds them is the traffic, x once on the way
// down, base and out once on the way up, and, for a few rows with an adapter each, the adapters themselves.  Two launches.  Down: a
// workgroup takes a tile of rows, up to 64 ranks and a segment of the width, which its four waves share out, so that none loads what another does;
// the segments' sums go to scratch.  Up: a workgroup adds the segments' sums of its tile of rows, keeps them in LDS and walks a strip of columns.
//
// Rows of one tile may take different adapters.  In a product D = M N with the rows as N's columns a lane of the matrix core's result holds values of one row only, so a
// tile is multiplied by an adapter as it is and the lanes of other rows drop what comes out: no operand is masked, and what one request's rows or matrices hold,
// numbers or not, cannot reach another's.  The tile's different adapters are counted off: workgroup z of `slots` takes every slots-th of them.
#include "common.h"

namespace {

constexpr int MAX_SLICES = 4;
constexpr int MAX_RANK = 256;
constexpr int WAVES = 4;
constexpr int SEGMENT = 512;                // of the width: what a workgroup of the way down takes at least, and always in 32 bits, where the order of a sum must not depend on the batch

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

struct Slices {                             // of the columns: slice s begins at begin[s] and reads block s of the ranks; its strips begin at strip[s]
    int n;
    int begin[MAX_SLICES + 1];
    int strip[MAX_SLICES + 1];
};

// What a lane of a wave holds of 16 rows of an operand, and the product of two such pieces onto 16 x 16 sums.  Lane l has row l % 16; of a block of
// BLOCK numbers along the sum it has two runs of RUN, at RUN * (l / 16) and half a block further.
template <bool LOW> struct Piece;
template <> struct Piece<true> {            // bfloat16: 128 bytes of a row a block, two instructions
    static constexpr int BLOCK = 64, RUN = 8;
    uint4 v[2];
};
template <> struct Piece<false> {           // 32 bits: 128 bytes a block, eight instructions
    static constexpr int BLOCK = 32, RUN = 4;
    float4 v[2];
};

__device__ __forceinline__ floatx4 times(const Piece<true>& m, const Piece<true>& n, floatx4 sum) {
#pragma unroll
    for (int h = 0; h < 2; ++h) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, m.v[h]), __builtin_bit_cast(bf16x8, n.v[h]), sum, 0, 0, 0);
    return sum;
}
__device__ __forceinline__ floatx4 times(const Piece<false>& m, const Piece<false>& n, floatx4 sum) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum = __builtin_amdgcn_mfma_f32_16x16x4f32(m.v[h].x, n.v[h].x, sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_f32_16x16x4f32(m.v[h].y, n.v[h].y, sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_f32_16x16x4f32(m.v[h].z, n.v[h].z, sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_f32_16x16x4f32(m.v[h].w, n.v[h].w, sum, 0, 0, 0);
    }
    return sum;
}

// Numbers k .. k + RUN of a row, 0 from `end` on.  ALIGNED: `end` is a multiple of RUN and the row begins at a whole run of loads.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load_run(const bf16_t* __restrict__ row, int k, int end) {
    if (ALIGNED) return k < end ? *reinterpret_cast<const uint4*>(row + k) : uint4{0u, 0u, 0u, 0u};
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < end ? row[k + i] : 0u;
    return uint4{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
}
template <bool ALIGNED>
__device__ __forceinline__ float4 load_run_f32(const float* __restrict__ row, int k, int end) {
    if (ALIGNED) return k < end ? *reinterpret_cast<const float4*>(row + k) : float4{0.f, 0.f, 0.f, 0.f};
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < end ? row[k + i] : 0.f;
    return float4{v[0], v[1], v[2], v[3]};
}
template <bool ALIGNED>
__device__ __forceinline__ float4 load_run_f32(const bf16_t* __restrict__ row, int k, int end) {
    if (ALIGNED) {
        if (k >= end) return float4{0.f, 0.f, 0.f, 0.f};
        const uint2 v = *reinterpret_cast<const uint2*>(row + k);
        return float4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
    }
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < end ? bf16_to_f32(row[k + i]) : 0.f;
    return float4{v[0], v[1], v[2], v[3]};
}
template <bool ALIGNED, typename T>
__device__ __forceinline__ void load_piece(Piece<true>& p, const T* __restrict__ row, int k, int end, int group) {
#pragma unroll
    for (int h = 0; h < 2; ++h) p.v[h] = load_run<ALIGNED>((const bf16_t*)row, k + 32 * h + 8 * group, end);
}
template <bool ALIGNED, typename T>
__device__ __forceinline__ void load_piece(Piece<false>& p, const T* __restrict__ row, int k, int end, int group) {
#pragma unroll
    for (int h = 0; h < 2; ++h) p.v[h] = load_run_f32<ALIGNED>(row, k + 16 * h + 4 * group, end);
}

// The different adapters of a tile of at most 64 rows, one after the other: `next` gives the next one and the rows that take it, as bits.  Every
// wave of a workgroup counts them off for itself.
struct Tile {
    int id;                                 // this lane's row's adapter, -1 for none
    unsigned long long left;                // rows whose adapter has not come yet

    __device__ Tile(const int* __restrict__ ids, int first, int rows, int n_rows, int n_adapters) {
        const int lane = threadIdx.x & 63;
        id = -1;
        if (lane < rows && first + lane < n_rows) id = ids[first + lane];
        if (id >= n_adapters) id = -1;
        left = __ballot(id >= 0);
    }
    __device__ int next(unsigned long long& rows) {
        const int e = __shfl(id, __ffsll((long long)left) - 1, 64);
        rows = __ballot(id == e);
        left &= ~rows;
        return e;
    }
};

// Down: sums[segment][row][rank] over a segment of the width.  NT tiles of 16 rows, MT tiles of 16 ranks.  blockIdx: (tile of rows, segment, group of ranks * slots + slot).
template <bool LOW, typename X, typename W, int NT, int MT, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES) void adapters_down_kernel(const X* __restrict__ x, long ldx, const W* __restrict__ a, const int* __restrict__ ids, float* __restrict__ sums,
                                                                   int n_rows, int width, int ranks, int n_adapters, int segment, int slots) {
    typedef Piece<LOW> P;
    __shared__ floatx4 meet[2][NT * MT * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & 15, group = lane >> 4;
    const int first_row = blockIdx.x * 16 * NT, slot = blockIdx.z % slots, first_rank = blockIdx.z / slots * 16 * MT;
    const int begin = blockIdx.y * segment, end = min(width, begin + segment);
    Tile tile(ids, first_row, 16 * NT, n_rows, n_adapters);
    const X* xr[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) xr[j] = x + (size_t)min(first_row + 16 * j + at, n_rows - 1) * ldx;
    for (int count = 0; tile.left != 0; ++count) {
        unsigned long long rows;
        const int e = tile.next(rows);
        if (count % slots != slot) continue;
        const W* ar[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) ar[i] = a + ((size_t)e * ranks + min(first_rank + 16 * i + at, ranks - 1)) * width;
        floatx4 sum[NT][MT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) sum[j][i] = floatx4{0.f, 0.f, 0.f, 0.f};
        constexpr int STEP = P::BLOCK * WAVES;
        P xp[NT], ap[MT];
        int k = begin + wave * P::BLOCK;
#pragma unroll
        for (int j = 0; j < NT; ++j) load_piece<ALIGNED>(xp[j], xr[j], k, end, group);
#pragma unroll
        for (int i = 0; i < MT; ++i) load_piece<ALIGNED>(ap[i], ar[i], k, end, group);
        for (; k < end; k += STEP) {                      // the next block is on its way while this one is multiplied
            P xn[NT], an[MT];
#pragma unroll
            for (int j = 0; j < NT; ++j) load_piece<ALIGNED>(xn[j], xr[j], k + STEP, end, group);
#pragma unroll
            for (int i = 0; i < MT; ++i) load_piece<ALIGNED>(an[i], ar[i], k + STEP, end, group);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) sum[j][i] = times(ap[i], xp[j], sum[j][i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) xp[j] = xn[j];
#pragma unroll
            for (int i = 0; i < MT; ++i) ap[i] = an[i];
        }
        // (wave 0 + wave 2) + (wave 1 + wave 3)
        if (wave >= 2) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) meet[wave - 2][(j * MT + i) * 64 + lane] = sum[j][i];
        }
        __syncthreads();
        if (wave < 2) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) sum[j][i] += meet[wave][(j * MT + i) * 64 + lane];
        }
        __syncthreads();
        if (wave == 1) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) meet[0][(j * MT + i) * 64 + lane] = sum[j][i];
        }
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (!(rows >> (16 * j + at) & 1)) continue;
                float* to = sums + ((size_t)blockIdx.y * n_rows + first_row + 16 * j + at) * ranks;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const floatx4 s = sum[j][i] + meet[0][(j * MT + i) * 64 + lane];
                    const int rank = first_rank + 16 * i + 4 * group;
                    if ((ranks & 3) == 0) {
                        if (rank < ranks) *reinterpret_cast<floatx4*>(to + rank) = s;
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (rank + c < ranks) to[rank + c] = s[c];
                    }
                }
            }
        }
        __syncthreads();                                   // (the next adapter's sums meet in the same place)
    }
}

// 4 numbers of base or out at once.
__device__ __forceinline__ floatx4 load4(const float* p) { return *reinterpret_cast<const floatx4*>(p); }
__device__ __forceinline__ floatx4 load4(const bf16_t* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return floatx4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
}
__device__ __forceinline__ void store4(float* p, floatx4 v) { *reinterpret_cast<floatx4*>(p) = v; }
__device__ __forceinline__ void store4(bf16_t* p, floatx4 v) { *reinterpret_cast<uint2*>(p) = uint2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])}; }

// Up: NT tiles of 16 rows, a strip of columns, 32 at a time and wave: of each such step the lane of row r and group g has columns 8 g .. 8 g + 7, so that a row's four lanes
// write whole lines.  The sums of A x are bfloat16 in two pieces where B is multiplied as bfloat16 (a half step of 2^-8 is left of a half step of 2^-8: one piece alone would lose more than
// the 32-bit result keeps), 32-bit otherwise.  blockIdx: (strip, tile of rows, slot).
template <bool LOW, typename W, typename S, typename O, int NT, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES) void adapters_up_kernel(const float* __restrict__ sums, const W* __restrict__ b, const float* __restrict__ scales, const int* __restrict__ ids,
                                                                 const S* base, long ldb, O* out, long ldo, int n_rows, int rank, int n_segments, Slices slices,
                                                                 int strip_columns, int n_adapters, int slots, int vectors) {
    typedef Piece<LOW> P;
    extern __shared__ __align__(16) unsigned char room[];
    const int padded = (rank + P::BLOCK / 2 - 1) / (P::BLOCK / 2) * (P::BLOCK / 2), pitch = padded + P::RUN;      // (rows of LDS a run further apart than a multiple of all banks)
    bf16_t* high = (bf16_t*)room;                          // [16 NT][pitch], and the second pieces behind
    bf16_t* low = high + 16 * NT * pitch;
    float* whole = (float*)room;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & 15, group = lane >> 4;
    const int first_row = blockIdx.y * 16 * NT, slot = blockIdx.z;
    int s = 0;
    while (s + 1 < slices.n && (int)blockIdx.x >= slices.strip[s + 1]) ++s;
    const int begin = slices.begin[s] + ((int)blockIdx.x - slices.strip[s]) * strip_columns, end = min(slices.begin[s + 1], begin + strip_columns);
    const int columns = slices.begin[slices.n], ranks = rank * slices.n;
    Tile tile(ids, first_row, 16 * NT, n_rows, n_adapters);

    // Base with the adapter's share, or without (`e` < 0), for the rows in `rows`.
    if (slot == 0) {                                       // rows without an adapter
        unsigned long long none = ~tile.left;
        const int there = min(16 * NT, n_rows - first_row);
        none &= there < 64 ? (1ull << there) - 1 : ~0ull;
        if ((const void*)base != (const void*)out) {
            while (none != 0) {
                const int row = first_row + __ffsll((long long)none) - 1;
                none &= none - 1;
                for (int c = begin + threadIdx.x; c < end; c += 64 * WAVES) store_f32(out, (size_t)row * ldo + c, load_f32(base, (size_t)row * ldb + c));
            }
        }
    }
    for (int count = 0; tile.left != 0; ++count) {
        unsigned long long rows;
        const int e = tile.next(rows);
        if (count % slots != slot) continue;
        const float scale = scales != nullptr ? scales[e] : 1.f;
        __syncthreads();                                   // (the adapter before has been read)
        for (int item = threadIdx.x; item < 16 * NT * padded; item += 64 * WAVES) {
            const int r = item / padded, k = item % padded;
            float v = 0.f;
            if (k < rank && (rows >> r & 1)) {
                const float* from = sums + (size_t)(first_row + r) * ranks + s * rank + k;
                for (int seg = 0; seg < n_segments; ++seg) v += from[(size_t)seg * n_rows * ranks];
                v *= scale;
            }
            if (LOW) {
                const bf16_t h = f32_to_bf16(v);
                high[r * pitch + k] = h;
                low[r * pitch + k] = f32_to_bf16(v - bf16_to_f32(h));
            } else {
                whole[r * pitch + k] = v;
            }
        }
        __syncthreads();
        const W* be = b + (size_t)e * columns * rank;
        for (int c0 = begin + 32 * wave; c0 < end; c0 += 32 * WAVES) {
            floatx4 sum[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) sum[j][h] = floatx4{0.f, 0.f, 0.f, 0.f};
            const W* br[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) br[h] = be + (size_t)min(c0 + 8 * (at >> 2) + 4 * h + (at & 3), end - 1) * rank;
            const int c = c0 + 8 * group;
            for (int k = 0; k < padded; k += P::BLOCK / 2) {
                const int mine = k + P::RUN * group;
                if constexpr (LOW) {
                    uint4 m[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) m[h] = load_run<ALIGNED>((const bf16_t*)br[h], mine, rank);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const bf16x8 th = *reinterpret_cast<const bf16x8*>(high + (16 * j + at) * pitch + mine), tl = *reinterpret_cast<const bf16x8*>(low + (16 * j + at) * pitch + mine);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            sum[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, m[h]), tl, sum[j][h], 0, 0, 0);
                            sum[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, m[h]), th, sum[j][h], 0, 0, 0);
                        }
                    }
                } else {
                    float4 m[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) m[h] = load_run_f32<ALIGNED>(br[h], mine, rank);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const float4 t = *reinterpret_cast<const float4*>(whole + (16 * j + at) * pitch + mine);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            sum[j][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[h].x, t.x, sum[j][h], 0, 0, 0);
                            sum[j][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[h].y, t.y, sum[j][h], 0, 0, 0);
                            sum[j][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[h].z, t.z, sum[j][h], 0, 0, 0);
                            sum[j][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[h].w, t.w, sum[j][h], 0, 0, 0);
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (!(rows >> (16 * j + at) & 1)) continue;
                const size_t row = first_row + 16 * j + at;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = c + 4 * h;
                    if (vectors && col + 4 <= end) {
                        store4(out + row * ldo + col, load4(base + row * ldb + col) + sum[j][h]);
                    } else {
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (col + u < end) store_f32(out, row * ldo + col + u, load_f32(base, row * ldb + col + u) + sum[j][h][u]);
                    }
                }
            }
        }
    }
}

bool aligned(const void* p, int bytes) { return (size_t)p % bytes == 0; }

struct Call {
    const void* x; long ldx; const void* a; const void* b; const int* ids; const float* scales; const void* base; long ldb; void* out; long ldo; float* sums;
    int n_rows, width, columns, rank, n_adapters, n_segments, segment;
    Slices slices;
    hipStream_t stream;
};

template <bool LOW, typename X, typename W, int NT, int MT>
void down_sized(const Call& c, int slots) {
    const int ranks = c.rank * c.slices.n, run = Piece<LOW>::RUN;
    const dim3 grid((c.n_rows + 16 * NT - 1) / (16 * NT), c.n_segments, (ranks + 16 * MT - 1) / (16 * MT) * slots);
    const bool even = c.width % run == 0 && c.ldx % run == 0 && aligned(c.x, run * sizeof(X)) && aligned(c.a, run * sizeof(W));
    if (even) adapters_down_kernel<LOW, X, W, NT, MT, true><<<grid, 64 * WAVES, 0, c.stream>>>((const X*)c.x, c.ldx, (const W*)c.a, c.ids, c.sums, c.n_rows, c.width, ranks, c.n_adapters, c.segment, slots);
    else adapters_down_kernel<LOW, X, W, NT, MT, false><<<grid, 64 * WAVES, 0, c.stream>>>((const X*)c.x, c.ldx, (const W*)c.a, c.ids, c.sums, c.n_rows, c.width, ranks, c.n_adapters, c.segment, slots);
}

// Bytes of LDS that the way up keeps `rows` rows' sums in.
template <bool LOW> int up_lds(int rows, int rank) {
    typedef Piece<LOW> P;
    return rows * ((rank + P::BLOCK / 2 - 1) / (P::BLOCK / 2) * (P::BLOCK / 2) + P::RUN) * 4;
}
int tiles_of_rows(const Call& c) { return c.n_rows <= 128 || up_lds<true>(64, c.rank) > 65536 ? 1 : 4; }
int slots_of(const Call& c, int tile_rows) {
    const int most = min(min(tile_rows, c.n_rows), c.n_adapters);
    return tile_rows == 16 ? most : min(most, 4);
}

template <bool LOW, typename X, typename W>
void down(const Call& c) {
    const int ranks = c.rank * c.slices.n, groups = (ranks + 63) / 64, mt = ((ranks + groups - 1) / groups + 15) / 16;
    const int nt = tiles_of_rows(c), slots = slots_of(c, 16 * nt);
#define GI_DOWN(NT) (mt == 1 ? down_sized<LOW, X, W, NT, 1>(c, slots) : mt == 2 ? down_sized<LOW, X, W, NT, 2>(c, slots) : mt == 3 ? down_sized<LOW, X, W, NT, 3>(c, slots) : down_sized<LOW, X, W, NT, 4>(c, slots))
    if (nt == 1) GI_DOWN(1);
    else GI_DOWN(4);
#undef GI_DOWN
}

template <bool LOW, typename W, typename S, typename O, int NT>
void up_sized(const Call& c) {
    typedef Piece<LOW> P;
    const int slots = slots_of(c, 16 * NT), tiles = (c.n_rows + 16 * NT - 1) / (16 * NT), lds = up_lds<LOW>(16 * NT, c.rank);
    // A strip's workgroup first makes its rows' sums, so strips are as long as leaves every compute unit a few workgroups.
    int strip = 128;
    while (strip < 1024 && (long)tiles * ((c.columns + strip - 1) / strip) > 2048) strip *= 2;
    Slices slices = c.slices;
    for (int s = 0; s < slices.n; ++s) slices.strip[s + 1] = slices.strip[s] + (slices.begin[s + 1] - slices.begin[s] + strip - 1) / strip;
    bool vectors = c.ldb % 4 == 0 && c.ldo % 4 == 0 && aligned(c.base, 4 * sizeof(S)) && aligned(c.out, 4 * sizeof(O));
    for (int s = 0; s < slices.n; ++s) vectors = vectors && slices.begin[s] % 4 == 0;
    const bool even = c.rank % P::RUN == 0 && aligned(c.b, P::RUN * sizeof(W));
    const dim3 grid(slices.strip[slices.n], tiles, slots);
    if (even) adapters_up_kernel<LOW, W, S, O, NT, true><<<grid, 64 * WAVES, lds, c.stream>>>(c.sums, (const W*)c.b, c.scales, c.ids, (const S*)c.base, c.ldb, (O*)c.out, c.ldo, c.n_rows, c.rank,
                                                                                              c.n_segments, slices, strip, c.n_adapters, slots, vectors);
    else adapters_up_kernel<LOW, W, S, O, NT, false><<<grid, 64 * WAVES, lds, c.stream>>>(c.sums, (const W*)c.b, c.scales, c.ids, (const S*)c.base, c.ldb, (O*)c.out, c.ldo, c.n_rows, c.rank,
                                                                                          c.n_segments, slices, strip, c.n_adapters, slots, vectors);
}

template <bool LOW, typename W, typename S, typename O>
void up(const Call& c) {
    if (tiles_of_rows(c) == 1) up_sized<LOW, W, S, O, 1>(c);
    else up_sized<LOW, W, S, O, 4>(c);
}

template <bool LOW, typename W>
void up_typed(const Call& c, int base_type, int out_type) {
    if (base_type == GI_BF16) out_type == GI_BF16 ? up<LOW, W, bf16_t, bf16_t>(c) : up<LOW, W, bf16_t, float>(c);
    else out_type == GI_BF16 ? up<LOW, W, float, bf16_t>(c) : up<LOW, W, float, float>(c);
}

}  // namespace

// The segments of the width on the way down.
GI_API int gi_adapters_segments(int n_rows, int width) { return (width + SEGMENT - 1) / SEGMENT; }

// sums: gi_adapters_segments(n_rows, width) * n_rows * rank * n_slices floats, 16-byte aligned.
GI_API int gi_adapters_add(const void* x, int x_type, long ldx, const void* a, const void* b, int w_type, const int* ids, const float* scales, const void* base, int base_type, long ldb,
                           void* out, int out_type, long ldo, float* sums, int n_rows, int width, int columns, int rank, int n_slices, const int* slice_columns, int n_adapters,
                           hipStream_t stream) {
    GI_REQUIRE(n_rows > 0 && width > 0 && columns > 0 && rank > 0 && n_adapters > 0 && ldx >= width && ldb >= columns && ldo >= columns,
               "adapters_add: bad sizes (rows %d, width %d, columns %d, rank %d, adapters %d, strides %ld %ld %ld)", n_rows, width, columns, rank, n_adapters, ldx, ldb, ldo);
    GI_REQUIRE(rank <= MAX_RANK, "adapters_add: rank %d, at most %d is taken", rank, MAX_RANK);
    GI_REQUIRE(n_slices >= 1 && n_slices <= MAX_SLICES, "adapters_add: %d packed projections, 1 to %d are taken", n_slices, MAX_SLICES);
    GI_REQUIRE(sums != nullptr && aligned(sums, 16), "adapters_add: scratch is missing");
    Call c{x, ldx, a, b, ids, scales, base, ldb, out, ldo, sums, n_rows, width, columns, rank, n_adapters, gi_adapters_segments(n_rows, width), SEGMENT, Slices{n_slices, {0}, {0}}, stream};
    for (int s = 0; s < n_slices; ++s) {
        GI_REQUIRE(slice_columns[s] > 0, "adapters_add: a packed projection of %d columns", slice_columns[s]);
        c.slices.begin[s + 1] = c.slices.begin[s] + slice_columns[s];
    }
    GI_REQUIRE(c.slices.begin[n_slices] == columns, "adapters_add: the packed projections have %d columns, out has %d", c.slices.begin[n_slices], columns);
    GI_REQUIRE(c.n_segments <= 65535 && (n_rows + 15) / 16 <= 65535, "adapters_add: %d rows of %d numbers are too many for one launch", n_rows, width);
    const bool low = x_type == GI_BF16 && w_type == GI_BF16;
    if (low) down<true, bf16_t, bf16_t>(c);
    else if (x_type == GI_BF16) down<false, bf16_t, float>(c);
    else if (w_type == GI_BF16) down<false, float, bf16_t>(c);
    else down<false, float, float>(c);
    GI_CHECK_LAUNCH("adapters_add (down)");
    if (low) up_typed<true, bf16_t>(c, base_type, out_type);
    else if (w_type == GI_BF16) up_typed<false, bf16_t>(c, base_type, out_type);
    else up_typed<false, float>(c, base_type, out_type);
    GI_CHECK_LAUNCH("adapters_add (up)");
    return 0;
}
