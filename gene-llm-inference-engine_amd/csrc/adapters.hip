// Low-rank adapters of many requests beside a product that all rows share.
//
// Row t of a batch belongs to a request whose adapter is e = ids[t], and gets out[t] = base[t] + scale_e * B_e (A_e x_t): A_e is [rank, width], B_e is
// [columns, rank].  Where the product is several projections packed into one (queries, keys and values), A_e holds a block of `rank` rows for
// each and the columns of projection s read block s.  A number outside 0 .. adapters-1 is no adapter: out[t] = base[t].
//
// Both ways are matrix products of few ranks (8 to 64 as a rule), far below the matrix cores' rate: what bounds them is the traffic, x once on the way
// down, base and out once on the way up, and, for a few rows with an adapter each, the adapters themselves.  Two launches, which leave the sums A x of every
// row in scratch between them.  A few rows are taken one by one (the last kernels below).  More are cut into tiles: runs of neighbours with one adapter, ended at every 64th row too, as a
// request's rows lie together.  How many tiles there are only the device knows: every workgroup of the way down counts them for itself and takes every so manieth piece of work, and they leave the way up a list.
#include "common.h"
#include "lanes.h"

#include <type_traits>

namespace {

constexpr int MAX_SLICES = 4;
constexpr int MAX_RANK = 256;
constexpr int ANY_WAVES = 4, UP_WAVES = 4, UP_NT = 64 * UP_WAVES;
constexpr int SEGMENT = 256;                // of the width: the least that a workgroup of the way down takes
constexpr int EXACT_SEGMENTS = 12;          // in 32 bits, where the order of a sum must not depend on the batch, as many of the width at most, whatever the number of rows
constexpr int TILE = 64;                    // rows

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// Numbers side by side that begin wherever one of their kind may: memory takes 4 to 16 bytes at once from any place.
struct __attribute__((packed, aligned(2))) Low8 { uint32_t x, y, z, w; };
struct __attribute__((packed, aligned(2))) Low4 { uint32_t x, y; };
struct __attribute__((packed, aligned(2))) Low2 { uint32_t x; };
struct __attribute__((packed, aligned(4))) High4 { float x, y, z, w; };

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
    typedef bf16_t T;
    typedef uint4 V;
    V v[2];
};
template <> struct Piece<false> {           // 32 bits: 128 bytes a block, eight instructions
    static constexpr int BLOCK = 32, RUN = 4;
    typedef float T;
    typedef float4 V;
    V v[2];
};

__device__ __forceinline__ floatx4 times(const Piece<true>& m, const Piece<true>& n, floatx4 sum) {
#pragma unroll
    for (int h = 0; h < 2; ++h) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, m.v[h]), __builtin_bit_cast(bf16x8, n.v[h]), sum, 0, 0, 0);
    return sum;
}
__device__ __forceinline__ floatx4 times(const float4& m, const float4& n, floatx4 sum) {
    sum = __builtin_amdgcn_mfma_f32_16x16x4f32(m.x, n.x, sum, 0, 0, 0);
    sum = __builtin_amdgcn_mfma_f32_16x16x4f32(m.y, n.y, sum, 0, 0, 0);
    sum = __builtin_amdgcn_mfma_f32_16x16x4f32(m.z, n.z, sum, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(m.w, n.w, sum, 0, 0, 0);
}
__device__ __forceinline__ floatx4 times(const Piece<false>& m, const Piece<false>& n, floatx4 sum) { return times(m.v[1], n.v[1], times(m.v[0], n.v[0], sum)); }

// Numbers k .. k + RUN of a row, 0 from `end` on, by loads of AT_ONCE numbers: `end` is a multiple of that, not 0, and the row begins at a whole run of loads.  What lies beyond is asked for at the last
// load's place and dropped: a branch around a load would make the wave wait for all its loads where the first is used.
template <int AT_ONCE>
__device__ __forceinline__ uint4 load_run(const bf16_t* __restrict__ row, int k, int end) {
    if constexpr (AT_ONCE == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + min(k, end - 8));
        const bool in = k < end;
        return uint4{in ? v.x : 0u, in ? v.y : 0u, in ? v.z : 0u, in ? v.w : 0u};
    } else if constexpr (AT_ONCE == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + min(k, end - 4)), w = *reinterpret_cast<const uint2*>(row + min(k + 4, end - 4));
        const bool in = k < end, more = k + 4 < end;
        return uint4{in ? v.x : 0u, in ? v.y : 0u, more ? w.x : 0u, more ? w.y : 0u};
    } else {
        uint32_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = row[min(k + i, end - 1)];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < end ? v[i] : 0u;
        return uint4{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
    }
}
template <int AT_ONCE, typename T>
__device__ __forceinline__ float4 load_run_f32(const T* __restrict__ row, int k, int end) {
    float v[4];
    if constexpr (AT_ONCE == 4) {
        const int from = min(k, end - 4);
        if constexpr (std::is_same<T, float>::value) {
            const float4 w = *reinterpret_cast<const float4*>(row + from);
            v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(row + from);
            v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u); v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = load_f32(row, (size_t)min(k + i, end - 1));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < end ? v[i] : 0.f;
    return float4{v[0], v[1], v[2], v[3]};
}
template <int AT_ONCE, typename T>
__device__ __forceinline__ void load_piece(Piece<true>& p, const T* __restrict__ row, int k, int end, int group) {
#pragma unroll
    for (int h = 0; h < 2; ++h) p.v[h] = load_run<AT_ONCE>((const bf16_t*)row, k + 32 * h + 8 * group, end);
}
template <int AT_ONCE, typename T>
__device__ __forceinline__ void load_piece(Piece<false>& p, const T* __restrict__ row, int k, int end, int group) {
#pragma unroll
    for (int h = 0; h < 2; ++h) p.v[h] = load_run_f32<AT_ONCE>(row, k + 16 * h + 4 * group, end);
}

// A whole piece, from any place.
__device__ __forceinline__ void load_whole(Piece<true>& p, const bf16_t* __restrict__ row, int k, int group) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const Low8 v = *reinterpret_cast<const Low8*>(row + k + 32 * h + 8 * group);
        p.v[h] = uint4{v.x, v.y, v.z, v.w};
    }
}
__device__ __forceinline__ void load_whole(Piece<false>& p, const float* __restrict__ row, int k, int group) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const High4 v = *reinterpret_cast<const High4*>(row + k + 16 * h + 4 * group);
        p.v[h] = float4{v.x, v.y, v.z, v.w};
    }
}
__device__ __forceinline__ void load_whole(Piece<false>& p, const bf16_t* __restrict__ row, int k, int group) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const Low4 v = *reinterpret_cast<const Low4*>(row + k + 16 * h + 4 * group);
        p.v[h] = float4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
    }
}

// The tiles of a batch, counted by every workgroup: a tile begins at every 64th row and where a row's adapter is not its neighbour's.
constexpr int COUNTS = 1024;
template <int WAVES>                        // of a workgroup
struct Tiles {
    const int* ids;
    int n_rows, each, entries;              // rows; blocks of 64 rows that one count is of; counts

    __device__ unsigned long long begins(int block) const {            // the rows of a block at which tiles begin
        const int lane = threadIdx.x & 63, i = block * TILE + lane, mine = ids[min(i, n_rows - 1)], neighbour = lane_before(mine);
        return __ballot(i < n_rows && (lane == 0 || mine != neighbour));
    }
    // before[c]: tiles before the rows of count c; the number of all tiles comes back.
    __device__ int count(int* before) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, blocks = (n_rows + TILE - 1) / TILE;
        each = (blocks + COUNTS - 1) / COUNTS;
        entries = (blocks + each - 1) / each;
        constexpr int AT_ONCE = 8;                                     // counts of a wave whose rows' numbers are asked for together
        for (int c = wave; c < entries; c += AT_ONCE * WAVES) {
            int sum[AT_ONCE] = {};
            for (int b = 0; b < each; ++b) {
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) sum[u] += __popcll(begins((c + u * WAVES) * each + b));       // (a block beyond the rows has none)
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
                if (lane == 0 && c + u * WAVES < entries) before[c + u * WAVES] = sum[u];
        }
        __syncthreads();
        // every wave adds the counts up for itself and wave 0 lays the sums down
        int total = 0;
        int mine[COUNTS / 64];
#pragma unroll
        for (int u = 0; u < COUNTS / 64; ++u) {
            if (u * 64 >= entries) break;
            const int c = u * 64 + lane, v = c < entries ? before[c] : 0;
            const int upto = sum_up_to(v);
            mine[u] = total + upto - v;
            total += of_lane(upto, 63);
        }
        __syncthreads();
        if (wave == 0)
#pragma unroll
            for (int u = 0; u < COUNTS / 64; ++u) {
                if (u * 64 >= entries) break;
                if (u * 64 + lane < entries) before[u * 64 + lane] = mine[u];
            }
        __syncthreads();
        return total;
    }
    // Tile `which`: its first row, how many, and their adapter.  The same in every lane.
    __device__ void find(const int* before, int which, int& first, int& rows, int& id) const {
        const int lane = threadIdx.x & 63;
        int c = -1;
        for (int u = 0; u < entries; u += 64) c += __popcll(__ballot(u + lane < entries && before[u + lane] <= which));      // the last count that begins at or before it
        int left = which - before[c], block = c * each;
        unsigned long long at = begins(block);
        while (left >= __popcll(at)) {
            left -= __popcll(at);
            at = begins(++block);
        }
        const int place = __ffsll((long long)__ballot((at >> lane & 1) && __popcll(at & ((1ull << lane) - 1)) == left)) - 1;
        const unsigned long long behind = place < 63 ? at >> (place + 1) : 0;
        first = __builtin_amdgcn_readfirstlane(block * TILE + place);
        rows = __builtin_amdgcn_readfirstlane(min(behind != 0 ? __ffsll((long long)behind) : TILE - place, n_rows - block * TILE - place));
        id = __builtin_amdgcn_readfirstlane(ids[block * TILE + place]);
    }
};

struct Tile {                               // of the list that the way down leaves
    int first, rows, id, unused;
};

// A workgroup's pieces of work, every gridDim.x-th of `tiles` times `parts`, without a division for each.
struct Share {
    int tile, part, parts, by_tiles, by_parts;
    __device__ explicit Share(int of) : tile(blockIdx.x / of), part(blockIdx.x % of), parts(of), by_tiles(gridDim.x / of), by_parts(gridDim.x % of) {}
    __device__ void next() {
        tile += by_tiles;
        part += by_parts;
        if (part >= parts) { part -= parts; ++tile; }
    }
};

// ------------------------------------------------------------------ down, in tiles
// sums[segment][row][rank] of a tile, a segment of the width and a group of 16 MT ranks.  A workgroup's waves share out the segment, every second block of 128 bytes a row, so that none
// loads what the other does.  In the product D = M N the ranks are M's rows and the tile's rows N's columns: a lane of the result has values of one row only, and rows behind the tile's
// last are loaded as that one and dropped.
struct Down {
    Tile* list;
    int* n_listed;
    int n_rows, width, ranks, n_adapters, segment, n_segments, n_parts;       // parts: segments times groups of ranks
    long ldx;
};

template <int WAVES, int MT>
__device__ __forceinline__ void store_sums(floatx4 (&sum)[4][MT], unsigned char* meet, float* __restrict__ sums, const Down& d, int segment, int first_row, int rows, int first_rank) {
    // the waves' meet in `meet`, 4 KB * MT of each, which no wave reads as anything else any more
    floatx4* at = (floatx4*)meet;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
            if (16 * j < rows) at[(wave * 4 * MT + j * MT + i) * 64 + lane] = sum[j][i];
    __syncthreads();
    for (int item = threadIdx.x; item < 4 * MT * 64; item += 64 * WAVES) {
        const int l = item & 63, j = item / 64 / MT, i = item / 64 % MT;
        const int row = 16 * j + (l & 15), rank = first_rank + 16 * i + 4 * (l >> 4);
        if (row >= rows || rank >= d.ranks) continue;
        floatx4 s = at[item];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += at[item + w * 4 * MT * 64];
        float* to = sums + ((size_t)segment * d.n_rows + first_row + row) * d.ranks + rank;
        if ((d.ranks & 3) == 0) {
            *reinterpret_cast<floatx4*>(to) = s;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (rank + c < d.ranks) to[c] = s[c];
        }
    }
    __syncthreads();
}

// Rows of one type, 16-byte loads.  Global memory goes straight into LDS (a lane's 16 bytes land behind the lane's before it), every wave through a ring of its own, so that no barrier stands in the loop: in registers the
// operands' layout, neighbouring lanes in different rows, would take a load through the first-level cache in 64 pieces of 16 bytes instead of 16 whole sectors.  A stage is 64 rows of x and 16 MT of A,
// 128 bytes each, its 16-byte chunk c of a row at place c ^ (row / 2 % 8), so that 16 rows' chunks lie in different banks (the counters show no conflict).
// 4,096 rows of 14,336, rank 64: 37.5 us for 117 MB, 9 of them for counting tiles, the first loads and joining the waves' sums (without the products the time is the same); 2,048 of 2,048, rank 32, 6.7;
// 531 of 4,096, rank 3 * 24, 10.2; 301 of 2,048 in 32 bits, rank 10, 6.9.
constexpr int STAGES = 2;                   // (a third makes no difference of 1%: other workgroups of the unit load meanwhile)
template <int MT> constexpr int stage_bytes() { return (TILE + 16 * MT) * 128; }

template <bool LOW, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void adapters_down_kernel(const typename Piece<LOW>::T* __restrict__ x, const typename Piece<LOW>::T* __restrict__ a, const int* __restrict__ ids,
                                                           float* __restrict__ sums, Down d) {
    typedef Piece<LOW> P;
    typedef typename P::T T;
    constexpr int BYTES = stage_bytes<MT>(), LOADS = BYTES / 1024, STEP = P::BLOCK * WAVES;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ int before[COUNTS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & 15, group = lane >> 4;
    Tiles<WAVES> tiles{ids, d.n_rows, 0, 0};
    const int n_tiles = tiles.count(before);
    unsigned char* mine = ring + wave * STAGES * BYTES;
    const unsigned mine_at = (unsigned)(size_t)(lds_ptr_t)mine;
    for (Share work(d.n_parts); work.tile < n_tiles; work.next()) {
        int first_row, rows, e;
        const int part = work.part, which = work.tile;
        tiles.find(before, which, first_row, rows, e);
        if (part == 0 && threadIdx.x == 0) {
            d.list[which] = Tile{first_row, rows, e, 0};
            *d.n_listed = n_tiles;
        }
        if (e < 0 || e >= d.n_adapters) continue;
        const int segment = part % d.n_segments, first_rank = part / d.n_segments * 16 * MT;
        const int begin = segment * d.segment, end = min(d.width, begin + d.segment), k0 = begin + wave * P::BLOCK;
        const int whole = max(0, (end - k0 + (WAVES - 1) * P::BLOCK) / STEP);          // this wave's blocks
        const T* ae = a + (size_t)e * d.ranks * d.width;
        const T* from[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int row = 8 * i + (lane >> 3), c = (lane & 7) ^ (row >> 1 & 7);
            from[i] = (row < TILE ? x + (size_t)(first_row + min(row, rows - 1)) * d.ldx : ae + (size_t)min(first_rank + row - TILE, d.ranks - 1) * d.width) + k0 + P::RUN * c;
        }
        auto ask = [&](int block) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const unsigned to = __builtin_amdgcn_readfirstlane(mine_at + block % STAGES * BYTES + i * 1024);
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from[i] + (size_t)block * STEP) : "memory", "m0");
            }
        };
        floatx4 sum[4][MT];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) sum[j][i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s)
            if (s < whole) ask(s);
        for (int block = 0; block < whole; ++block) {
            // the block before has been read into registers; the next goes where it was
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (block + STAGES - 1 < whole) ask(block + STAGES - 1);
            const int ahead = min(whole - 1 - block, STAGES - 1);                      // blocks that may still be on their way
            if (ahead >= 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
            else if (ahead == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const unsigned char* stage = mine + block % STAGES * BYTES;
            P ap[MT];
            const int swizzle = at >> 1;                                               // (16 rows further it is the same)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    ap[i].v[h] = *reinterpret_cast<const typename P::V*>(stage + (TILE + 16 * i + at) * 128 + ((4 * h + group) ^ swizzle) * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (16 * j >= rows) break;
                P xp;
#pragma unroll
                for (int h = 0; h < 2; ++h) xp.v[h] = *reinterpret_cast<const typename P::V*>(stage + (16 * j + at) * 128 + ((4 * h + group) ^ swizzle) * 16);
#pragma unroll
                for (int i = 0; i < MT; ++i) sum[j][i] = times(ap[i], xp, sum[j][i]);
            }
        }
        if (k0 + whole * STEP < end) {                     // what is left of the segment behind the last block
            const int k = k0 + whole * STEP;
            P ap[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) load_piece<P::RUN>(ap[i], ae + (size_t)min(first_rank + 16 * i + at, d.ranks - 1) * d.width, k, end, group);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (16 * j >= rows) break;
                P xp;
                load_piece<P::RUN>(xp, x + (size_t)(first_row + min(16 * j + at, rows - 1)) * d.ldx, k, end, group);
#pragma unroll
                for (int i = 0; i < MT; ++i) sum[j][i] = times(ap[i], xp, sum[j][i]);
            }
        }
        store_sums<WAVES, MT>(sum, ring, sums, d, segment, first_row, rows, first_rank);
    }
}

// Operands of two types, or rows that do not begin at 16 bytes: through registers, in the same order, whole blocks by wide loads from any place.  2,048 rows of 4,096 onto 4,096, rank 16, both ways: two types 29 us, as
// both of 32 bits 27; rows at odd places 31 (32 bits) and 32 (bfloat16, at even ones 25).
template <bool LOW, typename X, typename W>
__global__ __launch_bounds__(64 * ANY_WAVES) void adapters_down_any_kernel(const X* __restrict__ x, const W* __restrict__ a, const int* __restrict__ ids, float* __restrict__ sums, Down d) {
    typedef Piece<LOW> P;
    constexpr int MT = 2;
    __shared__ __align__(16) unsigned char meet[ANY_WAVES * 4 * MT * 1024];
    __shared__ int before[COUNTS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & 15, group = lane >> 4;
    Tiles<ANY_WAVES> tiles{ids, d.n_rows, 0, 0};
    const int n_tiles = tiles.count(before);
    for (Share work(d.n_parts); work.tile < n_tiles; work.next()) {
        int first_row, rows, e;
        const int part = work.part, which = work.tile;
        tiles.find(before, which, first_row, rows, e);
        if (part == 0 && threadIdx.x == 0) {
            d.list[which] = Tile{first_row, rows, e, 0};
            *d.n_listed = n_tiles;
        }
        if (e < 0 || e >= d.n_adapters) continue;
        const int segment = part % d.n_segments, first_rank = part / d.n_segments * 16 * MT;
        const int begin = segment * d.segment, end = min(d.width, begin + d.segment);
        const W* ar[MT];
        const X* xr[4];
#pragma unroll
        for (int i = 0; i < MT; ++i) ar[i] = a + ((size_t)e * d.ranks + min(first_rank + 16 * i + at, d.ranks - 1)) * d.width;
#pragma unroll
        for (int j = 0; j < 4; ++j) xr[j] = x + (size_t)(first_row + min(16 * j + at, rows - 1)) * d.ldx;
        floatx4 sum[4][MT];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) sum[j][i] = floatx4{0.f, 0.f, 0.f, 0.f};
        int k = begin + wave * P::BLOCK;
        for (; k + P::BLOCK <= end; k += P::BLOCK * ANY_WAVES) {
            P ap[MT], xp[4];
#pragma unroll
            for (int i = 0; i < MT; ++i) load_whole(ap[i], ar[i], k, group);
#pragma unroll
            for (int j = 0; j < 4; ++j) load_whole(xp[j], xr[j], k, group);             // (rows behind the last are that one)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) sum[j][i] = times(ap[i], xp[j], sum[j][i]);
        }
        if (k < end) {
            P ap[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) load_piece<1>(ap[i], ar[i], k, end, group);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (16 * j >= rows) break;
                P xp;
                load_piece<1>(xp, xr[j], k, end, group);
#pragma unroll
                for (int i = 0; i < MT; ++i) sum[j][i] = times(ap[i], xp, sum[j][i]);
            }
        }
        store_sums<ANY_WAVES, MT>(sum, meet, sums, d, segment, first_row, rows, first_rank);
    }
}

// ------------------------------------------------------------------ up, in tiles
// 4 numbers of base, as they lie in memory and as numbers, and of out.
__device__ __forceinline__ uint4 raw4(const unsigned char* base, uint32_t i, bool low) {
    if (!low) {
        const High4 v = *reinterpret_cast<const High4*>(base + 4 * i);
        return uint4{__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w)};
    }
    const Low4 v = *reinterpret_cast<const Low4*>(base + 2 * i);
    return uint4{v.x, v.y, 0u, 0u};
}
__device__ __forceinline__ floatx4 numbers4(uint4 v, bool low) {
    if (!low) return __builtin_bit_cast(floatx4, v);
    return floatx4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
}
__device__ __forceinline__ void store4(unsigned char* out, uint32_t i, floatx4 v, bool low) {
    if (low) *reinterpret_cast<Low4*>(out + 2 * i) = Low4{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
    else *reinterpret_cast<High4*>(out + 4 * i) = High4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ float number1(const void* base, size_t i, bool low) { return low ? load_f32((const bf16_t*)base, i) : load_f32((const float*)base, i); }
__device__ __forceinline__ void store1(void* out, size_t i, float v, bool low) { low ? store_f32((bf16_t*)out, i, v) : store_f32((float*)out, i, v); }

struct Rows {                               // base and out
    const void* base;
    void* out;
    long ldb, ldo;
    bool low_base, low_out;                 // bfloat16
};

constexpr int PIECES = 3;                   // bfloat16 numbers that hold a 32-bit one: each the first 8 bits of what the ones before leave of its 24, cut off, so that none passes the number

// One run along the ranks of 16 columns of B.
template <bool LOW> struct Run { uint4 v; };
template <> struct Run<false> { float4 v; };
template <int AT_ONCE, typename W> __device__ __forceinline__ void load_b(Run<true>& m, const W* row, int k, int rank) { m.v = load_run<AT_ONCE>((const bf16_t*)row, k, rank); }
template <int AT_ONCE, typename W> __device__ __forceinline__ void load_b(Run<false>& m, const W* row, int k, int rank) { m.v = load_run_f32<AT_ONCE>(row, k, rank); }

// One run of a row's sums, in pieces; they lie `apart` numbers behind one another.
template <bool LOW> struct Held { bf16x8 v[PIECES]; };
template <> struct Held<false> { float4 v; };
__device__ __forceinline__ void load_row(Held<true>& t, const bf16_t* row, int apart) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) t.v[p] = *reinterpret_cast<const bf16x8*>(row + p * apart);
}
__device__ __forceinline__ floatx4 times(const Held<true>& t, const Run<true>& n, floatx4 sum) {
#pragma unroll
    for (int p = PIECES - 1; p >= 0; --p) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(t.v[p], __builtin_bit_cast(bf16x8, n.v), sum, 0, 0, 0);
    return sum;
}
__device__ __forceinline__ void load_row(Held<false>& t, const float* row, int) { t.v = *reinterpret_cast<const float4*>(row); }
__device__ __forceinline__ floatx4 times(const Held<false>& t, const Run<false>& n, floatx4 sum) { return times(t.v, n.v, sum); }

// A strip's workgroup first makes its rows' sums, so strips are as long as leaves every compute unit (of 256) two or three workgroups, by the number of tiles that the way down has counted
// (600 rows with adapters of their own, 4,096 columns, rank 32: 135 us both ways; with strips for as many rows in whole tiles 466).  Aimed at 350 and 700
// workgroups, 1,024 rows of 2,048 32-bit columns and rank 64 take 36.4 and 29.1 us both ways, 2,048 rows of 2,048 columns and rank 32 19.1 either way.  All four waves have columns of their own, 256 a step of the
// strip (strips of other multiples of 64: 531 rows 31.0 us instead of 26.5), or, where there are no 256 for each, rows of the same 64 (301 rows of 1,024 in 32 bits: 13.0 us instead of 14.5).  Strips end at 512
// columns (8,192 rows of 14,336 columns: 236 us at 256, 219 at 512, 239 at 1,024).
__host__ __device__ inline int strip_bits(int n_tiles, int columns) {          // 64, 256 or 512 columns
    const long work = (long)n_tiles * columns;
    return work <= 700l * 64 ? 6 : work <= 700l * 256 ? 8 : 9;
}

// A tile and a strip of columns.  The workgroup first adds up its rows' sums over the segments and keeps them in LDS: where B is bfloat16 and so multiplied, in PIECES, which lose nothing of their 24 bits.
// Then a wave takes 64 columns at a time and of them 16 rows after 16 rows, with the columns' runs of B in registers throughout (loaded, they lie as the matrix cores want them, every lane in another
// row of B: 64 accesses to the first-level cache a load); where the strip is no wider than 64 columns the waves share out the rows.  In the product D = M N the rows are M's and the columns
// N's: number n of the four products of a step has columns 4 l + n, l = 0 .. 15, so that a lane ends with four neighbours and sixteen lanes with whole lines of base and out.  As on the way down no
// row's values meet another's.  FOURS: a projection has four columns or more, so base and out come four at a time.  AT_ONCE: numbers of B that one load brings.  KS: runs of ranks that a wave keeps; 0 for any number,
// loaded again for every 16 rows (8,192 rows of 14,336 columns, rank 16: 239 us kept, 272 loaded again).  LOW_BASE, LOW_OUT: of aligned ones whether they are bfloat16 (a branch on it where they are loaded would have every load waited for); `io` says it of others.
// 4,096 rows of 4,096 32-bit columns, rank 64: 41 us for the 134 MB of base and out (a copy of as much takes 25; every one of a tile's eight strips adds up its rows' sums over the segments anew, 25 MB in all,
// before its first product, with one step's base under way beside it: no more is known of the difference); 531 of 6,144, rank 24, onto bfloat16 10.3; 2,048 of 2,048, rank 32, 9.4; 301 of 2,048 in 32 bits,
// rank 10, 8.4.  Asking for a whole tile's base at once instead of 16 rows ahead makes it no faster: 4,096 rows of 4,096 both ways 50 us instead of 47, with 256 registers instead of 141.
template <bool LOW, typename W, bool FOURS, int AT_ONCE, int KS, bool LOW_BASE, bool LOW_OUT>
__global__ __launch_bounds__(UP_NT) void adapters_up_kernel(const float* __restrict__ sums, const W* __restrict__ b, const float* __restrict__ scales, const Tile* __restrict__ list,
                                                            const int* __restrict__ n_listed, Rows io, int n_rows, int rank, int n_segments, Slices slices, int n_adapters) {
    typedef Piece<LOW> P;
    typedef typename P::T T;
    extern __shared__ __align__(16) unsigned char room[];
    constexpr int DEPTH = P::BLOCK / 2;                    // ranks of a matrix instruction (of four, in 32 bits)
    const int padded = KS > 0 ? KS * DEPTH : (rank + DEPTH - 1) / DEPTH * DEPTH, pitch = padded + P::RUN, apart = TILE * pitch;       // (rows of LDS a run further apart than a multiple of all banks)
    T* held = (T*)room;                                    // [pieces][TILE][pitch], the largest piece first
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & 15, group = lane >> 4;
    const int columns = slices.begin[slices.n], ranks = rank * slices.n, n_tiles = *n_listed, bits = strip_bits(n_tiles, columns), strip_columns = 1 << bits;
    auto strips_of = [&](int s) { return (slices.begin[s + 1] - slices.begin[s] + strip_columns - 1) >> bits; };
    int n_strips = 0;
    for (int s = 0; s < slices.n; ++s) n_strips += strips_of(s);
    for (Share work(n_strips); work.tile < n_tiles; work.next()) {
        int strip = work.part, s = 0;
        for (; s + 1 < slices.n && strip >= strips_of(s); ++s) strip -= strips_of(s);
        const int begin = slices.begin[s] + strip * strip_columns, end = min(slices.begin[s + 1], begin + strip_columns);
        const Tile tile = list[work.tile];
        const int first_row = tile.first, rows = tile.rows, e = tile.id;
        if (e < 0 || e >= n_adapters) {                    // rows without an adapter
            if (io.base != io.out)
                for (int r = first_row; r < first_row + rows; ++r)
                    for (int c = begin + threadIdx.x; c < end; c += UP_NT) store1(io.out, (size_t)r * io.ldo + c, number1(io.base, (size_t)r * io.ldb + c, io.low_base), io.low_out);
            continue;
        }
        const W* be = b + (size_t)e * columns * rank;
        const bool by_rows = strip_columns == 64;
        const int j_step = by_rows ? UP_WAVES : 1, last_j = (rows - 1) / 16;
        const unsigned char* base_at = (const unsigned char*)io.base + (size_t)first_row * io.ldb * (io.low_base ? 2 : 4);
        unsigned char* out_at = (unsigned char*)io.out + (size_t)first_row * io.ldo * (io.low_out ? 2 : 4);
        Run<LOW> br[KS == 0 ? 1 : KS][4];
        uint4 next[4];
        auto ask_b = [&](int c0) {                         // for a step's columns of B
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int n = 0; n < 4; ++n) load_b<AT_ONCE>(br[k][n], be + (size_t)(min(c0 + 4 * at, end - 4) + n) * rank, DEPTH * k + P::RUN * group, rank);
        };
        // Rows behind the last are taken as that one throughout, and columns behind the end as the last four: their lanes load and store what the lanes that own them do, at the same time.  Without a branch
        // around any store the wait for a load counts what was asked for behind it, and no load waits for a store's end.
        auto ask_base = [&](int c0, int j) {
            if constexpr (FOURS)
#pragma unroll
                for (int i = 0; i < 4; ++i) next[i] = raw4(base_at, (uint32_t)(min(16 * j + 4 * group + i, rows - 1) * (int)io.ldb + min(c0 + 4 * at, end - 4)), LOW_BASE);
        };
        int c0 = begin + (by_rows ? 0 : 64 * wave);
        const int j0 = by_rows ? wave : 0;
        const bool idle = c0 >= end || j0 > last_j;
        if (!idle) {                                       // the first step's come while the rows' sums are made
            ask_b(c0);
            ask_base(c0, j0);
        }
        const float scale = scales != nullptr ? scales[e] : 1.f;
        const int n_fours = ((rows + 15) & ~15) * (padded / 4);
        const size_t further = (size_t)n_rows * ranks;
        __syncthreads();                                   // (the item before has been read)
        for (int i0 = threadIdx.x; i0 < n_fours; i0 += 2 * UP_NT) {            // four ranks of a row at a time, and twice that, of four segments
            floatx4 v[2];
            const float* from[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int i = min(i0 + q * UP_NT, n_fours - 1);
                from[q] = sums + (size_t)(first_row + min(i / (padded / 4), rows - 1)) * ranks + s * rank;
                v[q] = floatx4{0.f, 0.f, 0.f, 0.f};
            }
            for (int seg = 0; seg < n_segments; seg += 4) {
                floatx4 part[4][2];
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int k = min(i0 + q * UP_NT, n_fours - 1) % (padded / 4) * 4;
                        const float* p = from[q] + min(seg + u, n_segments - 1) * further;
                        if ((rank & 3) == 0) part[u][q] = *reinterpret_cast<const floatx4*>(p + min(k, rank - 4));
                        else
#pragma unroll
                            for (int c = 0; c < 4; ++c) part[u][q][c] = p[min(k + c, rank - 1)];
                    }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        if (seg + u < n_segments) v[q] += part[u][q];
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int i = i0 + q * UP_NT, r = i / (padded / 4), k = i % (padded / 4) * 4;
                if (i >= n_fours) break;
                v[q] *= scale;
#pragma unroll
                for (int c = 0; c < 4; ++c) v[q][c] = k + c < rank ? v[q][c] : 0.f;
                if constexpr (LOW) {
#pragma unroll
                    for (int p = 0; p < PIECES; ++p) {
                        uint32_t top[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            top[c] = __float_as_uint(v[q][c]) & 0xffff0000u;
                            const float left = v[q][c] - __uint_as_float(top[c]);
                            v[q][c] = left == left ? left : 0.f;                       // (nothing is left of an infinity, or of no number)
                        }
                        *reinterpret_cast<uint2*>(held + p * apart + r * pitch + k) = uint2{top[0] >> 16 | top[1], top[2] >> 16 | top[3]};
                    }
                } else {
                    *reinterpret_cast<floatx4*>(held + r * pitch + k) = v[q];
                }
            }
        }
        __syncthreads();
        if (idle) continue;
        const int further_columns = by_rows ? 64 : 64 * UP_WAVES;
        while (true) {
            const int col = FOURS ? min(c0 + 4 * at, end - 4) : c0 + 4 * at;
            auto products = [&](int j, floatx4 (&sum)[4]) {
#pragma unroll
                for (int n = 0; n < 4; ++n) sum[n] = floatx4{0.f, 0.f, 0.f, 0.f};
                const T* row = held + (16 * j + at) * pitch + P::RUN * group;
                Held<LOW> t;
                if constexpr (KS > 0) {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        load_row(t, row + DEPTH * k, apart);
#pragma unroll
                        for (int n = 0; n < 4; ++n) sum[n] = times(t, br[k][n], sum[n]);
                    }
                } else {
                    for (int k = 0; k < padded; k += DEPTH) {
#pragma unroll
                        for (int n = 0; n < 4; ++n) load_b<AT_ONCE>(br[0][n], be + (size_t)(FOURS ? col + n : min(col + n, end - 1)) * rank, k + P::RUN * group, rank);
                        load_row(t, row + k, apart);
#pragma unroll
                        for (int n = 0; n < 4; ++n) sum[n] = times(t, br[0][n], sum[n]);
                    }
                }
            };
            if (!FOURS || end - c0 < 4) {                  // one by one; of the last four columns those before c0 are another wave's, which may have stored them already
#pragma unroll 1
                for (int j = j0; j <= last_j; j += j_step) {
                    floatx4 sum[4];
                    products(j, sum);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = 16 * j + 4 * group + i;
                        if (r >= rows) continue;
                        const uint32_t to = (uint32_t)(r * (int)io.ldo + col);
#pragma unroll
                        for (int n = 0; n < 4; ++n)
                            if (col + n >= c0 && col + n < end) store1(out_at, to + n, number1(base_at, (size_t)(uint32_t)(r * (int)io.ldb + col + n), io.low_base) + sum[n][i], io.low_out);
                    }
                }
            } else {
#pragma unroll 1
                for (int j = j0; j <= last_j; j += j_step) {
                    uint4 was[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) was[i] = next[i];
                    const bool last = j + j_step > last_j;                             // the next columns' first rows are asked for behind these columns' last
                    ask_base(last ? c0 + further_columns : c0, last ? j0 : j + j_step);
                    floatx4 sum[4];
                    products(j, sum);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t to = (uint32_t)(min(16 * j + 4 * group + i, rows - 1) * (int)io.ldo + col);
                        store4(out_at, to, numbers4(was[i], LOW_BASE) + floatx4{sum[0][i], sum[1][i], sum[2][i], sum[3][i]}, LOW_OUT);
                    }
                }
            }
            c0 += further_columns;
            if (c0 >= end) break;
            ask_b(c0);
        }
    }
}

// ------------------------------------------------------------------ a few rows
template <int N> struct Some;               // N bfloat16 numbers, loaded at once
template <> struct Some<8> { Low8 v; __device__ float operator[](int i) const { const uint32_t w[4] = {v.x, v.y, v.z, v.w}; return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); } };
template <> struct Some<4> { Low4 v; __device__ float operator[](int i) const { const uint32_t w[2] = {v.x, v.y}; return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); } };
template <> struct Some<2> { Low2 v; __device__ float operator[](int i) const { return __uint_as_float(i & 1 ? v.x & 0xffff0000u : v.x << 16); } };
template <> struct Some<1> { bf16_t v; __device__ float operator[](int) const { return bf16_to_f32(v); } };

// Decoded rows, as a rule each with an adapter of its own: nothing is shared, the adapters' bytes bound it, and what counts is that all of them are asked for at once and few waits
// follow one another.  Every row is taken alone, without tiles.  Down: a workgroup has a row and one rank, its threads share out the width.  (With four ranks, which share the row's numbers, 8 rows of
// 4,096 onto 4,096, rank 32, take 6.2 us instead of 5.6, 128 rows 18.8 instead of 18.0; rows that share an adapter of 2 MB gain a tenth.)  64 rows of 4,096, rank 16: 4.1 us.
__global__ __launch_bounds__(256) void adapters_down_few_kernel(const bf16_t* __restrict__ x, long ldx, const bf16_t* __restrict__ a, const int* __restrict__ ids, float* __restrict__ sums,
                                                                int width, int ranks, int n_adapters) {
    __shared__ float red[4];
    const int row = blockIdx.y, tid = threadIdx.x;
    const int e = ids[row];
    if (e < 0 || e >= n_adapters) return;
    const bf16_t* xr = x + (size_t)row * ldx;
    const bf16_t* ar = a + ((size_t)e * ranks + blockIdx.x) * width;
    const int eights = width & ~7;
    float sum = tid < width - eights ? bf16_to_f32(xr[eights + tid]) * bf16_to_f32(ar[eights + tid]) : 0.f;
#pragma unroll 2
    for (int k = 8 * tid; k < eights; k += 2048) {
        const Some<8> xv = *reinterpret_cast<const Some<8>*>(xr + k), av = *reinterpret_cast<const Some<8>*>(ar + k);
#pragma unroll
        for (int u = 0; u < 8; ++u) sum = fmaf(xv[u], av[u], sum);
    }
    sum = over_wave(sum, Add());
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) sums[(size_t)row * ranks + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Up: a thread has FEW_COLUMNS columns, 256 apart, of a row; the row's sums come as scalars.  64 rows of 14,336, rank 16: 7.4 us for 37 MB (5 TB/s).
constexpr int FEW_COLUMNS = 2;
// The ranks' sums times N of them of each of a thread's columns, from rank k on.
template <int N>
__device__ __forceinline__ void add_ranks(float (&sum)[FEW_COLUMNS], const float* t, const bf16_t* const (&br)[FEW_COLUMNS], int k) {
    Some<N> v[FEW_COLUMNS];
#pragma unroll
    for (int c = 0; c < FEW_COLUMNS; ++c) v[c] = *reinterpret_cast<const Some<N>*>(br[c] + k);
#pragma unroll
    for (int c = 0; c < FEW_COLUMNS; ++c)
#pragma unroll
        for (int u = 0; u < N; ++u) sum[c] = fmaf(t[k + u], v[c][u], sum[c]);
}
__device__ __forceinline__ void add_last_ranks(float (&sum)[FEW_COLUMNS], const float* t, const bf16_t* const (&br)[FEW_COLUMNS], int rank) {       // those behind the last eight
    int k = rank & ~7;
    if (rank & 4) { add_ranks<4>(sum, t, br, k); k += 4; }
    if (rank & 2) { add_ranks<2>(sum, t, br, k); k += 2; }
    if (rank & 1) add_ranks<1>(sum, t, br, k);
}

__global__ __launch_bounds__(256) void adapters_up_few_kernel(const float* __restrict__ sums, const bf16_t* __restrict__ b, const float* __restrict__ scales, const int* __restrict__ ids,
                                                              Rows io, int rank, Slices slices, int n_adapters) {
    const int row = blockIdx.y;
    int s = 0;
    while (s + 1 < slices.n && (int)blockIdx.x >= slices.strip[s + 1]) ++s;
    const int begin = slices.begin[s] + ((int)blockIdx.x - slices.strip[s]) * 256 * FEW_COLUMNS + threadIdx.x, end = slices.begin[s + 1];
    const int e = ids[row];
    const bool some = e >= 0 && e < n_adapters;
    if (!some && io.base == io.out) return;
    float was[FEW_COLUMNS], sum[FEW_COLUMNS];
#pragma unroll
    for (int c = 0; c < FEW_COLUMNS; ++c) {
        was[c] = number1(io.base, (size_t)row * io.ldb + min(begin + 256 * c, end - 1), io.low_base);
        sum[c] = 0.f;
    }
    if (some) {
        const float* t = sums + (size_t)row * rank * slices.n + s * rank;
        const bf16_t* br[FEW_COLUMNS];
#pragma unroll
        for (int c = 0; c < FEW_COLUMNS; ++c) br[c] = b + ((size_t)e * slices.begin[slices.n] + min(begin + 256 * c, end - 1)) * rank;
        const float scale = scales != nullptr ? scales[e] : 1.f;
        for (int k = 0; k + 8 <= rank; k += 8) add_ranks<8>(sum, t, br, k);
        add_last_ranks(sum, t, br, rank);
#pragma unroll
        for (int c = 0; c < FEW_COLUMNS; ++c) was[c] = fmaf(scale, sum[c], was[c]);
    }
#pragma unroll
    for (int c = 0; c < FEW_COLUMNS; ++c)
        if (begin + 256 * c < end) store1(io.out, (size_t)row * io.ldo + begin + 256 * c, was[c], io.low_out);
}

bool aligned(const void* p, int bytes) { return (size_t)p % bytes == 0; }

// Both ways in one launch, where making a row's sums anew for every strip of its columns costs less than a second launch: a wave makes every fourth sum, then a thread has its columns as above.  One
// row of 2,048 onto 2,048, rank 16: 4.4 us, the waits of three loads that follow one another.
__global__ __launch_bounds__(256) void adapters_both_few_kernel(const bf16_t* __restrict__ x, long ldx, const bf16_t* __restrict__ a, const bf16_t* __restrict__ b, const float* __restrict__ scales,
                                                                const int* __restrict__ ids, Rows io, int width, int rank, Slices slices, int n_adapters) {
    __shared__ float t[MAX_RANK];
    const int row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = 0;
    while (s + 1 < slices.n && (int)blockIdx.x >= slices.strip[s + 1]) ++s;
    const int begin = slices.begin[s] + ((int)blockIdx.x - slices.strip[s]) * 256 * FEW_COLUMNS + threadIdx.x, end = slices.begin[s + 1];
    const int e = ids[row];
    const bool some = e >= 0 && e < n_adapters;
    if (!some && io.base == io.out) return;
    float was[FEW_COLUMNS], sum[FEW_COLUMNS];
#pragma unroll
    for (int c = 0; c < FEW_COLUMNS; ++c) {
        was[c] = number1(io.base, (size_t)row * io.ldb + min(begin + 256 * c, end - 1), io.low_base);
        sum[c] = 0.f;
    }
    if (some) {
        const bf16_t* br[FEW_COLUMNS];
        Some<8> v[FEW_COLUMNS] = {};
#pragma unroll
        for (int c = 0; c < FEW_COLUMNS; ++c) {
            br[c] = b + ((size_t)e * slices.begin[slices.n] + min(begin + 256 * c, end - 1)) * rank;
            if (rank >= 8) v[c] = *reinterpret_cast<const Some<8>*>(br[c]);
        }
        const float scale = scales != nullptr ? scales[e] : 1.f;
        const bf16_t* xr = x + (size_t)row * ldx;
        const bf16_t* ae = a + ((size_t)e * slices.n + s) * rank * width;
        const int eights = width & ~7;
        for (int k0 = 0; k0 < rank; k0 += 16) {            // four sums of a wave at a time
            const bf16_t* ar[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ar[i] = ae + (size_t)min(k0 + wave + 4 * i, rank - 1) * width;
            float four[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) four[i] = lane < width - eights ? bf16_to_f32(xr[eights + lane]) * bf16_to_f32(ar[i][eights + lane]) : 0.f;
#pragma unroll 2
            for (int k = 8 * lane; k < eights; k += 512) {
                const Some<8> xv = *reinterpret_cast<const Some<8>*>(xr + k);
                Some<8> av[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) av[i] = *reinterpret_cast<const Some<8>*>(ar[i] + k);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 8; ++u) four[i] = fmaf(xv[u], av[i][u], four[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                four[i] = over_wave(four[i], Add());
                if (lane == 0 && k0 + wave + 4 * i < rank) t[k0 + wave + 4 * i] = four[i];
            }
        }
        __syncthreads();
        for (int k = 0; k + 8 <= rank; k += 8) {
#pragma unroll
            for (int c = 0; c < FEW_COLUMNS; ++c) {
                const Some<8> now = v[c];
                if (k + 16 <= rank) v[c] = *reinterpret_cast<const Some<8>*>(br[c] + k + 8);
#pragma unroll
                for (int u = 0; u < 8; ++u) sum[c] = fmaf(t[k + u], now[u], sum[c]);
            }
        }
        add_last_ranks(sum, t, br, rank);
#pragma unroll
        for (int c = 0; c < FEW_COLUMNS; ++c) was[c] = fmaf(scale, sum[c], was[c]);
    }
#pragma unroll
    for (int c = 0; c < FEW_COLUMNS; ++c)
        if (begin + 256 * c < end) store1(io.out, (size_t)row * io.ldo + begin + 256 * c, was[c], io.low_out);
}

struct Call {
    const void* x; long ldx; const void* a; const void* b; const int* ids; const float* scales; Rows io; float* sums; Tile* list; int* n_listed;
    int n_rows, width, columns, rank, n_adapters, segment, n_segments;
    Slices slices;
    bool fours;                             // every projection has four columns or more
    hipStream_t stream;
};

// At most so many tiles: every 64th row begins one, and every row may.  Workgroups beyond the work there is leave at once, ones short of it come again.
long most_tiles(int n_rows) { return n_rows; }
// ... and about so many where the rows are a few requests'.
long usual_tiles(int n_rows) { return (n_rows + TILE - 1) / TILE; }

// Lets a kernel have `bytes` of LDS, asked for once per device.
constexpr int MAX_DEVICES = 64;
int raise_lds(const void* kernel, int bytes, bool (&raised)[MAX_DEVICES]) {
    int device = -1;
    if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= MAX_DEVICES) return gi_fail("adapters_add: no current device");
    if (!raised[device]) {
        if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return gi_fail("adapters_add: cannot reserve %d bytes of LDS", bytes);
        raised[device] = true;
    }
    return 0;
}

template <bool LOW, int MT, int WAVES>
int down_launch(const Call& c, Down d) {
    constexpr int lds = WAVES * STAGES * stage_bytes<MT>();
    static_assert(lds >= WAVES * 4 * MT * 1024 && lds + 4 * COUNTS <= 163840, "the waves' sums meet in the ring");
    d.n_parts = d.n_segments * ((d.ranks + 16 * MT - 1) / (16 * MT));
    const long items = most_tiles(c.n_rows) * d.n_parts;
    const int grid = (int)min(items, (long)gi_compute_units() * (163840 / (lds + 4 * COUNTS)));
    typedef typename Piece<LOW>::T T;
    static bool raised[MAX_DEVICES] = {};
    if (raise_lds((const void*)adapters_down_kernel<LOW, MT, WAVES>, lds, raised) != 0) return -1;
    adapters_down_kernel<LOW, MT, WAVES><<<grid, 64 * WAVES, lds, c.stream>>>((const T*)c.x, (const T*)c.a, c.ids, c.sums, d);
    return 0;
}

// Four waves share a tile's segment, always in 32 bits, where the order of sums must not depend on the batch, or two.  Twice as many loads are under way with four, but of their workgroups a compute unit holds one
// only: they gain where its tiles are whole (16,384 rows of 1,024, rank 16, both ways: 45.2 us instead of 50.9; 4,096 of 14,336, rank 64: 78.9 instead of 81.7; 301 of 1,024 in 32 bits 11.5 instead of 12.9) and lose
// where requests of one row bring many tiles more (531 rows of 4,096, of them 19 alone, rank 3 * 24: 22.1 instead of 20.5).  Those are few beside the tiles of 2,048 rows.
template <bool LOW, int MT>
int down_sized(const Call& c, const Down& d) {
    if constexpr (LOW)
        if (c.n_rows < 2048) return down_launch<LOW, MT, 2>(c, d);
    return down_launch<LOW, MT, 4>(c, d);
}

template <bool LOW, typename X, typename W>
int down(const Call& c) {
    const int ranks = c.rank * c.slices.n, run = Piece<LOW>::RUN;
    Down d{c.list, c.n_listed, c.n_rows, c.width, ranks, c.n_adapters, c.segment, c.n_segments, 0, c.ldx};
    const bool even = c.width % run == 0 && c.ldx % run == 0 && aligned(c.x, run * sizeof(X)) && aligned(c.a, run * sizeof(W));
    if constexpr (std::is_same<X, W>::value) {
        if (even) {
            const int groups = (ranks + 63) / 64, mt = ((ranks + groups - 1) / groups + 15) / 16;
            return mt == 1 ? down_sized<LOW, 1>(c, d) : mt == 2 ? down_sized<LOW, 2>(c, d) : mt == 3 ? down_sized<LOW, 3>(c, d) : down_sized<LOW, 4>(c, d);
        }
    }
    d.n_parts = d.n_segments * ((ranks + 31) / 32);
    const int grid = (int)min(most_tiles(c.n_rows) * d.n_parts, (long)gi_compute_units() * 8);
    adapters_down_any_kernel<LOW, X, W><<<grid, 64 * ANY_WAVES, 0, c.stream>>>((const X*)c.x, (const W*)c.a, c.ids, c.sums, d);
    return 0;
}

// Bytes of LDS that the way up keeps a tile's sums in.
template <bool LOW, int KS> constexpr int up_lds(int rank) {
    constexpr int DEPTH = Piece<LOW>::BLOCK / 2;
    if (KS > 0) rank = KS * DEPTH;
    return TILE * ((rank + DEPTH - 1) / DEPTH * DEPTH + Piece<LOW>::RUN) * (LOW ? 2 * PIECES : 4);
}

template <bool LOW, typename W, bool FOURS, int AT_ONCE, int KS, bool LOW_BASE, bool LOW_OUT>
int up_launch(const Call& c) {
    static bool raised[MAX_DEVICES] = {};
    constexpr int most = up_lds<LOW, KS>(MAX_RANK);
    if (raise_lds((const void*)adapters_up_kernel<LOW, W, FOURS, AT_ONCE, KS, LOW_BASE, LOW_OUT>, most, raised) != 0) return -1;
    const int grid = (int)min((long)c.n_rows * ((c.columns + 63) / 64 + c.slices.n), 4l * gi_compute_units());
    adapters_up_kernel<LOW, W, FOURS, AT_ONCE, KS, LOW_BASE, LOW_OUT><<<grid, UP_NT, up_lds<LOW, KS>(c.rank), c.stream>>>(c.sums, (const W*)c.b, c.scales, c.list, c.n_listed, c.io, c.n_rows, c.rank,
                                                                                                               c.n_segments, c.slices, c.n_adapters);
    return 0;
}

template <bool LOW, typename W, int AT_ONCE, int KS>
int up_sized(const Call& c) {
    if (c.io.low_base) return c.io.low_out ? up_launch<LOW, W, true, AT_ONCE, KS, true, true>(c) : up_launch<LOW, W, true, AT_ONCE, KS, true, false>(c);
    return c.io.low_out ? up_launch<LOW, W, true, AT_ONCE, KS, false, true>(c) : up_launch<LOW, W, true, AT_ONCE, KS, false, false>(c);
}

template <bool LOW, typename W>
int up(const Call& c) {
    const int steps = (c.rank + Piece<LOW>::BLOCK / 2 - 1) / (Piece<LOW>::BLOCK / 2);
    // What a wave keeps of B it has for all rows of a tile: of four runs that pays where it takes them all (8,192 rows of 14,336 columns, rank 128: 309 us both ways instead of 526; 4,096 of 4,096, rank 96, 58 instead
    // of 68), not where the waves share the rows out (600 of 4,096, rank 128: 43 us instead of 32; 1,024 of 2,048 in 32 bits, rank 64, 28 instead of 26).
    const bool keeps_four = steps <= 4 && strip_bits((int)usual_tiles(c.n_rows), c.columns) > 6;       // (then the strips there are, of at least as many tiles, are no shorter)
    // B's rows begin at whole loads only where the rank is a multiple of one, so of other ranks B comes in halves of a run or number by number, and again for every 16 rows once a run of ranks does not hold
    // them.  2,048 rows of 4,096 onto 4,096, both ways: bfloat16, rank 31, 32: 31 and 26 us; 33, 36, 40: 57, 34 and 30; 50, 56: 67 and 30; 32 bits, rank 10, 16: 29 and 26 us; 33, 36: 66 and 40; 50, 56: 102 and 44.
    // (An adapter filled up with zeros to the next multiple of 8 gives the same numbers at that rank's time.)
    constexpr int RUN = Piece<LOW>::RUN;
    if (!c.fours) return up_launch<LOW, W, false, 1, 0, false, false>(c);
    if (c.rank % RUN == 0 && aligned(c.b, RUN * sizeof(W)))
        return steps == 1 ? up_sized<LOW, W, RUN, 1>(c) : steps == 2 ? up_sized<LOW, W, RUN, 2>(c) : keeps_four ? up_sized<LOW, W, RUN, 4>(c) : up_sized<LOW, W, RUN, 0>(c);
    if constexpr (LOW)
        if (c.rank % 4 == 0 && aligned(c.b, 8)) return steps == 1 ? up_sized<LOW, W, 4, 1>(c) : up_sized<LOW, W, 4, 0>(c);
    return steps == 1 ? up_sized<LOW, W, 1, 1>(c) : up_sized<LOW, W, 1, 0>(c);
}

// bfloat16 rows few enough that loading an adapter once for every row that takes it costs less than tiles that share it.  Only the device knows which rows share:
// with an adapter a row tiles lose (64 rows of 4,096 onto 4,096, rank 32: 10.5 us against 15.5; 256: 31 against 45; 512 of 2,048 onto 2,048, rank 16: 17 against 46), with one for all the two meet at some
// 150 MB loaded (256 of 4,096 onto 4,096: 134 MB, 12.5 us against 13.5; 128 of 8,192 onto 2,048, rank 64: 168 MB, 19.1 against 19.6; 512 of 2,048 onto 8,192, rank 16: as many, 17.8 against 14.7; 256 of 8,192 onto
// 2,048: 336 MB, 36 against 20, and 102 against 76 with an adapter each) and at fewer where there are more rows (768 of 2,048 onto 2,048: 100 MB, 12.6 against 13.0; 1,024: 134 MB, 16.9 against 13.7).
bool few_rows(const Call& c) {
    const long loaded = 2l * c.n_rows * c.rank * ((long)c.slices.n * c.width + c.columns);
    return c.n_rows <= 512 && loaded <= 160 << 20;
}

void add_few(const Call& c) {
    const int ranks = c.rank * c.slices.n;
    Slices slices = c.slices;
    for (int s = 0; s < slices.n; ++s) slices.strip[s + 1] = slices.strip[s] + (slices.begin[s + 1] - slices.begin[s] + 256 * FEW_COLUMNS - 1) / (256 * FEW_COLUMNS);
    const dim3 strips(slices.strip[slices.n], c.n_rows);
    const long again = (long)c.rank * c.width * 2;         // bytes of A that every strip's workgroup reads
    // One launch takes the host 3 us less than two, and the device no longer where a workgroup reads 64 KB of A again (1 row of 2,048 onto 2,048 or 8,192, rank 16: 4.1 and 4.2 us against 4.6 and 4.7); at 128 KB 5.1 us
    // against 4.7, at 256 KB 7.7 against 5.5, and 40 rows onto 8,192 columns 6.7 against 5.6.
    if (again <= 64 << 10 && again * strips.x * strips.y <= 16 << 20) {
        adapters_both_few_kernel<<<strips, 256, 0, c.stream>>>((const bf16_t*)c.x, c.ldx, (const bf16_t*)c.a, (const bf16_t*)c.b, c.scales, c.ids, c.io, c.width, c.rank, slices, c.n_adapters);
        return;
    }
    adapters_down_few_kernel<<<dim3(ranks, c.n_rows), 256, 0, c.stream>>>((const bf16_t*)c.x, c.ldx, (const bf16_t*)c.a, c.ids, c.sums, c.width, ranks, c.n_adapters);
    adapters_up_few_kernel<<<strips, 256, 0, c.stream>>>(c.sums, (const bf16_t*)c.b, c.scales, c.ids, c.io, c.rank, slices, c.n_adapters);
}

// In 32 bits only the width says how long a segment is: few rows want many (64 of 14,336 onto 4,096, rank 16: 18.8, 20.0 and 22.8 us with 16, 12 and 8 at most, 21.8 always at 256 numbers), many rows few
// (2,048 of 4,096: 30.3, 26.3, 26.4 and 30.4 us; 4,096 of 14,336, rank 64: 180, 169, 155 and 246).  Otherwise there are as many as give every compute unit (of 256) a workgroup: the sums of every segment are written and read again, and with two workgroups a unit
// the way down gains less than the way up loses (4,096 rows of 14,336, rank 64, both ways: 84 us aimed at 500 workgroups, 79 at 250, 114 at 125; 531 rows of 4,096, rank 3 * 24: 24.7 at 500, 20.3 at 250).  Nor
// more than 8: 256 rows of 8,192, rank 64, take 29.2, 22.0, 20.8 and 20.5 us with any number, 16, 12 and 8 at most, 64 of 4,096, rank 32, with an adapter each 19.1, 19.0, 15.5 and 15.5.
int segment_of(int n_rows, int width, int ranks, bool low) {
    if (!low) return (width + EXACT_SEGMENTS * SEGMENT - 1) / (EXACT_SEGMENTS * SEGMENT) * SEGMENT;
    const long segments = min(max(250 / (usual_tiles(n_rows) * ((ranks + 63) / 64)), 1l), 8l);
    return (int)(((width + segments - 1) / segments + SEGMENT - 1) / SEGMENT * SEGMENT);
}

}  // namespace

// Floats of scratch that gi_adapters_add needs, 16-byte aligned: the sums of every segment of the width, the list of tiles and its length.
static long segments_for(int x_type, int w_type, int n_rows, int width, int ranks) {
    const int segment = segment_of(n_rows, width, ranks, x_type == GI_BF16 && w_type == GI_BF16);
    return (width + segment - 1) / segment;
}
static long sums_for(int x_type, int w_type, int n_rows, int width, int ranks) { return (segments_for(x_type, w_type, n_rows, width, ranks) * n_rows * ranks + 3) / 4 * 4; }
GI_API long gi_adapters_scratch_floats(int x_type, int w_type, int n_rows, int width, int rank, int n_slices) {
    return sums_for(x_type, w_type, n_rows, width, rank * n_slices) + 4 * (long)n_rows + 4;
}

GI_API int gi_adapters_add(const void* x, int x_type, long ldx, const void* a, const void* b, int w_type, const int* ids, const float* scales, const void* base, int base_type, long ldb,
                           void* out, int out_type, long ldo, float* scratch, int n_rows, int width, int columns, int rank, int n_slices, const int* slice_columns, int n_adapters,
                           hipStream_t stream) {
    GI_REQUIRE(n_rows > 0 && width > 0 && columns > 0 && rank > 0 && n_adapters > 0 && ldx >= width && ldb >= columns && ldo >= columns,
               "adapters_add: bad sizes (rows %d, width %d, columns %d, rank %d, adapters %d, strides %ld %ld %ld)", n_rows, width, columns, rank, n_adapters, ldx, ldb, ldo);
    GI_REQUIRE(rank <= MAX_RANK, "adapters_add: rank %d, at most %d is taken", rank, MAX_RANK);
    GI_REQUIRE(n_slices >= 1 && n_slices <= MAX_SLICES, "adapters_add: %d packed projections, 1 to %d are taken", n_slices, MAX_SLICES);
    GI_REQUIRE(ldb <= 1 << 23 && ldo <= 1 << 23, "adapters_add: rows of base and out %ld and %ld numbers apart, at most %d are taken", ldb, ldo, 1 << 23);
    GI_REQUIRE(n_rows <= 1 << 20 && width <= 1 << 24 && columns <= 1 << 22, "adapters_add: %d rows of %d numbers onto %d columns are too many for one launch", n_rows, width, columns);
    GI_REQUIRE(scratch != nullptr && aligned(scratch, 16), "adapters_add: scratch is missing");
    const bool low = x_type == GI_BF16 && w_type == GI_BF16;
    Tile* list = (Tile*)(scratch + sums_for(x_type, w_type, n_rows, width, rank * n_slices));
    Call c{x, ldx, a, b, ids, scales, Rows{base, out, ldb, ldo, base_type == GI_BF16, out_type == GI_BF16}, scratch, list, (int*)(list + n_rows), n_rows, width, columns, rank, n_adapters,
           segment_of(n_rows, width, rank * n_slices, low), (int)segments_for(x_type, w_type, n_rows, width, rank * n_slices), Slices{n_slices, {0}, {0}}, true, stream};
    for (int s = 0; s < n_slices; ++s) {
        GI_REQUIRE(slice_columns[s] > 0, "adapters_add: a packed projection of %d columns", slice_columns[s]);
        c.fours = c.fours && slice_columns[s] >= 4;
        c.slices.begin[s + 1] = c.slices.begin[s] + slice_columns[s];
    }
    GI_REQUIRE(c.slices.begin[n_slices] == columns, "adapters_add: the packed projections have %d columns, out has %d", c.slices.begin[n_slices], columns);
    if (low && few_rows(c)) {
        add_few(c);
        GI_CHECK_LAUNCH("adapters_add (few rows)");
        return 0;
    }
    const int went = low ? down<true, bf16_t, bf16_t>(c) : x_type == GI_BF16 ? down<false, bf16_t, float>(c) : w_type == GI_BF16 ? down<false, float, bf16_t>(c) : down<false, float, float>(c);
    if (went != 0) return went;
    GI_CHECK_LAUNCH("adapters_add (down)");
    const int came = low ? up<true, bf16_t>(c) : w_type == GI_BF16 ? up<false, bf16_t>(c) : up<false, float>(c);
    if (came != 0) return came;
    GI_CHECK_LAUNCH("adapters_add (up)");
    return 0;
}
