// Drafted tokens judged against the target's probabilities, with the uniform numbers given.
//
// Request r brings n drafts x_0 .. x_{n-1}, the target's rows of logits l_0 .. l_n (one further than its drafts), a temperature T, uniform
// numbers u_0 .. u_K and, where a model drafted, that model's rows m_0 .. m_{n-1}.  With p_j = softmax(l_j / T) and q_j = softmax(m_j / T), or
// all of q_j on x_j where there are no rows of the drafter's, draft x_j stays if those before it do and u_j q_j(x_j) < p_j(x_j).  Behind the a
// drafts that stay comes one token more: drawn from max(p_a - q_a, 0) where draft a fell, from p_n where none did.  So the tokens are
// distributed as if each had been drawn from the target's p (Leviathan, Kalman, Matias 2023; Chen et al. 2023).  A draw is by the inverse
// distribution in index order: the first token whose running sum is greater than u_K times the whole.
//
// A running sum over a hundred thousand tokens is compared with a number that falls anywhere between: in 32 bits one draw in some thousands
// comes out a token off.  So weights exp((l - max) / T) are made and added up in 64-bit arithmetic, which this chip does at the rate of 32; of
// a weight's bits 39 are good (2e-12 relative), a running sum keeps what its additions leave.
//
// Three launches.  All rows once, in runs of 4,096 logits: the runs' maxima and sums.  Then, per request and run, the verdict (every
// workgroup of a request comes to it by itself, from the runs' numbers) and, where a draft fell, the run's share of what is drawn from.
// Then a request's draw.  What bounds them: of many rows the logits' bytes and, as much, the weights' instructions (64 requests, 401 rows of
// 128,256 tokens, 206 MB: 49 + 20 + 8 us); of a few the waits that follow one another (one request with 4 drafts, 9 such rows: 4.5 + 7.0 +
// 6.1 us).  A last workgroup that draws by itself instead of a third launch has to see what the others wrote: with fences, which write caches
// back, one request took 29.7 us instead of 20.5, 64 took 121 instead of 81.  (Stores past the caches and a relaxed counter, as the matrix
// products' workgroups meet, were not tried here.)
#include "common.h"
#include "lanes.h"

namespace {

constexpr int CHUNK = 4096;                 // logits of a row that a workgroup takes
constexpr int MAX_CHUNKS = 1024;            // runs of a row: as many as the threads that draw (a vocabulary of 4 M tokens)
constexpr int MAX_DRAFTS = 64;
constexpr int MAX_ROWS = 2 * MAX_DRAFTS + 1;

constexpr double NOTHING_LEFT = 1e-12;      // of p beside q

enum { DONE = 0, PLAIN = 1, LESS_ROW = 2, LESS_TOKEN = 3 };       // what a request's last token is drawn from: nothing, p, max(p - q, 0), p without x

struct Verdict {                            // of one request
    int kept, kind, row, x;                 // drafts that stay; what is drawn from; row kept's place among the target's; the draft that fell
    float top_p, top_q;                     // the largest logit of the two rows
    double sum_p, sum_q;                    // and their sums of exp((l - max) / T)
};

struct Inputs {
    const float* logits;
    const float* drafter;                   // or null
    const int* drafts;
    const int* n_drafts;                    // or null: K everywhere
    const int* first_row;                   // or null: r (K + 1)
    const float* temperature;
    const float* uniform;
    long stride, drafter_request, drafter_row;
    int n_requests, K, vocab, n_rows, n_chunks;
};

__device__ __forceinline__ bool arg_max_asked(float t) { return !(t > 0.f); }

// How many drafts the request brings and where its rows begin; -1 if they do not lie among the rows given.
__device__ __forceinline__ int drafts_of(const Inputs& in, int r, long& first) {
    const int n = in.n_drafts == nullptr ? in.K : min(max(in.n_drafts[r], 0), in.K);
    first = in.first_row == nullptr ? (long)r * (in.K + 1) : (long)in.first_row[r];
    return first >= 0 && first + n < in.n_rows ? n : -1;
}

__device__ __forceinline__ float number(float v) { return v == v ? v : -INFINITY; }        // (what is no number is no token)

// Weights exp((l - top) / T) of a row whose largest logit is `top`: 1 for the largest, 0 for what is no token (-infinity, NaN) and below
// 2^-1020.  With m = (l - top) log2(e) / T, n the nearest integer (what is left in the low bits of a sum with 1.5 * 2^52) and f = m - n, 2^m
// is 2^n (1 + f q(f)), q the polynomial through (2^f - 1) / f at eight Chebyshev points of [-1/2, 1/2]: off by 2e-12 relative, less than a
// draw over a million tokens can notice.  No scaling by an instruction of its own: those, as conversions, run at a quarter of the rate, and
// instructions are what bounds a sum over many rows (a vector instruction in four fifths of the cycles).  A polynomial of nine points (4e-14)
// with a product of its own for m takes 55 us for 401 rows of 128,256 tokens that take 51 so.
__device__ __forceinline__ double horner(double f, double q, double c) {        // f q + c, the coefficient in scalar registers: as the accumulator it would be moved there for every step
    double out;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(out) : "v"(f), "v"(q), "s"(c));
    return out;
}
struct Scale {                              // of a request: its division is done while loads are awaited
    double per, least;                      // log2(e) / T, never 0; logits so far below the largest weigh less than 2^-1020
    __device__ explicit Scale(float t) : per(fmax(1.4426950408889634 / (double)t, 1e-300)), least(fmax(-707.0 * (double)t, -1e303)) {}
};
struct Weigher {
    double top, per, least;
    bool plain;                             // the largest is not infinite
    __device__ Weigher(float largest, const Scale& s) : top((double)largest), per(s.per), least(s.least), plain(largest < INFINITY) {}
    __device__ double power(double below) const {                               // of a logit so far below the largest, not less than `least`
        const double shifted = fma(below, per, 6755399441055744.0), f = fma(below, per, 6755399441055744.0 - shifted);
        double q = 1.325080551750225e-06;
        q = horner(f, q, 1.5303700711365693e-05);
        q = horner(f, q, 0.00015403475186530786);
        q = horner(f, q, 0.0013333478473685416);
        q = horner(f, q, 0.00961812913523614);
        q = horner(f, q, 0.055504109063258665);
        q = horner(f, q, 0.24022650695888503);
        q = horner(f, q, 0.6931471805568324);
        const long long w = __double_as_longlong(fma(f, q, 1.0)), n = __double_as_longlong(shifted);
        return __hiloint2double((int)(w >> 32) + ((int)n << 20), (int)w);
    }
    __device__ double fast(float l) const {
        const double below = (double)l - top;
        return below > least ? power(below) : 0.0;
    }
    __device__ double beside_1(float l) const { return power(fmax((double)l - top, least)); }      // to be added to 1 or more: 2^-1020 instead of 0, an instruction less
    __device__ double any(float l) const { return plain ? fast(l) : l == INFINITY ? 1.0 : 0.0; }
};

// A thread's logits of a run that NT threads share: `v[4 u + c]` is number begin + 4 (tid + NT u) + c where four may be loaded at once, number begin + tid + NT (4 u + c) otherwise; -infinity behind `end`.
template <int NT>
struct RunOf {
    static constexpr int PER = CHUNK / NT;
    int begin, end;
    bool fours;
    __device__ RunOf(const float* row, int run, int vocab) : begin(run * CHUNK), end(min(vocab, run * CHUNK + CHUNK)), fours((vocab & 3) == 0 && ((size_t)row & 15) == 0) {}
    __device__ int at(int j) const { return fours ? begin + 4 * ((int)threadIdx.x + NT * (j >> 2)) + (j & 3) : begin + (int)threadIdx.x + NT * j; }
    __device__ void load(const float* __restrict__ row, float (&v)[PER]) const {
        const float* from = row + begin;
        const int there = end - begin;
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));                       // (worked out anew for every row: kept over a loop, the sixteen places would cost registers, and waves)
        if (fours && there == CHUNK) {
#pragma unroll
            for (int u = 0; u < PER / 4; ++u) {
                const float4 w = reinterpret_cast<const float4*>(from + 4 * NT * u)[tid];
                v[4 * u] = w.x; v[4 * u + 1] = w.y; v[4 * u + 2] = w.z; v[4 * u + 3] = w.w;
            }
        } else if (fours) {
#pragma unroll
            for (int u = 0; u < PER / 4; ++u) {
                const int i = 4 * (tid + NT * u);
                const float4 w = *reinterpret_cast<const float4*>(from + min(i, there - 4));
                const bool in = i < there;
                v[4 * u] = in ? w.x : -INFINITY; v[4 * u + 1] = in ? w.y : -INFINITY; v[4 * u + 2] = in ? w.z : -INFINITY; v[4 * u + 3] = in ? w.w : -INFINITY;
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = tid + NT * j;
                const float w = from[min(i, there - 1)];
                v[j] = i < there ? w : -INFINITY;
            }
        }
    }
};

// Largest logit (with its lowest index) and sum of exp((l - that) / T) of every run: workgroup (run, request, group of rows).  Of the rows that the request has, the target's 0 .. n and the drafter's 0 .. n - 1 behind
// them, every gridDim.z-th is a workgroup's.  4.5 us for 9 rows of 128,256 tokens, 7.7 for 192 greedy ones of 32,003 (3.2 TB/s), 49 for 401 of 128,256 (4.2 TB/s; the loads alone take 40).
constexpr int PARTS_NT = 256;
__global__ __launch_bounds__(PARTS_NT) void parts_kernel(Inputs in, float* __restrict__ part_m, int* __restrict__ part_i, double* __restrict__ part_s) {
    constexpr int NT = PARTS_NT, PER = CHUNK / NT, WAVES = NT / 64;
    __shared__ float sv[2][WAVES];
    __shared__ int si[2][WAVES];
    __shared__ double red[2][WAVES];
    const int r = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    long first;
    const int n = drafts_of(in, r, first);
    if (n < 0) return;
    const float t = in.temperature[r];
    const bool greedy = arg_max_asked(t);
    const Scale scale(t);
    const int n_rows = n + 1 + (greedy || in.drafter == nullptr ? 0 : n);
    for (int i = blockIdx.z, turn = 0; i < n_rows; i += gridDim.z, turn ^= 1) {          // (two places for what meets in LDS in turn: one barrier a meeting)
        const float* row = i <= n ? in.logits + (first + i) * in.stride : in.drafter + r * in.drafter_request + (i - n - 1) * in.drafter_row;
        const RunOf<NT> run(row, blockIdx.x, in.vocab);
        float v[PER];
        run.load(row, v);
        float bv = -INFINITY;
#pragma unroll
        for (int j = 0; j < PER; ++j) bv = fmaxf(bv, v[j]);            // (NaN is passed over)
        bv = over_wave(bv, Larger());
        if (lane == 0) sv[turn][wave] = bv;
        barrier_lds();
        bv = sv[turn][0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) bv = fmaxf(bv, sv[turn][w]);
        const size_t at = ((size_t)r * (2 * in.K + 1) + (i <= n ? i : in.K + i - n)) * in.n_chunks + blockIdx.x;
        if (greedy) {                                                   // the lowest place of the largest (of -infinity where there are only such and NaN)
            int mine = PER;
#pragma unroll
            for (int j = PER - 1; j >= 0; --j) mine = number(v[j]) == bv ? j : mine;
            int bi = mine < PER && run.at(mine) < run.end ? run.at(mine) : 0x7fffffff;       // (a thread's numbers ascend)
            bi = over_wave(bi, Lesser());
            if (lane == 0) si[turn][wave] = bi;
            barrier_lds();
            if (tid == 0) {
#pragma unroll
                for (int w = 1; w < WAVES; ++w) bi = min(bi, si[turn][w]);
                part_m[at] = bv;
                part_i[at] = bi;
            }
            continue;
        }
        const Weigher weigh(bv, scale);
        double sum = 0.0;
        if (weigh.plain) {
#pragma unroll
            for (int j = 0; j < PER; ++j) sum += weigh.beside_1(v[j]);
        } else {
            for (int k = run.begin + tid; k < run.end; k += NT) sum += weigh.any(row[k]);
        }
        sum = over_wave(sum, Add());
        if (lane == 0) red[turn][wave] = sum;
        barrier_lds();
        if (tid == 0) {
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum += red[turn][w];
            part_m[at] = bv;
            part_s[at] = bv > -INFINITY ? sum : 0.0;
        }
    }
}

// The weight token i is drawn with, up to a factor that all of a request's tokens share.
struct Drawn {
    Weigher p, q;
    double over_p, over_q;
    int kind, x;
    __device__ Drawn(const Verdict& v, const Scale& s) : p(v.top_p, s), q(v.top_q, s), over_p(v.sum_p > 0.0 ? 1.0 / v.sum_p : 0.0), over_q(v.sum_q > 0.0 ? 1.0 / v.sum_q : 0.0), kind(v.kind), x(v.x) {}
    __device__ bool plain() const { return p.plain && (kind != LESS_ROW || q.plain); }
    __device__ double weight(float target, float drafter, bool left_out) const {       // of plain rows
        const double w = p.fast(target);
        return kind == LESS_ROW ? fmax(w * over_p - q.fast(drafter) * over_q, 0.0) : left_out ? 0.0 : w;
    }
    __device__ double any(float target, float drafter, int i) const {
        const double w = p.any(target);
        return kind == LESS_ROW ? fmax(w * over_p - q.any(drafter) * over_q, 0.0) : kind == LESS_TOKEN && i == x ? 0.0 : w;
    }
};

// Which drafts stay, and the sums over runs of what is drawn from, where the parts do not hold them already: every run of a request whose
// drafter's row is taken off, and the run that a draft is left out of.  Workgroup (run, request); run 0's writes what the request has so far.
// 7.0 us for one request with 4 drafts, 20 for 64 with up to 7, which read two rows of 128,256 again each (58 MB), once the verdict says
// which: its waits (6 us) have nothing beside them, and of the 2,048 workgroups of 256 threads 1,280 fit at once (81 registers, five a compute
// unit), so the rest come to their verdict, and wait, after these.
template <int NT>
__global__ __launch_bounds__(NT) void judge_kernel(Inputs in, const float* __restrict__ part_m, const int* __restrict__ part_i, const double* __restrict__ part_s, Verdict* __restrict__ verdicts,
                                                   double* __restrict__ rest, int* __restrict__ tokens, int* __restrict__ counts) {
    __shared__ float top[MAX_ROWS];
    __shared__ int arg[MAX_ROWS];
    __shared__ double whole[MAX_ROWS];
    __shared__ int drafted[MAX_DRAFTS];
    __shared__ int stays;                                   // drafts before the first that falls
    constexpr int PER = CHUNK / NT, WAVES = NT / 64;
    __shared__ double red[WAVES];
    const int r = blockIdx.y, tid = threadIdx.x, K = in.K, member = tid & 15;
    int x = -1;                                             // this thread's draft, its logits, its number
    float target_x = -INFINITY, drafter_x = -INFINITY, u = 0.f;
    if (tid < K) x = in.drafts[(size_t)r * K + tid];        // (asked for before it is known whether the request brings it: the waits for both are one)
    long first;
    const int n = drafts_of(in, r, first);
    const float t = in.temperature[r];
    const bool greedy = arg_max_asked(t);
    if (greedy && blockIdx.x != 0) return;
    if (tid < K) drafted[tid] = x;
    if (tid < n) {
        if (x < 0 || x >= in.vocab) x = -1;
        if (x >= 0 && !greedy) {
            target_x = in.logits[(first + tid) * in.stride + x];
            if (in.drafter != nullptr) drafter_x = in.drafter[r * in.drafter_request + tid * in.drafter_row + x];
            u = in.uniform[(size_t)r * (K + 1) + tid];
        }
    }
    const Scale scale(t);
    for (int z = tid >> 4; z < 2 * K + 1; z += NT / 16) {   // sixteen lanes a row
        if (n < 0 || (z <= K ? z > n : (in.drafter == nullptr || z - K - 1 >= n || greedy))) continue;
        const size_t at = ((size_t)r * (2 * K + 1) + z) * in.n_chunks;
        float largest = -INFINITY;
        int place = 0x7fffffff;
        double sum = 0.0;
        for (int c0 = 0; c0 < in.n_chunks; c0 += 64) {      // (once, for up to 262,144 tokens)
            float m[4];
            int i[4] = {};
            double s[4] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = c0 + member + 16 * j;
                m[j] = -INFINITY;
                if (c < in.n_chunks) {
                    m[j] = part_m[at + c];
                    if (greedy) i[j] = part_i[at + c];
                    else s[j] = part_s[at + c];
                }
            }
            const float bv = over_16(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), Larger());
            const float now = fmaxf(largest, bv);
            if (greedy) {
                if (now > largest) place = 0x7fffffff;      // (a place of an earlier run that holds as much is lower)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + member + 16 * j < in.n_chunks && m[j] == now) place = min(place, i[j]);
            } else {
                const Weigher weigh(now, scale);
                double more = 0.0;
#pragma unroll
                for (int j = 0; j < 4; ++j) more += s[j] * weigh.any(m[j]);
                sum = sum * weigh.any(largest) + over_16(more, Add());
            }
            largest = now;
        }
        place = over_16(place, Lesser());
        if (member == 0) { top[z] = largest; arg[z] = place; whole[z] = sum; }
    }
    __syncthreads();
    static_assert(MAX_DRAFTS == 64, "one wave judges the drafts");
    if (tid < MAX_DRAFTS) {
        bool stay = false;
        if (tid < n && x >= 0) {
            if (greedy) {
                stay = x == arg[tid];
            } else {
                // u q / whole_q < p / whole_p; a row without a token has no probabilities (its sum and all its weights are 0)
                const double p = whole[tid] > 0.0 ? Weigher(top[tid], scale).any(target_x) / whole[tid] : 0.0;
                double q = 1.0;
                if (in.drafter != nullptr) q = whole[K + 1 + tid] > 0.0 ? Weigher(top[K + 1 + tid], scale).any(drafter_x) / whole[K + 1 + tid] : 0.0;
                stay = (double)u * q < p;
            }
        }
        const unsigned long long fell = __ballot(!stay);    // (the places behind the request's drafts among them)
        if (tid == 0) stays = fell != 0 ? __ffsll((long long)fell) - 1 : MAX_DRAFTS;
    }
    __syncthreads();
    const int kept = min(max(n, 0), stays);
    Verdict v{kept, DONE, kept, -1, 0.f, 0.f, 0.0, 0.0};
    if (n >= 0 && !greedy) {
        v.top_p = top[kept];
        v.sum_p = whole[kept];
        v.kind = PLAIN;
        if (kept < n) {
            v.x = drafted[kept];
            if (in.drafter != nullptr) {
                v.kind = LESS_ROW;
                v.top_q = top[K + 1 + kept];
                v.sum_q = whole[K + 1 + kept];
            } else if (v.x >= 0 && v.x < in.vocab) {
                v.kind = LESS_TOKEN;
            }
        }
    }
    if (blockIdx.x == 0) {
        if (tid <= K) tokens[(size_t)r * (K + 1) + tid] = tid < kept ? drafted[tid] : greedy && n >= 0 && tid == kept ? arg[kept] : -1;
        if (tid == 0) {
            counts[r] = n < 0 ? 0 : kept + 1;
            verdicts[r] = v;
        }
    }
    if (v.kind != LESS_ROW && !(v.kind == LESS_TOKEN && v.x / CHUNK == (int)blockIdx.x)) return;
    const float* row = in.logits + (first + v.row) * in.stride;
    const float* drafter = v.kind == LESS_ROW ? in.drafter + r * in.drafter_request + v.row * in.drafter_row : row;
    const RunOf<NT> run(row, blockIdx.x, in.vocab), other(drafter, blockIdx.x, in.vocab);
    float a[PER], b[PER];
    double sum = 0.0;
    const Drawn drawn(v, scale);
    if (run.fours == other.fours && drawn.plain()) {
        run.load(row, a);
        if (v.kind == LESS_ROW) other.load(drafter, b);
        int left_out = -1;                                  // which of this thread's numbers x is
        if (v.kind == LESS_TOKEN)
            for (int j = 0; j < PER; ++j) left_out = run.at(j) == v.x ? j : left_out;
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += drawn.weight(a[j], b[j], j == left_out);       // (nothing behind the end)
    } else {
        for (int i = run.begin + tid; i < run.end; i += NT) sum += drawn.any(row[i], drafter[i], i);
    }
    sum = over_wave(sum, Add());
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sum += red[w];
        rest[(size_t)r * in.n_chunks + blockIdx.x] = sum;
    }
}

// The draw: one workgroup a request.  The run is found among the runs' sums (by a prefix sum over a wave's lanes, which share the runs out, and a walk over one lane's), then the token in the run: a
// thread owns four consecutive tokens, a prefix sum over the threads finds the thread, which walks its tokens.  6 us for one request, 8 for 64, all of it waits; with 256 threads, sixteen tokens each, 5 us more.
constexpr int PICK_NT = 1024, PICK_WAVES = PICK_NT / 64, PICK_PER = CHUNK / PICK_NT;
__global__ __launch_bounds__(PICK_NT) void pick_kernel(Inputs in, const Verdict* __restrict__ verdicts, const float* __restrict__ part_m, const double* __restrict__ part_s,
                                                       const double* __restrict__ rest, int* __restrict__ tokens) {
    __shared__ double sums[MAX_CHUNKS];
    __shared__ double wave_total[PICK_WAVES];
    __shared__ double target, before_run;
    __shared__ int the_run, winner, last_one;
    const int r = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    // (asked for beside the verdict; a run whose share the verdict did not need has none there, and it is not looked at)
    const double left = tid < in.n_chunks ? rest[(size_t)r * in.n_chunks + tid] : 0.0;
    const float u = in.uniform[(size_t)r * (in.K + 1) + in.K];
    Verdict v = verdicts[r];
    if (v.kind == DONE) return;
    long first;
    drafts_of(in, r, first);
    const Scale scale(in.temperature[r]);
    const float* row = in.logits + (first + v.row) * in.stride;
    const float* drafter = v.kind == LESS_ROW ? in.drafter + r * in.drafter_request + v.row * in.drafter_row : row;
    const size_t parts = ((size_t)r * (2 * in.K + 1) + v.row) * in.n_chunks;
    for (int attempt = 0; attempt < 2; ++attempt) {
        if (tid < in.n_chunks) {                           // (MAX_CHUNKS threads)
            const bool own = v.kind == LESS_ROW || (v.kind == LESS_TOKEN && v.x / CHUNK == tid);
            sums[tid] = own ? left : part_s[parts + tid] * Weigher(v.top_p, scale).any(part_m[parts + tid]);
        }
        __syncthreads();
        if (wave == 0) {
            const int each = (in.n_chunks + 63) / 64, from = lane * each, to = min(in.n_chunks, from + each);
            double mine = 0.0;
            for (int c = from; c < to; ++c) mine += sums[c];
            const double upto = sum_up_to(mine), below = lane_before(upto), total = of_lane(upto, 63);       // (the lane before's, 0 for the first)
            const double goal = (double)u * total;
            const unsigned long long beyond = __ballot(goal < upto && mine > 0.0), some = __ballot(mine > 0.0);
            // the first lane whose runs end beyond the goal; by rounding, or for u = 1, the last that weighs anything
            // (what rounding leaves of p beside an equal q is nothing: as much as that is a chance that no draft has to fall by)
            const int owner = v.kind == LESS_ROW && total <= NOTHING_LEFT ? -1 : beyond != 0 ? __ffsll((long long)beyond) - 1 : some != 0 ? 63 - __clzll((long long)some) : -1;
            if (lane == owner) {
                double walked = below, before_last = walked;
                int run = -1, last = -1;
                for (int c = from; c < to && run < 0; ++c) {
                    if (!(sums[c] > 0.0)) continue;        // (the goal may lie a rounding below `below`, where no lane before holds it: a run of no weight is none to draw from)
                    last = c;
                    before_last = walked;
                    if (goal < walked + sums[c]) run = c;
                    walked += sums[c];
                }
                the_run = run >= 0 ? run : last;
                before_run = before_last;                  // (the last seen, be it the one that holds the goal or not)
                target = goal;
            }
            if (owner < 0 && lane == 0) the_run = -1;
        }
        if (tid == 0) winner = 0x7fffffff;
        if (tid == 64) last_one = -1;
        __syncthreads();
        if (the_run >= 0 || v.kind == PLAIN) break;
        v.kind = PLAIN;                                    // nothing is left of p beside q: p itself
        __syncthreads();
    }
    const int run = the_run;
    if (run < 0) {                                         // a row without a token
        if (tid == 0) tokens[(size_t)r * (in.K + 1) + v.kept] = 0;
        return;
    }
    const int begin = run * CHUNK, end = min(in.vocab, begin + CHUNK), lo = begin + tid * PICK_PER;
    const Drawn drawn(v, scale);
    double w[PICK_PER], mine = 0.0;
    int last = -1;                                         // the last token that weighs anything
#pragma unroll
    for (int j = 0; j < PICK_PER; ++j) {
        const int i = min(lo + j, end - 1);
        w[j] = drawn.any(row[i], drafter[i], i);
        if (lo + j >= end) w[j] = 0.0;
        mine += w[j];
        if (w[j] > 0.0) last = lo + j;
    }
    const double upto = sum_up_to(mine), below = lane_before(upto);
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    static_assert(PICK_WAVES == 16, "a wave's sixteen lanes add up the waves' sums");
    const double totals = sum_up_to(lane < PICK_WAVES ? wave_total[lane] : 0.0);
    double walk = before_run + (wave > 0 ? of_lane(totals, wave - 1) : 0.0) + below;
    int hit = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < PICK_PER; ++j) {
        walk += w[j];
        if (hit == 0x7fffffff && w[j] > 0.0 && walk > target) hit = lo + j;
    }
    // the lowest token that reaches beyond the goal: of a wave, then of all
    const unsigned long long hits = __ballot(hit != 0x7fffffff), some = __ballot(last >= 0);
    if (hits != 0 && lane == __ffsll((long long)hits) - 1) atomicMin(&winner, hit);
    if (some != 0 && lane == 63 - __clzll((long long)some)) atomicMax(&last_one, last);
    __syncthreads();
    if (tid == 0) tokens[(size_t)r * (in.K + 1) + v.kept] = max(winner != 0x7fffffff ? winner : last_one, 0);
}

}  // namespace

// Bytes of scratch that gi_verify_drafts needs.
GI_API long gi_verify_drafts_scratch_bytes(int n_requests, int K, int vocab) {
    const long runs = (vocab + CHUNK - 1) / CHUNK, rows = (long)n_requests * (2 * K + 1);
    return rows * runs * 16 + (long)n_requests * (runs * 8 + (long)sizeof(Verdict));
}

// tokens [n_requests, K + 1]: the drafts that stay, the token behind them, -1; counts: how many tokens that is, 0 (and -1 throughout) for a request whose
// rows do not lie among the n_rows given.
GI_API int gi_verify_drafts(const float* logits, int n_rows, long stride, const float* drafter, long drafter_request, long drafter_row, const int* drafts, const int* n_drafts,
                            const int* first_row, const float* temperature, const float* uniform, int* tokens, int* counts, void* scratch, int n_requests, int K, int vocab,
                            hipStream_t stream) {
    GI_REQUIRE(n_requests > 0 && n_requests <= 65535 && K >= 0 && K <= MAX_DRAFTS && vocab > 0 && n_rows > 0 && stride >= vocab,
               "verify_drafts: bad sizes (requests %d, drafts %d of at most %d, vocab %d, rows %d, stride %ld)", n_requests, K, MAX_DRAFTS, vocab, n_rows, stride);
    GI_REQUIRE(scratch != nullptr && (size_t)scratch % 8 == 0, "verify_drafts: scratch is missing");
    const int n_chunks = (vocab + CHUNK - 1) / CHUNK;
    GI_REQUIRE(n_chunks <= MAX_CHUNKS, "verify_drafts: a vocabulary of %d tokens is more than %d runs of %d", vocab, MAX_CHUNKS, CHUNK);
    const Inputs in{logits, drafter, drafts, n_drafts, first_row, temperature, uniform, stride, drafter_request, drafter_row, n_requests, K, vocab, n_rows, n_chunks};
    const size_t rows = (size_t)n_requests * (2 * K + 1);
    double* part_s = (double*)scratch;
    double* rest = part_s + rows * n_chunks;
    Verdict* verdicts = (Verdict*)(rest + (size_t)n_requests * n_chunks);
    float* part_m = (float*)(verdicts + n_requests);
    int* part_i = (int*)(part_m + rows * n_chunks);
    const int most = drafter != nullptr ? 2 * K + 1 : K + 1;
    // A workgroup adds up several of a request's rows where there are more than 32 workgroups a compute unit without: their start costs as much as a short run.  Aimed at 8, 16, 32 and 200 of them, 64 requests with up to
    // 15 rows of 128,256 tokens took 99, 89, 83 and 95 us in all; a few requests have a workgroup for every row and run either way.
    const int groups = (int)min((long)most, max(1l, 32 * (long)gi_compute_units() / ((long)n_chunks * n_requests)));
    parts_kernel<<<dim3(n_chunks, n_requests, groups), PARTS_NT, 0, stream>>>(in, part_m, part_i, part_s);
    GI_CHECK_LAUNCH("verify_drafts (parts)");
    // 1,024 threads where there is a compute unit for every workgroup, 256 otherwise: 1 and 8 requests with 4 drafts of a model, 128,256 tokens, take 16.4 and 22.1 us in all instead of 17.6 and 23.6; 16 and 64 would take
    // 33.5 and 105 instead of 31.3 and 84.  (The sums of all rows take longer with more threads even for one request.)
    const dim3 runs(n_chunks, n_requests);
    if ((long)n_chunks * n_requests <= gi_compute_units()) judge_kernel<1024><<<runs, 1024, 0, stream>>>(in, part_m, part_i, part_s, verdicts, rest, tokens, counts);
    else judge_kernel<256><<<runs, 256, 0, stream>>>(in, part_m, part_i, part_s, verdicts, rest, tokens, counts);
    GI_CHECK_LAUNCH("verify_drafts (judge)");
    pick_kernel<<<n_requests, PICK_NT, 0, stream>>>(in, verdicts, part_m, part_s, rest, tokens);
    GI_CHECK_LAUNCH("verify_drafts (pick)");
    return 0;
}
