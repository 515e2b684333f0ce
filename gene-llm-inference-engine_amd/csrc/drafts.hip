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
// comes out a token off.  So weights exp((l - max) / T) and all sums are held in 64 bits, which this chip computes at the rate of 32.
#include "common.h"

namespace {

constexpr int CHUNK = 4096;                 // logits of a row that a workgroup takes
constexpr int NT = 256;
constexpr int PER = CHUNK / NT;             // ... and a thread: in the pick as many consecutive ones
constexpr int MAX_CHUNKS = 1024;            // runs of a row that the pick holds in LDS (a vocabulary of 4 M tokens)
constexpr int MAX_DRAFTS = 64;
constexpr int MAX_ROWS = 2 * MAX_DRAFTS + 1;

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

// exp((l - top) / T): 1 for the largest, also where that is infinite; 0 for -infinity.
__device__ __forceinline__ double weight(float l, float top, double inv_t) {
    if (l == top) return top == -INFINITY ? 0.0 : 1.0;
    const double d = (double)l - (double)top;
    return d > -1e300 ? exp(d * inv_t) : 0.0;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

__device__ __forceinline__ void better(float& bv, int& bi, float ov, int oi) {
    if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
}

// Largest logit (with its lowest index) and sum of exp((l - that) / T) of every run of CHUNK logits: workgroup (run, request, row), rows 0 .. K
// the target's, K + 1 .. 2 K the drafter's.
__global__ __launch_bounds__(NT) void parts_kernel(Inputs in, float* __restrict__ part_m, int* __restrict__ part_i, double* __restrict__ part_s) {
    __shared__ float sv[4];
    __shared__ int si[4];
    __shared__ double red[4];
    const int r = blockIdx.y, z = blockIdx.z, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    long first;
    const int n = drafts_of(in, r, first);
    const float t = in.temperature[r];
    const bool greedy = arg_max_asked(t);
    if (n < 0 || (z <= in.K ? z > n : (z - in.K - 1 >= n || greedy))) return;
    const float* row = z <= in.K ? in.logits + (first + z) * in.stride : in.drafter + r * in.drafter_request + (z - in.K - 1) * in.drafter_row;
    const int begin = blockIdx.x * CHUNK, end = min(in.vocab, begin + CHUNK);
    float v[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) v[u] = row[min(begin + tid + NT * u, end - 1)];
    float bv = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int i = begin + tid + NT * u;
        v[u] = i < end ? number(v[u]) : -INFINITY;
        if (i < end && (v[u] > bv || bi == 0x7fffffff)) { bv = v[u]; bi = i; }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) better(bv, bi, __shfl_xor(bv, off, 64), __shfl_xor(bi, off, 64));
    if (lane == 0) { sv[wave] = bv; si[wave] = bi; }
    __syncthreads();
    bv = sv[0]; bi = si[0];
    for (int w = 1; w < 4; ++w) better(bv, bi, sv[w], si[w]);
    double sum = 0.0;
    if (!greedy) {
        const double inv_t = 1.0 / (double)t;
#pragma unroll
        for (int u = 0; u < PER; ++u) sum += weight(v[u], bv, inv_t);
        sum = wave_sum_f64(sum);
        if (lane == 0) red[wave] = sum;
        __syncthreads();
    }
    if (tid == 0) {
        const size_t at = ((size_t)r * (2 * in.K + 1) + z) * in.n_chunks + blockIdx.x;
        part_m[at] = bv;
        part_i[at] = bi;
        part_s[at] = greedy ? 0.0 : ((red[0] + red[1]) + red[2]) + red[3];
    }
}

// Which drafts stay: one workgroup a request, a wave a row.
__global__ __launch_bounds__(NT) void judge_kernel(Inputs in, const float* __restrict__ part_m, const int* __restrict__ part_i,
                                                   const double* __restrict__ part_s, Verdict* __restrict__ verdicts, int* __restrict__ tokens,
                                                   int* __restrict__ counts) {
    __shared__ float top[MAX_ROWS];
    __shared__ int arg[MAX_ROWS];
    __shared__ double whole[MAX_ROWS];
    __shared__ int stays[MAX_DRAFTS];
    const int r = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, K = in.K;
    long first;
    const int n = drafts_of(in, r, first);
    const float t = in.temperature[r];
    const bool greedy = arg_max_asked(t);
    const double inv_t = greedy ? 0.0 : 1.0 / (double)t;
    for (int z = wave; z < 2 * K + 1; z += 4) {
        if (n < 0 || (z <= K ? z > n : (in.drafter == nullptr || z - K - 1 >= n || greedy))) continue;
        const size_t at = ((size_t)r * (2 * K + 1) + z) * in.n_chunks;
        float bv = -INFINITY;
        int bi = 0x7fffffff;
        for (int c = lane; c < in.n_chunks; c += 64) better(bv, bi, part_m[at + c], part_i[at + c]);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) better(bv, bi, __shfl_xor(bv, off, 64), __shfl_xor(bi, off, 64));
        double sum = 0.0;
        if (!greedy)
            for (int c = lane; c < in.n_chunks; c += 64) sum += part_s[at + c] * weight(part_m[at + c], bv, inv_t);
        sum = wave_sum_f64(sum);
        if (lane == 0) { top[z] = bv; arg[z] = bi; whole[z] = sum; }
    }
    __syncthreads();
    if (tid < MAX_DRAFTS) {
        bool stay = false;
        if (tid < n) {
            const int x = in.drafts[(size_t)r * K + tid];
            if (x >= 0 && x < in.vocab) {
                if (greedy) {
                    stay = x == arg[tid];
                } else {
                    const double p = weight(number(in.logits[(first + tid) * in.stride + x]), top[tid], inv_t);
                    double q = 1.0, whole_q = 1.0;
                    if (in.drafter != nullptr) {
                        q = weight(number(in.drafter[r * in.drafter_request + tid * in.drafter_row + x]), top[K + 1 + tid], inv_t);
                        whole_q = whole[K + 1 + tid];
                    }
                    // u q / whole_q < p / whole_p; a row without a token has no probabilities (its sum and all its weights are 0)
                    const double u = (double)in.uniform[(size_t)r * (K + 1) + tid];
                    stay = u * (whole_q > 0.0 ? q / whole_q : 0.0) < (whole[tid] > 0.0 ? p / whole[tid] : 0.0);
                }
            }
        }
        stays[tid] = stay;
    }
    __syncthreads();
    int kept = 0;
    while (kept < n && stays[kept]) ++kept;
    if (tid <= K) {
        const int x = tid < kept ? in.drafts[(size_t)r * K + tid] : -1;
        tokens[(size_t)r * (K + 1) + tid] = greedy && n >= 0 && tid == kept ? arg[kept] : x;
    }
    if (tid == 0) {
        counts[r] = n < 0 ? 0 : kept + 1;
        Verdict v{kept, DONE, kept, -1, 0.f, 0.f, 0.0, 0.0};
        if (n >= 0 && !greedy) {
            v.top_p = top[kept];
            v.sum_p = whole[kept];
            v.kind = PLAIN;
            if (kept < n) {
                v.x = in.drafts[(size_t)r * K + kept];
                if (in.drafter != nullptr) {
                    v.kind = LESS_ROW;
                    v.top_q = top[K + 1 + kept];
                    v.sum_q = whole[K + 1 + kept];
                } else if (v.x >= 0 && v.x < in.vocab) {
                    v.kind = LESS_TOKEN;
                }
            }
        }
        verdicts[r] = v;
    }
}

// The weight token i is drawn with, up to a factor that all of a request's tokens share.
__device__ __forceinline__ double drawn_weight(const Verdict& v, const float* __restrict__ row, const float* __restrict__ drafter, int i, double inv_t) {
    const double p = weight(number(row[i]), v.top_p, inv_t);
    if (v.kind == LESS_ROW) {
        const double q = v.sum_q > 0.0 ? weight(number(drafter[i]), v.top_q, inv_t) / v.sum_q : 0.0;
        return fmax((v.sum_p > 0.0 ? p / v.sum_p : 0.0) - q, 0.0);
    }
    return v.kind == LESS_TOKEN && i == v.x ? 0.0 : p;
}

// Sums of those weights over runs, where the parts do not hold them already: every run of a request whose drafter's row is taken off, and the run
// that a draft is left out of.
__global__ __launch_bounds__(NT) void rest_kernel(Inputs in, const Verdict* __restrict__ verdicts, double* __restrict__ rest) {
    __shared__ double red[4];
    const int r = blockIdx.y, tid = threadIdx.x;
    const Verdict v = verdicts[r];
    if (v.kind != LESS_ROW && !(v.kind == LESS_TOKEN && v.x / CHUNK == (int)blockIdx.x)) return;
    long first;
    drafts_of(in, r, first);
    const float* row = in.logits + (first + v.row) * in.stride;
    const float* drafter = in.drafter == nullptr ? nullptr : in.drafter + r * in.drafter_request + v.row * in.drafter_row;
    const double inv_t = 1.0 / (double)in.temperature[r];
    const int begin = blockIdx.x * CHUNK, end = min(in.vocab, begin + CHUNK);
    double sum = 0.0;
    for (int i = begin + tid; i < end; i += NT) sum += drawn_weight(v, row, drafter, i, inv_t);
    sum = wave_sum_f64(sum);
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) rest[(size_t)r * in.n_chunks + blockIdx.x] = ((red[0] + red[1]) + red[2]) + red[3];
}

// The draw: one workgroup a request.  The run is found among the runs' sums, then the token in the run: a thread owns PER consecutive tokens,
// a prefix sum over the threads finds the thread, which walks its tokens.
__global__ __launch_bounds__(NT) void pick_kernel(Inputs in, const Verdict* __restrict__ verdicts, const float* __restrict__ part_m, const double* __restrict__ part_s,
                                                  const double* __restrict__ rest, int* __restrict__ tokens) {
    __shared__ double sums[MAX_CHUNKS];
    __shared__ double wave_total[4];
    __shared__ double target, before_run;
    __shared__ int the_run, winner, last_of_wave[4];
    const int r = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    Verdict v = verdicts[r];
    if (v.kind == DONE) return;
    long first;
    drafts_of(in, r, first);
    const float* row = in.logits + (first + v.row) * in.stride;
    const float* drafter = in.drafter == nullptr ? nullptr : in.drafter + r * in.drafter_request + v.row * in.drafter_row;
    const double inv_t = 1.0 / (double)in.temperature[r];
    const size_t parts = ((size_t)r * (2 * in.K + 1) + v.row) * in.n_chunks;
    for (int attempt = 0; attempt < 2; ++attempt) {
        for (int c = tid; c < in.n_chunks; c += NT) {
            const bool own = v.kind == LESS_ROW || (v.kind == LESS_TOKEN && v.x / CHUNK == c);
            sums[c] = own ? rest[(size_t)r * in.n_chunks + c] : part_s[parts + c] * weight(part_m[parts + c], v.top_p, inv_t);
        }
        __syncthreads();
        if (tid == 0) {
            double total = 0.0;
            for (int c = 0; c < in.n_chunks; ++c) total += sums[c];
            const double goal = (double)in.uniform[(size_t)r * (in.K + 1) + in.K] * total;
            double before = 0.0, before_last = 0.0;
            int run = -1, last = -1;
            for (int c = 0; c < in.n_chunks && run < 0; ++c) {
                if (goal < before + sums[c]) run = c;
                else {
                    if (sums[c] > 0.0) { last = c; before_last = before; }
                    before += sums[c];
                }
            }
            the_run = run >= 0 ? run : last;               // (rounding, or u = 1: the last run that weighs anything; -1: none does)
            before_run = run >= 0 ? before : before_last;
            target = goal;
        }
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
    const int begin = run * CHUNK, end = min(in.vocab, begin + CHUNK), lo = begin + tid * PER;
    double w[PER], mine = 0.0;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        w[u] = lo + u < end ? drawn_weight(v, row, drafter, lo + u, inv_t) : 0.0;
        mine += w[u];
    }
    double upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double below = __shfl_up(upto, off, 64);
        if (lane >= off) upto += below;
    }
    if (lane == 63) wave_total[wave] = upto;
    if (tid == 0) winner = 0x7fffffff;
    int last = -1;                                         // the last token that weighs anything
#pragma unroll
    for (int u = 0; u < PER; ++u)
        if (w[u] > 0.0) last = lo + u;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) last = max(last, __shfl_xor(last, off, 64));
    if (lane == 0) last_of_wave[wave] = last;
    const double below_lane = __shfl_up(upto, 1, 64);
    __syncthreads();
    double walk = before_run;
    for (int k = 0; k < wave; ++k) walk += wave_total[k];
    if (lane) walk += below_lane;
    int hit = 0x7fffffff;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        walk += w[u];
        if (hit == 0x7fffffff && w[u] > 0.0 && walk > target) hit = lo + u;
    }
    if (hit != 0x7fffffff) atomicMin(&winner, hit);
    __syncthreads();
    if (tid == 0) {
        int pick = winner;
        if (pick == 0x7fffffff) pick = max(max(last_of_wave[0], last_of_wave[1]), max(last_of_wave[2], last_of_wave[3]));
        tokens[(size_t)r * (in.K + 1) + v.kept] = max(pick, 0);
    }
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
    parts_kernel<<<dim3(n_chunks, n_requests, drafter != nullptr ? 2 * K + 1 : K + 1), NT, 0, stream>>>(in, part_m, part_i, part_s);
    GI_CHECK_LAUNCH("verify_drafts (parts)");
    judge_kernel<<<n_requests, NT, 0, stream>>>(in, part_m, part_i, part_s, verdicts, tokens, counts);
    GI_CHECK_LAUNCH("verify_drafts (judge)");
    rest_kernel<<<dim3(n_chunks, n_requests), NT, 0, stream>>>(in, verdicts, rest);
    GI_CHECK_LAUNCH("verify_drafts (rest)");
    pick_kernel<<<n_requests, NT, 0, stream>>>(in, verdicts, part_m, part_s, rest, tokens);
    GI_CHECK_LAUNCH("verify_drafts (pick)");
    return 0;
}
