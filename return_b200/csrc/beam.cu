// Beam search's selection: of all continuations of a request's beams, beams x vocabulary, the `keep` with the highest total
//   total(b, v) = score[b] + logits[b, v] - log(sum_u exp(logits[b, u])),
// falling, ties to the lowest (b, v).  A total that is no number (a row with a NaN or +inf, a row of -inf alone) counts as -inf, and so
// do all of a row whose score is not finite.
//
// The logits are read once.  beam_chunk_kernel: a CTA holds a chunk of a row in registers, works out its maximum and sum of
// exponentials, and writes its `keep` best: the order within a row is that of the logits.  Each warp's r-th highest lane maximum,
// r = keep / warps rounded up, is passed by r values of that warp, so the lowest of these over the warps is passed by `keep`
// values of the chunk and by few more; those are collected in shared memory, ranked by counting, and written in order.  Where
// more than COLLECT values pass (equal logits), the best are taken one by one.
// beam_merge_kernel: a CTA a request puts the rows' sums together and takes the best of all chunks' lists the same way.  Totals are
// compared in 64 bits, so that logits which differ keep their order however far down the scores are; one rounding at the store.
#include "common.cuh"

#define BEAM_MAX_KEEP 128
#define BEAM_MAX_BEAMS 64

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int COLLECT = 512;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
template <typename T> __device__ __forceinline__ T lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -INFINITY; }
template <> __device__ __forceinline__ double lowest<double>() { return -(double)INFINITY; }

template <typename T> __device__ __forceinline__ T warp_top(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const T w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}
// The r-th highest of a warp's values, equal ones counted one by one; -inf where there are fewer.
template <typename T> __device__ __forceinline__ T warp_rth(T v, int r, int lane) {
    T top = lowest<T>();
    bool out = false;
    for (int i = 0; i < r; ++i) {
        top = warp_top(out ? lowest<T>() : v);
        const unsigned who = __ballot_sync(0xffffffffu, !out && v == top);
        if (who == 0u) return lowest<T>();                    // fewer than r lanes
        if (lane == __ffs(who) - 1) out = true;
    }
    return top;
}
// Whether (a, i) comes before (b, j).
template <typename T> __device__ __forceinline__ bool before(T a, int i, T b, int j) { return a > b || (a == b && i < j); }

// Ranks what was collected and hands the first `keep` to put(rank, value, index).
template <typename T, typename Put>
__device__ __forceinline__ void rank_collected(const T* value, const int* index, int n, int keep, int tid, Put put) {
    for (int i = tid; i < n; i += THREADS) {
        const T v = value[i];
        const int at = index[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += before(value[j], index[j], v, at) ? 1 : 0;
        if (rank < keep) put(rank, v, at);
    }
}
// The best of every thread's (value, index), for all threads.  `sv`, `si`: WARPS + 1 entries.
template <typename T>
__device__ __forceinline__ void block_best(T& v, int& at, T* sv, int* si, int tid) {
    auto better = [&](T w, int k) { if (before(w, k, v, at)) { v = w; at = k; } };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const T w = __shfl_xor_sync(0xffffffffu, v, o);
        const int k = __shfl_xor_sync(0xffffffffu, at, o);
        better(w, k);
    }
    if ((tid & 31) == 0) { sv[tid >> 5] = v; si[tid >> 5] = at; }
    __syncthreads();
    v = sv[0]; at = si[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) better(sv[w], si[w]);
    __syncthreads();
}

constexpr int NONE = 0x7fffffff;              // the index of no candidate: behind every other of its value

// EPT values a thread; VEC: rows begin on 16-byte boundaries.  grid: (chunks, rows).
template <int EPT, bool VEC>
__global__ void __launch_bounds__(THREADS)
beam_chunk_kernel(const float* __restrict__ logits, long long ld, int V, int keep, float* __restrict__ chunk_ms, float* __restrict__ cand_x,
                  int* __restrict__ cand_at) {
    __shared__ float s_top[WARPS], s_pass[WARPS], s_sum[WARPS], s_x[COLLECT];
    __shared__ int s_at[COLLECT], s_n;
    __shared__ float s_bv[WARPS + 1];
    __shared__ int s_bi[WARPS + 1];
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int base = blockIdx.x * THREADS * EPT;
    const float* row = logits + (long long)blockIdx.y * ld;
    float x[EPT];
    auto place = [&](int e) { return VEC ? base + 4 * (tid + (e >> 2) * THREADS) + (e & 3) : base + tid + e * THREADS; };
    if (VEC) {
#pragma unroll
        for (int e = 0; e < EPT; e += 4) {
            const int v = place(e);
            if (v + 3 < V) {
                const float4 f = __ldcs(reinterpret_cast<const float4*>(row + v));
                x[e] = f.x; x[e + 1] = f.y; x[e + 2] = f.z; x[e + 3] = f.w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[e + k] = v + k < V ? row[v + k] : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < EPT; ++e) x[e] = place(e) < V ? __ldcs(row + place(e)) : -INFINITY;
    }
    if (tid == 0) s_n = 0;
    float mine = -INFINITY;
#pragma unroll
    for (int e = 0; e < EPT; ++e) mine = fmaxf(mine, x[e]);
    // the warps whose lanes all have values: the last chunk of a row may leave some without
    const int full = min(WARPS, (V - base) / (VEC ? 128 : 32));
    const float top_w = warp_top(mine);
    const float pass_w = warp_rth(mine, (keep + max(full, 1) - 1) / max(full, 1), lane);
    if (lane == 0) { s_top[warp] = top_w; s_pass[warp] = pass_w; }
    __syncthreads();
    float top = s_top[0], pass = full > 0 ? s_pass[0] : -INFINITY;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) {
        top = fmaxf(top, s_top[w]);
        if (w < full) pass = fminf(pass, s_pass[w]);
    }
    const float ref = top == -INFINITY ? 0.f : top;           // a NaN, or +inf - +inf, makes the sum a NaN
    const float shift = -ref * LOG2E;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
        sum += fast_exp2(fmaf(x[e], LOG2E, shift));
        if (x[e] >= pass && place(e) < V) {
            const int i = atomicAdd(&s_n, 1);                 // the order of arrival does not matter: they are ranked
            if (i < COLLECT) { s_x[i] = x[e]; s_at[i] = place(e); }
        }
    }
    if (top == INFINITY) sum = __int_as_float(0x7fc00000);
    sum = warp_sum(sum);
    if (lane == 0) s_sum[warp] = sum;
    pdl_trigger_late();
    __syncthreads();
    const size_t chunk = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (tid == 0) {
        float all = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) all += s_sum[w];
        chunk_ms[2 * chunk] = top;
        chunk_ms[2 * chunk + 1] = all;
    }
    const int n = s_n;
    auto put = [&](int rank, float v, int at) { cand_x[chunk * keep + rank] = v; cand_at[chunk * keep + rank] = at; };
    if (n <= COLLECT) {
        rank_collected(s_x, s_at, n, keep, tid, put);
        for (int i = n + tid; i < keep; i += THREADS) put(i, -INFINITY, NONE);      // a chunk of fewer values, or of NaNs
        return;
    }
    float last = INFINITY;                                    // what was taken last: +inf, -1 before the first
    int last_at = -1;
    for (int k = 0; k < keep; ++k) {
        float v = -INFINITY;
        int at = NONE;
#pragma unroll
        for (int e = 0; e < EPT; ++e)
            if (place(e) < V && (k == 0 ? x[e] == x[e] : before(last, last_at, x[e], place(e))) && before(x[e], place(e), v, at)) { v = x[e]; at = place(e); }
        block_best(v, at, s_bv, s_bi, tid);
        if (tid == 0) put(k, v, at);
        last = v;
        last_at = at;
    }
}

// grid: requests.
__global__ void __launch_bounds__(THREADS)
beam_merge_kernel(const float* __restrict__ scores, const float* __restrict__ chunk_ms, const float* __restrict__ cand_x,
                  const int* __restrict__ cand_at, int beams, int V, int chunks, int keep, float* __restrict__ scores_out,
                  int* __restrict__ beams_out, int* __restrict__ tokens_out) {
    __shared__ double s_shift[BEAM_MAX_BEAMS];                // score - lse; NaN: the row counts as -inf
    __shared__ double s_v[COLLECT], s_pass[WARPS], s_bv[WARPS + 1];
    __shared__ int s_at[COLLECT], s_n, s_bi[WARPS + 1];
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, req = blockIdx.x;
    const double none = -(double)INFINITY;
    if (tid == 0) s_n = 0;
    for (int b = warp; b < beams; b += WARPS) {
        const float* ms = chunk_ms + 2 * (size_t)(req * beams + b) * chunks;
        float top = -INFINITY;
        for (int c = lane; c < chunks; c += 32) top = fmaxf(top, ms[2 * c]);
        top = warp_max(top);
        double sum = 0.0;
        for (int c = lane; c < chunks; c += 32) {
            const float m = ms[2 * c];
            sum += m == -INFINITY ? (double)ms[2 * c + 1] * 0.0 : (double)ms[2 * c + 1] * exp((double)m - (double)top);      // x 0: a NaN stays one
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const float score = scores[req * beams + b];
            s_shift[b] = top != -INFINITY && isfinite(score) ? (double)score - ((double)top + log(sum)) : __longlong_as_double(0x7ff8000000000000ll);
        }
    }
    __syncthreads();
    const int per_row = chunks * keep, total = beams * per_row;
    // candidate i of the request: its total and its place (b, v) in the order of ties; a dead row offers its first tokens
    auto candidate = [&](int i, double& v, long long& at) {
        const int b = i / per_row, k = i - b * per_row;
        const double shift = s_shift[b];
        if (isnan(shift)) {
            v = none;
            at = k < keep && k < V ? (long long)b * V + k : -1;
            return;
        }
        const size_t from = (size_t)(req * beams + b) * per_row + k;
        const int token = cand_at[from];
        v = (double)cand_x[from] + shift;
        at = token == NONE ? -1 : (long long)b * V + token;
        if (at < 0) v = none;
    };
    double mine = none;
    for (int i = tid; i < total; i += THREADS) {
        double v;
        long long at;
        candidate(i, v, at);
        if (at >= 0 && v > mine) mine = v;
    }
    const double pass_w = warp_rth(mine, (keep + WARPS - 1) / WARPS, lane);
    if (lane == 0) s_pass[warp] = pass_w;
    __syncthreads();
    double pass = s_pass[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) pass = s_pass[w] < pass ? s_pass[w] : pass;
    for (int i = tid; i < total; i += THREADS) {
        double v;
        long long at;
        candidate(i, v, at);
        if (at >= 0 && v >= pass) {
            const int n = atomicAdd(&s_n, 1);
            if (n < COLLECT) { s_v[n] = v; s_at[n] = (int)at; }
        }
    }
    __syncthreads();
    const int n = s_n;
    auto put = [&](int rank, double v, int at) {
        const size_t to = (size_t)req * keep + rank;
        scores_out[to] = (float)v;
        beams_out[to] = at / V;
        tokens_out[to] = at % V;
    };
    if (n <= COLLECT) {
        rank_collected(s_v, s_at, n, keep, tid, put);
        return;
    }
    double last = (double)INFINITY;
    int last_at = -1;
    for (int k = 0; k < keep; ++k) {
        double best = none;
        int best_at = NONE;
        for (int i = tid; i < total; i += THREADS) {
            double v;
            long long at;
            candidate(i, v, at);
            if (at >= 0 && before(last, last_at, v, (int)at) && before(v, (int)at, best, best_at)) { best = v; best_at = (int)at; }
        }
        block_best(best, best_at, s_bv, s_bi, tid);
        if (tid == 0) put(k, best, best_at);
        last = best;
        last_at = best_at;
    }
}

int chunk_values(long long rows, int V) {
    // short chunks where long ones would leave SMs without work
    const long long long_ctas = rows * ((V + THREADS * 32 - 1) / (THREADS * 32));
    return long_ctas >= 2 * rb_num_sms() ? THREADS * 32 : THREADS * 8;
}

}  // namespace

RB_EXPORT int rb_beam_max_keep() { return BEAM_MAX_KEEP; }
RB_EXPORT int rb_beam_max_beams() { return BEAM_MAX_BEAMS; }
// 4-byte words of scratch.
RB_EXPORT long long rb_beam_scratch(int rows, int V, int keep) {
    const int chunk = chunk_values(rows, V);
    const long long chunks = (V + chunk - 1) / chunk;
    return rows * chunks * (2 + 2ll * keep);
}

RB_EXPORT int rb_beam_select(const float* logits, long long ld, const float* scores, int requests, int beams, int V, int keep, float* scores_out,
                             int* beams_out, int* tokens_out, void* scratch, cudaStream_t st) {
    if (requests <= 0) return 0;
    const int rows = requests * beams;
    if (beams < 1 || beams > BEAM_MAX_BEAMS || keep < 1 || keep > BEAM_MAX_KEEP || V < 1 || rows > 65535) return (int)cudaErrorInvalidValue;
    if ((long long)beams * V > 0x7ffffffell || keep > (long long)beams * V) return (int)cudaErrorInvalidValue;
    const int chunk = chunk_values(rows, V), chunks = (V + chunk - 1) / chunk;
    float* ms = (float*)scratch;
    float* cand_x = ms + 2ll * rows * chunks;
    int* cand_at = (int*)(cand_x + (long long)rows * chunks * keep);
    const bool vec = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
    dim3 grid(chunks, rows);
    auto kernel = chunk == THREADS * 32 ? (vec ? beam_chunk_kernel<32, true> : beam_chunk_kernel<32, false>)
                                        : (vec ? beam_chunk_kernel<8, true> : beam_chunk_kernel<8, false>);
    int e = rb_launch_pdl(kernel, grid, dim3(THREADS), 0, st, logits, ld, V, keep, ms, cand_x, cand_at);
    if (e) return e;
    return rb_launch_pdl(beam_merge_kernel, dim3(requests), dim3(THREADS), 0, st, scores, ms, cand_x, cand_at, beams, V, chunks, keep,
                         scores_out, beams_out, tokens_out);
}
