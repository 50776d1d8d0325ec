// Beam search's selection: of all continuations of a request's beams, beams x vocabulary, the `keep` with the highest total
//   total(b, v) = score[b] + logits[b, v] - log(sum_u exp(logits[b, u])),
// falling, ties to the lowest (b, v).  A total that is no number (a row with a NaN or +inf, a row of -inf alone) counts as -inf, and so
// do all of a row whose score is not finite.
//
// The logits are read once.  beam_part_kernel: a CTA walks a part of a row tile by tile (the next ones on their way to shared memory, every
// thread its own values, so no barrier stands between them and their use), keeps each thread's maximum and sum of exponentials, and collects
// the values that may be among the part's `keep` best: the order within a row is that of the logits.  In the first tile each warp's r-th
// highest thread maximum, r = keep / warps rounded up, is passed by r values of that warp, so the lowest of these over the warps is passed by
// `keep` values and by few more; they are ranked by counting.  From then on what is above the keep-th best so far (an equal value comes later,
// hence behind it) is collected, without a barrier, and that bound is renewed behind 2, 4, 8, ... tiles: at most some `keep` values a tile of
// random logits.  Where what is collected overflows (rising logits) the part is walked once more, with a selection in every tile, and
// where a tile's own overflows (equal logits), its best are taken one by one.
// beam_merge_kernel: a CTA a request puts the rows' sums together and takes the best of all parts' lists.  Totals are
// compared in 64 bits, a logit less its row's maximum first, so that logits which differ keep their order whatever their size and however far down the
// scores are; one rounding at the store.  (Beside a score beyond some -2^50, a finite mask's, 64 bits do not tell words apart either: which of them are
// taken is then the lists' and the places' order.)  Sums of exponentials are float32; a term d below the
// maximum is off by 2^-22 + d 2^-23 of itself at most, whatever the logits' size.
//
// What bounds it: 128 rows of 151,936, the 16 best of eight beams, 27.4 us, of which the parts take 24 (3.2 TB/s; a stream alone would take 12): a CTA's first
// tile waits 2.3 us for memory and 4.6 for its selection, later tiles for the logits, the last ranking and sums 2 us, and 256 CTAs fill 108 of 148 SMs
// twice and the others once.  Four rows of 32,768: 7.9 us, a selection and a merge.  The first form, without the ring and
// the rising bound, took 40 and 10.9 us.
#include "pairs.cuh"

#define BEAM_MAX_KEEP 128
#define BEAM_MAX_BEAMS 64
#define BEAM_MAX_WORDS (1 << 29)              // of a row: twice a row's length and a few tiles stay within an int

namespace {

constexpr int PART_THREADS = 512, SHORT_THREADS = 256, MERGE_THREADS = 256;
constexpr int COLLECT = 512;
constexpr int RING = 3;                       // tiles on their way: two of 32 KB for each of two CTAs an SM
constexpr float LOG2E = 1.4426950408889634f;


// A value of a row and its place in one number that grows as the value does, and falls with the place: the order of the selection.  -0 is 0; a
// NaN is never asked about.  NONE, the lowest, is no value's.
typedef unsigned long long Key;
constexpr Key NONE = 0ull;
__device__ __forceinline__ Key key_of(float x, int at) {
    const unsigned u = __float_as_uint(x + 0.f);
    return (Key)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << 32 | (0xffffffffu - (unsigned)at);
}
__device__ __forceinline__ float value_of(Key k) {
    const unsigned u = (unsigned)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u ^ 0x80000000u) : ~u);
}
__device__ __forceinline__ int place_of(Key k) { return (int)(0xffffffffu - (unsigned)k); }

// The r-th highest of a warp's values, equal ones counted one by one; -inf where there are fewer.
__device__ __forceinline__ float warp_rth(float v, int r, int lane) {
    float top = -INFINITY;
    bool out = false;
    for (int i = 0; i < r; ++i) {
        top = warp_max(out ? -INFINITY : v);
        const unsigned who = __ballot_sync(0xffffffffu, !out && v == top);
        if (who == 0u) return -INFINITY;                      // fewer than r lanes
        if (lane == __ffs(who) - 1) out = true;
    }
    return top;
}
// How many of the n keys are higher than k; one key of room behind them.
__device__ __forceinline__ int rank_among(const Key* keys, int n, Key k) {
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + j);
        rank += (two.x > k ? 1 : 0) + (j + 1 < n && two.y > k ? 1 : 0);
    }
    return rank;
}
// The highest of every thread's key, for all threads.
template <int WARPS>
__device__ __forceinline__ Key block_best(Key k, Key* scratch, int tid) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Key other = __shfl_xor_sync(0xffffffffu, k, o);
        k = other > k ? other : k;
    }
    if ((tid & 31) == 0) scratch[tid >> 5] = k;
    __syncthreads();
    k = scratch[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) k = scratch[w] > k ? scratch[w] : k;
    __syncthreads();
    return k;
}

// T threads, E values a thread and tile; VEC: rows begin on 16-byte boundaries.  grid: (parts, rows).
template <int T, int E, bool VEC>
__global__ void __launch_bounds__(T, E == 16 ? 2 : 4)
beam_part_kernel(const float* __restrict__ logits, long long ld, int V, int part, int keep, float* __restrict__ part_ms, Key* __restrict__ cand) {
    constexpr int WARPS = T / 32, TILE = T * E;
    extern __shared__ __align__(16) float ring[];             // [RING][TILE]
    __shared__ __align__(16) Key s_key[2][COLLECT + 2];
    __shared__ Key s_best[WARPS];
    __shared__ float s_a[WARPS], s_b[WARPS];
    __shared__ int s_n;
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = blockIdx.x * part, end = min(V, first + part);
    const float* row = logits + (long long)blockIdx.y * ld;
    auto offset = [&](int e) { return VEC ? 4 * (tid + (e >> 2) * T) + (e & 3) : tid + e * T; };      // of a thread's value e in a tile
    auto ask = [&](int base, int stage) {
        float* to = ring + stage * TILE;
        if (VEC && base + TILE <= end) {
            const float* src = row + base + 4 * tid;
            const unsigned at = (unsigned)__cvta_generic_to_shared(to + 4 * tid);
#pragma unroll
            for (int e = 0; e < E; e += 4)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(at + (unsigned)(e * T * 4)), "l"(src + e * T));
        } else {
#pragma unroll
            for (int e = 0; e < E; e += VEC ? 4 : 1) {        // what lies behind the part is not looked at
                const int v = base + offset(e);
                const unsigned at = (unsigned)__cvta_generic_to_shared(to + offset(e));
                if (VEC) {
                    const int bytes = 4 * max(0, min(4, end - v));
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(at), "l"(bytes > 0 ? row + v : row), "r"(bytes));
                } else if (v < end) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(at), "l"(row + v));
                }
            }
        }
        asm volatile("cp.async.commit_group;\n" ::);
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) ask(first + i * TILE, i);      // tiles behind the part ask for nothing
    if (tid == 0) s_n = 0;
    int buf = 0, held = 0;                                    // what has been collected: s_key[buf][0 .. held)
    float above = -INFINITY;                                  // the keep-th best so far
    float top = -INFINITY, sum = 0.f;                         // this thread's maximum, and sum of 2^((x - maximum) log2(e))
    bool odd = false;                                         // +inf: the sum is no number
    auto collect = [&](float x, int at) {                     // the order of arrival does not matter: they are ranked
        const int i = atomicAdd(&s_n, 1);
        if (i < COLLECT) s_key[buf][i] = key_of(x, at);
    };
    // the collected ones in order, the first `keep` of them alone
    auto shorten = [&]() {
        for (int i = tid; i < held; i += T) {
            const Key k = s_key[buf][i];
            const int rank = rank_among(s_key[buf], held, k);
            if (rank < keep) s_key[buf ^ 1][rank] = k;
        }
        buf ^= 1;
        held = min(held, keep);
        if (tid == 0) s_n = held;
        __syncthreads();
        if (held == keep) above = value_of(s_key[buf][keep - 1]);
    };
    // a tile's values among the best: all threads together
    auto select = [&](int base, const float (&x)[E], float mine, bool is_first) {
        float bar = above;
        bool strict = true;
        const int passing = __syncthreads_count(is_first || mine > above);
        if (passing == 0) return;
        if (passing > COLLECT / 2 / E) {
            // the warps whose threads all have values: the last tile of a row may leave some without
            const int full = min(WARPS, (end - base) / (VEC ? 128 : 32));
            const float pass_w = warp_rth(mine, (keep + max(full, 1) - 1) / max(full, 1), lane);
            if (lane == 0) s_a[warp] = pass_w;
            __syncthreads();
            float pass = full > 0 ? s_a[0] : -INFINITY;
#pragma unroll
            for (int w = 1; w < WARPS; ++w)
                if (w < full) pass = fminf(pass, s_a[w]);
            if (is_first || pass > above) { bar = pass; strict = false; }
        }
        if (strict ? mine > bar : mine >= bar) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if ((strict ? x[e] > bar : x[e] >= bar) && base + offset(e) < end) collect(x[e], base + offset(e));
        }
        __syncthreads();
        const int now = s_n;
        __syncthreads();                                      // everyone has the count before shorten() writes the next one
        if (now > COLLECT) {                                  // no room: this tile's best one by one, behind what was held before
            Key last = ~0ull;
            for (int k = 0; k < keep; ++k) {
                Key best = NONE;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (base + offset(e) < end && x[e] == x[e]) {
                        const Key mine_e = key_of(x[e], base + offset(e));
                        if (mine_e < last && mine_e > best) best = mine_e;
                    }
                best = block_best<WARPS>(best, s_best, tid);
                if (tid == 0) s_key[buf][held + k] = best;
                last = best;
            }
            held += keep;
            __syncthreads();
            shorten();
        } else {
            held = now;
            if (is_first || held > COLLECT / 4) shorten();    // there is always room for another `keep`
        }
    };
    // a tile's values out of the ring, with the highest of each four and of all
    auto take = [&](const float* from, int base, float (&x)[E], float (&four)[E / 4]) {
        if (VEC) {
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(from + offset(e));
                x[e] = f.x; x[e + 1] = f.y; x[e + 2] = f.z; x[e + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = from[offset(e)];
        }
        if (base + TILE > end) {
#pragma unroll
            for (int e = 0; e < E; ++e) if (base + offset(e) >= end) x[e] = -INFINITY;
        }
        float best = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            four[e >> 2] = fmaxf(max3(x[e], x[e + 1], x[e + 2]), x[e + 3]);
            best = fmaxf(best, four[e >> 2]);
        }
        return best;
    };
    int stage = 0, due = first;
    for (int base = first; base < end; base += TILE) {
        ask(base + (RING - 1) * TILE, stage == 0 ? RING - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;\n" ::"n"(RING - 1));
        const float* from = ring + stage * TILE;
        stage = stage + 1 == RING ? 0 : stage + 1;
        float x[E], four[E / 4];
        const float mine = take(from, base, x, four);
        const float m = fmaxf(top, mine), ref = m == -INFINITY ? 0.f : m;
        unsigned long long tile = pack2(0.f, 0.f);            // a sum of few terms at a time keeps its rounding small
        // the maximum is taken off before the scale: a product of it would be off by what counts where logits are large, and infinite at the lowest
        const unsigned long long unit2 = pack2(LOG2E, LOG2E), back2 = pack2(-ref, -ref);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float y0, y1;
            unpack2(mul2(add2(pack2(x[e], x[e + 1]), back2), unit2), y0, y1);
            tile = add2(tile, pack2(fast_exp2(y0), fast_exp2(y1)));
        }
        float even, uneven;
        unpack2(tile, even, uneven);
        sum = sum * fast_exp2((top - ref) * LOG2E) + (even + uneven);       // 2^-inf before the first number
        top = m;
        odd = odd || m == INFINITY;
        if (base == first) {
            select(base, x, mine, true);
            due = base + TILE;
        } else {
            if (mine > above) {
                unsigned which = 0u;
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    if (four[e >> 2] > above) {
#pragma unroll
                        for (int k = e; k < e + 4; ++k) which |= x[k] > above ? 1u << k : 0u;
                    }
                for (; which != 0u; which &= which - 1u) {
                    const int e = __ffs(which) - 1;
                    collect(from[offset(e)], base + offset(e));
                }
            }
            if (base == due) {                                // twice as much has been seen: the keep-th best of it
                due = first + 2 * (base - first) + TILE;
                __syncthreads();
                const int now = s_n;
                __syncthreads();
                if (now <= COLLECT && now > keep) {
                    held = now;
                    shorten();
                }
            }
        }
    }
    __syncthreads();
    held = s_n;
    if (held > COLLECT) {                                     // once more, tile by tile
        asm volatile("cp.async.wait_group 0;\n" ::);          // of tiles behind the part: zeros that may still be on their way to the ring
        __syncthreads();
        if (tid == 0) s_n = 0;
        held = 0;
        above = -INFINITY;
        for (int base = first; base < end; base += TILE) {
            ask(base, 0);
            asm volatile("cp.async.wait_group 0;\n" ::);
            float x[E], four[E / 4];
            const float mine = take(ring, base, x, four);
            select(base, x, mine, base == first);
        }
        __syncthreads();
    }
    pdl_trigger_late();
    // the part's maximum and sum
    if (odd) sum = __int_as_float(0x7fc00000);
    const float top_w = warp_max(top);
    sum = warp_sum(top == -INFINITY ? sum * 0.f : sum * fast_exp2((top - top_w) * LOG2E));       // x 0: a NaN stays one
    if (lane == 0) { s_b[warp] = top_w; s_a[warp] = sum; }
    __syncthreads();
    const size_t slot = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (warp == 0) {
        const float m_w = lane < WARPS ? s_b[lane] : -INFINITY, l_w = lane < WARPS ? s_a[lane] : 0.f;
        const float m = warp_max(m_w), all = warp_sum(m_w == -INFINITY ? l_w * 0.f : l_w * fast_exp2((m_w - m) * LOG2E));
        if (lane == 0) {
            part_ms[2 * slot] = m;
            part_ms[2 * slot + 1] = all;
        }
    }
    // the list in order; short of `keep`: a part of fewer values, or of NaNs
    for (int i = tid; i < held; i += T) {
        const Key k = s_key[buf][i];
        const int rank = rank_among(s_key[buf], held, k);
        if (rank < keep) cand[slot * keep + rank] = k;
    }
    for (int i = held + tid; i < keep; i += T) cand[slot * keep + i] = NONE;
}

// Whether total a at place i comes before total b at place j.
__device__ __forceinline__ bool before(double a, int i, double b, int j) { return a > b || (a == b && i < j); }

// grid: requests.  A thread's first HELD candidates stay in registers.
constexpr int HELD = 4;
__global__ void __launch_bounds__(MERGE_THREADS)
beam_merge_kernel(const float* __restrict__ scores, const float* __restrict__ part_ms, const Key* __restrict__ cand, int beams, int V, int parts,
                  int keep, float* __restrict__ scores_out, int* __restrict__ beams_out, int* __restrict__ tokens_out) {
    constexpr int T = MERGE_THREADS, WARPS = T / 32;
    // a row's maximum, which is taken off its logits first (they are of one size, the score is not), and score - log(sum); NaN: the row counts as -inf
    __shared__ double s_top[BEAM_MAX_BEAMS], s_shift[BEAM_MAX_BEAMS];
    __shared__ double s_v[COLLECT];
    __shared__ int s_at[COLLECT], s_n, s_count[2];
    __shared__ __align__(16) float s_list[T];
    __shared__ float s_pass;
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, req = blockIdx.x;
    const double none = -(double)INFINITY;
    const int lists = beams * parts, per_row = parts * keep, total = beams * per_row;
    const Key* mine = cand + (size_t)req * total;
    // The bar: a list's q-th candidate stands for q that are no worse, so the nth highest of the lists' q-th candidates, q = keep / nth rounded
    // up, is passed by `keep` candidates and by few more.  A quarter of the lists has to get there: those of beams that are far behind do
    // not.  256 lists, evenly picked, will do.
    const int m = min(lists, T), nth = max(1, min(m / 4, keep)), q = (keep + nth - 1) / nth;
    const int my_list = (int)((long long)tid * lists / m);
    const Key asked = tid < m ? mine[(size_t)my_list * keep + q - 1] : NONE;
    Key first[HELD];                                          // asked for before the rows' sums are worked out
#pragma unroll
    for (int u = 0; u < HELD; ++u) first[u] = tid + u * T < total ? mine[tid + u * T] : NONE;
    if (tid == 0) { s_n = 0; s_pass = -INFINITY; s_count[0] = s_count[1] = 0; }
    for (int b = warp; b < beams; b += WARPS) {
        const float2* ms = reinterpret_cast<const float2*>(part_ms) + (size_t)(req * beams + b) * parts;
        const float score = scores[req * beams + b];
        float top = -INFINITY;
        for (int c = lane; c < parts; c += 32) top = fmaxf(top, ms[c].x);
        top = warp_max(top);
        double sum = 0.0;
        for (int c = lane; c < parts; c += 32) {
            const float2 p = ms[c];
            sum += p.x == -INFINITY ? (double)(p.y * 0.f) : (double)p.y * (double)expf(p.x - top);      // x 0: a NaN stays one
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            s_top[b] = (double)top;
            s_shift[b] = top != -INFINITY && isfinite(score) ? (double)score - log(sum) : __longlong_as_double(0x7ff8000000000000ll);
        }
    }
    __syncthreads();
    // candidate i of the request: its total and its place (b, v) in the order of ties, -1 where there is none; a dead row offers its first words
    auto candidate = [&](int i, Key key, double& v, int& at) {
        const int b = i / per_row, k = i - b * per_row;
        const double shift = s_shift[b];
        v = ((double)value_of(key) - s_top[b]) + shift;
        at = key == NONE ? -1 : b * V + place_of(key);
        if (isnan(shift)) {
            v = none;
            at = k < keep && k < V ? b * V + k : -1;
        }
    };
    float low = -INFINITY;                                    // rounded down to 32 bits, the bar is passed by no fewer
    if (tid < m) {
        double v;
        int at;
        candidate(my_list * keep + q - 1, asked, v, at);
        if (at >= 0) low = __double2float_rd(v);
        s_list[tid] = low;
    }
    __syncthreads();
    if (tid < m) {
        int ahead = 0;
        for (int j = 0; j < m; ++j) ahead += s_list[j] > low || (s_list[j] == low && j < tid) ? 1 : 0;
        if (ahead == nth - 1) s_pass = low;
    }
    __syncthreads();
    const double pass = s_pass;
    // f(total, place) for all of this thread's candidates
    auto each = [&](auto f) {
#pragma unroll
        for (int u = 0; u < HELD; ++u) {
            const int i = tid + u * T;
            if (i < total) {
                double v;
                int at;
                candidate(i, first[u], v, at);
                if (at >= 0) f(v, at);
            }
        }
        for (int i = tid + HELD * T; i < total; i += T) {
            double v;
            int at;
            candidate(i, mine[i], v, at);
            if (at >= 0) f(v, at);
        }
    };
    auto gather = [&](auto passes) {
        each([&](double v, int at) {
            if (passes(v, at)) {
                const int n = atomicAdd(&s_n, 1);
                if (n < COLLECT) { s_v[n] = v; s_at[n] = at; }
            }
        });
        __syncthreads();
        return s_n;
    };
    int n = gather([&](double v, int) { return v >= pass; });
    if (n > COLLECT) {
        // Too many: the bar is put between them by halving, by their totals as integers of the same order, and where as many are equal, by their
        // places.  `keep` pass `low` and do not pass `high`; of those whose total is the bar, last_at is the last place that passes.
        auto order = [](double v) {
            const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
            return (u >> 63) ? ~u : u | 0x8000000000000000ull;
        };
        auto passes = [&](double v, int at, unsigned long long bar, int to) {
            const unsigned long long o = order(v);
            return o > bar || (o == bar && at <= to);
        };
        int round = 0;
        auto count = [&](unsigned long long bar, int to) {
            int passing = 0;
            each([&](double v, int at) { passing += passes(v, at, bar, to) ? 1 : 0; });
            passing = __reduce_add_sync(0xffffffffu, passing);
            if (lane == 0) atomicAdd(&s_count[round], passing);
            __syncthreads();
            passing = s_count[round];
            round ^= 1;
            __syncthreads();
            if (tid == 0) s_count[round ^ 1] = 0;             // added to again behind the next call's barriers
            return passing;
        };
        unsigned long long low = order(pass), high = order((double)INFINITY) + 1;
        int last_at = beams * V - 1;
        bool fits = false;
        while (!fits && high - low > 1) {
            const unsigned long long mid = low + (high - low) / 2;
            const int passing = count(mid, last_at);
            if (passing >= keep) { low = mid; fits = passing <= COLLECT; } else high = mid;
        }
        for (int from = -1; !fits && last_at - from > 1;) {
            const int mid = from + (last_at - from) / 2, passing = count(low, mid);
            if (passing >= keep) { last_at = mid; fits = passing <= COLLECT; } else from = mid;
        }
        if (tid == 0) s_n = 0;
        __syncthreads();
        n = min(gather([&](double v, int at) { return passes(v, at, low, last_at); }), COLLECT);
    }
    for (int i = tid; i < n; i += T) {
        const double v = s_v[i];
        const int at = s_at[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += before(s_v[j], s_at[j], v, at) ? 1 : 0;
        if (rank < keep) {
            const size_t to = (size_t)req * keep + rank;
            scores_out[to] = (float)v;
            beams_out[to] = at / V;
            tokens_out[to] = at % V;
        }
    }
}

// How a row is cut: parts of `part` values.  Long ones for the kernel of 512 threads and 16 values a thread, two CTAs an SM, short ones for that
// of 256 and 4, which has a first tile's selection behind it sooner.
struct Cut {
    bool short_parts;
    int part, parts;
    Cut(long long rows, int V) {
        const int quads = (V + 3) / 4;
        auto values = [&](long long slots) {                  // parts that fill the device once
            const long long want = rows >= slots ? 1 : slots / rows;
            return 4 * (int)((quads + want - 1) / want);
        };
        part = values(2ll * rb_num_sms());
        short_parts = part < PART_THREADS * 16;
        if (short_parts) {
            part = values(4ll * rb_num_sms());
            if (part < SHORT_THREADS * 4) part = SHORT_THREADS * 4;            // a tile at least
        }
        parts = (V + part - 1) / part;
    }
};

}  // namespace

RB_EXPORT int rb_beam_max_keep() { return BEAM_MAX_KEEP; }
RB_EXPORT int rb_beam_max_beams() { return BEAM_MAX_BEAMS; }
RB_EXPORT int rb_beam_max_words() { return BEAM_MAX_WORDS; }
// 4-byte words of scratch: every part's maximum, sum, and list of keys of eight bytes.
RB_EXPORT long long rb_beam_scratch(int rows, int V, int keep) { return rows * (long long)Cut(rows, V).parts * (2 + 2ll * keep); }

RB_EXPORT int rb_beam_select(const float* logits, long long ld, const float* scores, int requests, int beams, int V, int keep, float* scores_out,
                             int* beams_out, int* tokens_out, void* scratch, cudaStream_t st) {
    if (requests <= 0) return 0;
    const int rows = requests * beams;
    if (beams < 1 || beams > BEAM_MAX_BEAMS || keep < 1 || keep > BEAM_MAX_KEEP || V < 1 || rows > 65535) return (int)cudaErrorInvalidValue;
    if (V > BEAM_MAX_WORDS || (long long)beams * V > 0x7ffffffell || keep > (long long)beams * V || ((uintptr_t)scratch & 15)) return (int)cudaErrorInvalidValue;
    const Cut cut(rows, V);
    float* ms = (float*)scratch;
    Key* cand = (Key*)(ms + 2ll * rows * cut.parts);
    const bool vec = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
    dim3 grid(cut.parts, rows);
    constexpr int SMEM = sizeof(float) * RING * PART_THREADS * 16;
    static PerDevice configured;
    const int rc = configured.once([&](int) {
        cudaError_t c = cudaFuncSetAttribute(beam_part_kernel<PART_THREADS, 16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (c == cudaSuccess) c = cudaFuncSetAttribute(beam_part_kernel<PART_THREADS, 16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        return c;
    });
    if (rc) return rc;
    auto kernel = cut.short_parts ? (vec ? beam_part_kernel<SHORT_THREADS, 4, true> : beam_part_kernel<SHORT_THREADS, 4, false>)
                                  : (vec ? beam_part_kernel<PART_THREADS, 16, true> : beam_part_kernel<PART_THREADS, 16, false>);
    int e = rb_launch_pdl(kernel, grid, dim3(cut.short_parts ? SHORT_THREADS : PART_THREADS),
                          cut.short_parts ? sizeof(float) * RING * SHORT_THREADS * 4 : (size_t)SMEM, st, logits, ld, V, cut.part, keep, ms, cand);
    if (e) return e;
    return rb_launch_pdl(beam_merge_kernel, dim3(requests), dim3(MERGE_THREADS), 0, st, scores, ms, cand, beams, V, cut.parts, keep, scores_out,
                         beams_out, tokens_out);
}
