// Attention of drafted trees over the paged cache: the step that checks several continuations of a request at once.
//
// A segment brings n nodes, its tree: parent[i] < i is the node before node i, the root (node 0 as a rule; any node with parent < 0) is
// the first token behind the segment's c cached ones.  The keys and values of node i already lie in slot c + i of the request's
// pages; its position is c + depth(i).  Node i sees the cached keys j < c, and of the tree itself and its ancestors.  With a
// window both must lie less than `window` positions back: j > c + depth(i) - window, depth(i) - depth(a) < window.
//   s = scale q.k   (softcap > 0: softcap tanh(s / softcap))
//   out = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink[h] - m))
// A block that the table marks as gone (-1) reads as keys and values of zero; a row that sees no key gets zeros.
//
// Which ancestors a node has is not read from a mask: a thread walks up its parents once (the list of a segment, at most
// TREE_MAX_NODES, is in shared memory) and keeps the bits.  A parent that is not below its child ends the walk, so a list that is no
// tree gives some mask, never a hang or a read out of range.
//
// Rows are (node, query head) pairs that share a key/value head, G = Hq / Hkv heads a node: row r is node r / G, head r % G.  The
// keys of a segment are split over CTAs, one for every `share` key tiles (0: one CTA walks them all); each leaves its unnormalised
// output, maximum and sum in float32, and tree_merge_kernel joins them in the order of the shares.  So the result depends
// on `share`, which the host works out from the step's lengths, and on nothing else of the launch.
#include "tc5.cuh"
#include "tma.cuh"

#define TREE_MAX_NODES 256
#define TREE_WORDS (TREE_MAX_NODES / 32)
#define TREE_MAX_D 256

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KEY_TILE = 64;                  // the unit of `share`

// What a CTA knows about its segment.
struct Segment {
    int q_begin, n, c, lo, hi, jt0, tiles, n_split;
    __device__ __forceinline__ Segment(const int* cu_q, const int* seg_pos0, int seg, int window, int share, int max_split) {
        q_begin = cu_q[seg];
        n = min(cu_q[seg + 1] - q_begin, TREE_MAX_NODES);
        c = max(seg_pos0[seg], 0);
        lo = window > 0 ? max(0, c - window + 1) : 0;         // the root's first key: no node sees an earlier one
        hi = c + n - 1;                                       // the last slot
        jt0 = lo / KEY_TILE;
        tiles = n > 0 ? hi / KEY_TILE - jt0 + 1 : 0;
        n_split = share > 0 ? min(max_split, max(1, (tiles + share - 1) / share)) : 1;
    }
};

// The node's own line: bit a of `line` for node x itself and its ancestors less than `window` steps up (window <= 0: all); returns
// the node's depth.  parent: the segment's list in shared memory.
__device__ __forceinline__ int tree_line(const int* parent, int x, int window, unsigned (&line)[TREE_WORDS]) {
#pragma unroll
    for (int w = 0; w < TREE_WORDS; ++w) line[w] = 0u;
    int depth = 0;
    for (int y = x;;) {
        if (window <= 0 || depth < window) line[y >> 5] |= 1u << (y & 31);
        const int up = parent[y];
        if (up < 0 || up >= y) break;
        y = up;
        ++depth;
    }
    return depth;
}
// Bits [at, at + 32) of a line; what lies outside it is zero.
__device__ __forceinline__ unsigned line_bits(const unsigned* line, int at) {
    if (at <= -32 || at >= TREE_MAX_NODES) return 0u;
    const int w = at >> 5, s = at & 31;                       // at < 0: w = -1
    const unsigned lo = w >= 0 ? line[w] : 0u, hi = w + 1 < TREE_WORDS ? line[w + 1] : 0u;
    return __funnelshift_r(lo, hi, s);
}

// ---------------------------------------------------------------------------------------- CUDA cores, any type and head size
constexpr int SW = 8, RW = 4;                 // warps, rows a warp
constexpr int SROWS = SW * RW;
constexpr int SKEYS = 32;                     // keys of a tile in shared memory

__device__ __forceinline__ void cp16(float* smem, const float* gmem, int bytes) {       // bytes behind `bytes` become zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((unsigned)__cvta_generic_to_shared(smem)), "l"(gmem), "r"(bytes));
}

// A warp owns four rows; lane j of a tile scores key j, the online softmax advances tile by tile, a lane keeps columns
// 4 lane + 128 k ..+ 3 of the rows' outputs.  The eight warps share a tile of keys and values in shared memory, the next one on
// its way meanwhile.  A key that a row does not see is left out, not multiplied by zero: it may hold anything.
// grid: (row blocks x kv heads, segments, splits).  NC: runs of 128 columns.
template <typename TA, int NC>
__global__ void __launch_bounds__(32 * SW, NC == 1 ? 2 : 1)
tree_simt_kernel(const TA* __restrict__ q, int ld, const TA* __restrict__ kpool, const TA* __restrict__ vpool,
                 const int* __restrict__ cu_q, const int* __restrict__ seg_pos0, const int* __restrict__ tree_parent,
                 const int* __restrict__ block_table, int bt_stride, int page_size, TA* __restrict__ out,
                 float* __restrict__ part_o, float* __restrict__ part_ml, int total_rows, int Hq, int Hkv, int D, float scale, int window,
                 float softcap, const float* __restrict__ sink, int share, int vec) {
    const int seg = blockIdx.y, kvh = blockIdx.x % Hkv, row0 = blockIdx.x / Hkv * SROWS, split = blockIdx.z, G = Hq / Hkv;
    const Segment sg(cu_q, seg_pos0, seg, window, share, gridDim.z);
    const int rows = min(SROWS, sg.n * G - row0);
    if (rows <= 0 || split >= sg.n_split) return;
    const int D4 = (D + 3) & ~3, pitch = D4 + 4;
    extern __shared__ __align__(16) float tree_smem[];
    float* qs = tree_smem;                                             // [SROWS][pitch]
    float* tiles = qs + SROWS * pitch;                                 // [2][keys, values][SKEYS][pitch]
    __shared__ int parent[TREE_MAX_NODES];
    __shared__ unsigned lines[SROWS][TREE_WORDS];
    __shared__ int depths[SROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int* bt = block_table + (size_t)seg * bt_stride;
    const size_t head_stride = (size_t)page_size * D;
    const int r0 = warp * RW, nr = min(RW, rows - r0);                 // this warp's rows (nr <= 0: none)

    // this CTA's keys: [j_begin, j_end)
    const int t0 = share > 0 ? split * share : 0, t1 = share > 0 && split + 1 < sg.n_split ? t0 + share : sg.tiles;
    const int j_begin = max((sg.jt0 + t0) * KEY_TILE, sg.lo / SKEYS * SKEYS), j_end = min((sg.jt0 + t1) * KEY_TILE, sg.hi + 1);

    const int per = D4 >> 2;
    auto fetch = [&](int j0, int buf) {
        float* ks = tiles + buf * 2 * SKEYS * pitch;
        int page_r[SKEYS / SW];                                        // looked up together, not one behind the other
#pragma unroll
        for (int i = 0; i < SKEYS / SW; ++i) {
            const int j = j0 + warp + i * SW;
            page_r[i] = j >= sg.lo && j < j_end ? bt[j / page_size] : -1;
        }
#pragma unroll
        for (int i = 0; i < SKEYS / SW; ++i) {
            const int jj = warp + i * SW, j = j0 + jj, page = page_r[i];
            const size_t at = page < 0 ? 0 : ((size_t)page * Hkv + kvh) * head_stride + (size_t)(j % page_size) * D;
            float* kd = ks + jj * pitch;
            float* vd = kd + SKEYS * pitch;
            for (int c = lane; c < per; c += 32) {
                const int d = 4 * c;
                if (vec) {
                    cp16(kd + d, reinterpret_cast<const float*>(kpool) + at + d, page < 0 ? 0 : 16);
                    cp16(vd + d, reinterpret_cast<const float*>(vpool) + at + d, page < 0 ? 0 : 16);
                } else {
                    for (int e = d; e < d + 4; ++e) {
                        const bool there = page >= 0 && e < D;
                        kd[e] = there ? to_f32(kpool[at + e]) : 0.f;
                        vd[e] = there ? to_f32(vpool[at + e]) : 0.f;
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;\n" ::);
    };
    fetch(j_begin, 0);
    for (int i = tid; i < sg.n; i += 32 * SW) parent[i] = tree_parent[sg.q_begin + i];
    for (int d = lane; d < D4; d += 32)                                // a warp reads its own rows only; rows that do not exist are zero
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const int row = row0 + r0 + i;
            qs[(r0 + i) * pitch + d] = i < nr && d < D ? to_f32(q[(size_t)(sg.q_begin + row / G) * ld + (size_t)(kvh * G + row % G) * D + d]) : 0.f;
        }
    __syncthreads();
    if (tid < rows) {
        unsigned line[TREE_WORDS];
        depths[tid] = tree_line(parent, (row0 + tid) / G, window, line);
#pragma unroll
        for (int w = 0; w < TREE_WORDS; ++w) lines[tid][w] = line[w];
    }
    __syncthreads();
    int lo[RW];
    float m[RW], l[RW], acc[RW][4 * NC];
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        lo[i] = window > 0 && i < nr ? max(0, sg.c + depths[r0 + i] - window + 1) : 0;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 4 * NC; ++c) acc[i][c] = 0.f;
    }
    int buf = 0;
    for (int j0 = j_begin; j0 < j_end; j0 += SKEYS, buf ^= 1) {
        asm volatile("cp.async.wait_group 0;\n" ::);
        __syncthreads();                                               // this tile is there, and the one before it has been used
        if (j0 + SKEYS < j_end) fetch(j0 + SKEYS, buf ^ 1);
        if (nr <= 0) continue;
        const float* ks = tiles + buf * 2 * SKEYS * pitch;
        const float* vs = ks + SKEYS * pitch;
        const int j = j0 + lane;
        float dot[RW];
#pragma unroll
        for (int i = 0; i < RW; ++i) dot[i] = 0.f;
        const float* kr = ks + lane * pitch;
        const float* qr = qs + r0 * pitch;
#pragma unroll 4
        for (int d = 0; d < D4; d += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                const float4 q4 = *reinterpret_cast<const float4*>(qr + i * pitch + d);
                dot[i] = fmaf(q4.x, k4.x, dot[i]);
                dot[i] = fmaf(q4.y, k4.y, dot[i]);
                dot[i] = fmaf(q4.z, k4.z, dot[i]);
                dot[i] = fmaf(q4.w, k4.w, dot[i]);
            }
        }
        float pj[RW];
        unsigned vis[RW];
        bool all = true;
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            vis[i] = 0u;
            pj[i] = 0.f;
            if (i >= nr) continue;
            const bool valid = j < j_end && (j < sg.c ? j >= lo[i] : (line_bits(lines[r0 + i], j0 - sg.c) >> lane) & 1u);
            vis[i] = __ballot_sync(0xffffffffu, valid);
            all = all && vis[i] == 0xffffffffu;
            if (vis[i] == 0u) continue;
            float s = -INFINITY;
            if (valid) {
                s = dot[i] * scale;
                if (softcap > 0.f) s = softcap * tanhf(s / softcap);
            }
            const float m_new = fmaxf(m[i], warp_max(s)), ref = m_new == -INFINITY ? 0.f : m_new;
            pj[i] = valid ? expf(s - ref) : 0.f;
            const float alpha = expf(m[i] - ref);                      // m = -inf on the first tile gives 0
            l[i] = l[i] * alpha + warp_sum(pj[i]);
#pragma unroll
            for (int c = 0; c < 4 * NC; ++c) acc[i][c] *= alpha;
            m[i] = m_new;
        }
#pragma unroll 4
        for (int jj = 0; jj < SKEYS; ++jj) {
            float4 v4[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c)
                v4[c] = 4 * lane + 128 * c < D4 ? *reinterpret_cast<const float4*>(vs + jj * pitch + 4 * lane + 128 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                const float p = __shfl_sync(0xffffffffu, pj[i], jj);
                if (!all && !((vis[i] >> jj) & 1u)) continue;          // uniform over the warp
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    acc[i][4 * c] = fmaf(p, v4[c].x, acc[i][4 * c]);
                    acc[i][4 * c + 1] = fmaf(p, v4[c].y, acc[i][4 * c + 1]);
                    acc[i][4 * c + 2] = fmaf(p, v4[c].z, acc[i][4 * c + 2]);
                    acc[i][4 * c + 3] = fmaf(p, v4[c].w, acc[i][4 * c + 3]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        if (i >= nr) continue;
        const int row = row0 + r0 + i, h = kvh * G + row % G;
        const size_t at = (size_t)(sg.q_begin + row / G) * Hq + h;
        if (sg.n_split > 1) {
            const size_t slot = (size_t)split * total_rows * Hq + at;
            if (lane == 0) {
                part_ml[2 * slot] = m[i] * LOG2E;                      // in units of log2, as the merge takes it
                part_ml[2 * slot + 1] = l[i];
            }
#pragma unroll
            for (int c = 0; c < 4 * NC; ++c) {
                const int d = 4 * lane + 128 * (c >> 2) + (c & 3);
                if (d < D) part_o[slot * D + d] = acc[i][c];
            }
        } else {
            if (sink != nullptr) l[i] += m[i] == -INFINITY ? 1.f : expf(sink[h] - m[i]);
            const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];
#pragma unroll
            for (int c = 0; c < 4 * NC; ++c) {
                const int d = 4 * lane + 128 * (c >> 2) + (c & 3);
                if (d < D) out[at * D + d] = from_f32<TA>(acc[i][c] * inv);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------- fifth-generation tensor cores
// bfloat16, head sizes 64 and 128.  A CTA (one an SM) owns rows of one segment and key/value head and walks its share of the keys in
// tiles of 64.  Two groups of four warps work side by side, so that one's waits pass while the other computes:
//   STREAMS        up to 128 rows: one query tile, the groups take the key tiles in turn, each with a maximum, sum and output of its own,
//                  joined at the end;
//   else           up to 256 rows: a query tile of 128 rows a group, both go through every key tile.
// Per key tile and group:
//   S = Q K^T      tcgen05.mma, M = 128, N = 64, in tensor memory, two buffers a group;
//   softmax        a row a thread (its TMEM lane), no shuffles; P rounded to bfloat16 into shared memory.  The reference maximum moves only
//                  when the true one has outrun it by 2^8, so O is rescaled in tensor memory a few times at most;
//   O += P V       tcgen05.mma, M = 128, N = head size, V as it lies in the cache.
// Warps: 8 of rows (those without rows have nothing to do, and nobody waits for them), for each group one that issues S and one that issues
// P V (an issuing thread pays some 230 cycles a wait and 60 to 90 an instruction, so two threads share that), one that gathers K and one
// that gathers V into the 128-byte swizzle, through rings of STAGES tiles: page by page with TMA where pages are 8, 16, 32 or a multiple of 64
// rows, else row by row with cp.async.
// Barriers: each ring stage has a full and an empty one; S, P and P V have one for each of two buffers.  A barrier's next phase always needs
// all of its waiters to have passed the current one, so no parity wait can fall two phases behind.
// A key tile that some row does not see in full is looked through for values that are no numbers before the products take it: they are
// set to zero there (zero times infinity would reach every row) and added to the rows that see them at the end.
using namespace tc5;

constexpr int QM = 128;                       // rows of a query tile
constexpr int KN = KEY_TILE;
constexpr float RESCALE_STEP = 8.0f;          // log2 units the true maximum may run ahead of the reference

template <int D, bool STREAMS> struct Shape {
    static constexpr int NQ = STREAMS ? 1 : 2;               // query tiles
    static constexpr int DS = D / 64;         // 64-wide slabs of the head size
    static constexpr unsigned Q_BYTES = DS * QM * 128, K_BYTES = DS * KN * 128, P_BYTES = QM * 128;
    static constexpr int STAGES = D == 128 ? (STREAMS ? 4 : 3) : (STREAMS ? 8 : 6);
    static constexpr int LAG = STAGES >= 4 ? 2 : 1;           // a tile is announced when this many later ones have been asked for
    static constexpr int THREADS = 32 * 14;
    static constexpr unsigned TMEM_COLS = 512, O_COL = 4 * KN;
    static constexpr int B_K_FULL = 0, B_V_FULL = STAGES, B_K_EMPTY = 2 * STAGES, B_V_EMPTY = 3 * STAGES, B_S = 4 * STAGES, B_P = B_S + 4,
                         B_PV = B_P + 4, B_Q = B_PV + 4, B_V_LAND = B_Q + 2, N_BARS = B_V_LAND + STAGES;
    static constexpr unsigned TAIL = N_BARS * 8 + 16 + TREE_MAX_NODES * 4;
    static constexpr unsigned SMEM_USED = NQ * Q_BYTES + 2 * STAGES * K_BYTES + 4 * P_BYTES + TAIL;
    static constexpr unsigned SMEM = SMEM_USED > 120 * 1024 ? SMEM_USED : 120 * 1024;       // one CTA an SM: it takes all of the tensor memory
    static_assert(SMEM <= 227 * 1024 && O_COL + 2 * D <= TMEM_COLS && STAGES > LAG, "a CTA's memories");
    static_assert(!STREAMS || STAGES % 2 == 0, "a ring stage belongs to one group, so that its barriers' phases come in turn");
};

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned long long pack2(float lo, float hi) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpack2(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ void cp16u(unsigned smem_addr, const void* gmem, bool pred) {
    const int bytes = pred ? 16 : 0;          // 0: nothing is read, the 16 bytes become zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_addr), "l"(gmem), "r"(bytes));
}
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
// tanh(x) = 1 - 2 / (e^(2x) + 1) with the hardware's 2^x and quotient: an absolute error of a few 1e-7.
__device__ __forceinline__ float fast_tanh(float x) { return 1.0f - __fdividef(2.0f, fast_exp2(x * (2.0f * LOG2E)) + 1.0f); }
// The halves of a word of two bfloat16 that are no finite numbers, as bits 15 and 31: an exponent of ones plus one carries into them.
__device__ __forceinline__ unsigned odd_halves(unsigned w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ unsigned long long below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

// Position -> (block, row in page): page sizes are powers of two in practice, any size works.
struct Paging {
    int page_size, shift;
    __device__ __forceinline__ explicit Paging(int p) : page_size(p), shift(-1) {
        if ((p & (p - 1)) == 0) shift = 31 - __clz(p);
    }
    __device__ __forceinline__ int block(int j) const { return shift >= 0 ? j >> shift : j / page_size; }
    __device__ __forceinline__ int row(int j) const { return shift >= 0 ? j & (page_size - 1) : j % page_size; }
};

// grid: (row blocks x kv heads, segments, splits).
template <int D, bool STREAMS>
__global__ void __launch_bounds__(Shape<D, STREAMS>::THREADS, 1)
tree_tc5_kernel(const bf16* __restrict__ q, int ld, const bf16* __restrict__ kpool, const bf16* __restrict__ vpool,
                const int* __restrict__ cu_q, const int* __restrict__ seg_pos0, const int* __restrict__ tree_parent,
                const int* __restrict__ block_table, int bt_stride, int page_size, bf16* __restrict__ out,
                float* __restrict__ part_o, float* __restrict__ part_ml, int total_rows, int Hq, int Hkv, float scale, int window,
                float softcap, const float* __restrict__ sink, int share, int* __restrict__ status, int by_tma,
                const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    typedef Shape<D, STREAMS> S;
    constexpr int STAGES = S::STAGES, NQ = S::NQ;
    // The swizzled tiles need 1024-byte alignment: the kernel has no static shared memory, so its window starts at the CTA's base.
    extern __shared__ __align__(1024) unsigned char tc5_smem[];
    if ((smem_u32(tc5_smem) & 1023u) != 0u) {
        if (threadIdx.x == 0) atomicExch(status, 2);
        return;
    }
    unsigned char* sQ = tc5_smem;                             // [query tile]
    unsigned char* sK = sQ + NQ * S::Q_BYTES;                 // [stage]
    unsigned char* sV = sK + STAGES * S::K_BYTES;             // [stage]
    unsigned char* sP = sV + STAGES * S::K_BYTES;             // [group][buffer]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(sP + 4 * S::P_BYTES);
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + S::N_BARS);
    volatile int* odd_values = reinterpret_cast<int*>(tmem_slot + 1);
    int* parent = reinterpret_cast<int*>(tmem_slot + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    const int seg = blockIdx.y, kvh = blockIdx.x % Hkv, row0 = blockIdx.x / Hkv * (NQ * QM), split = blockIdx.z, G = Hq / Hkv;
    const Segment sg(cu_q, seg_pos0, seg, window, share, gridDim.z);
    const int rows = min(NQ * QM, sg.n * G - row0);
    if (rows <= 0 || split >= sg.n_split) return;
    const int t0 = share > 0 ? split * share : 0, t1 = share > 0 && split + 1 < sg.n_split ? t0 + share : sg.tiles;
    const int jt_begin = sg.jt0 + t0, n_tiles = t1 - t0;      // one tile at least
    const int* bt_row = block_table + (size_t)seg * bt_stride;
    const Paging pg(page_size);
    const unsigned bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    // a group's rows (as warps), its key tiles, and the number of its i-th among the CTA's
    auto active_warps = [&](int g) { return max(0, min(4, (rows - (STREAMS ? 0 : g * QM) + 31) >> 5)); };
    auto tiles_of = [&](int g) { return STREAMS ? (n_tiles - g + 1) >> 1 : active_warps(g) > 0 ? n_tiles : 0; };
    auto tile_no = [&](int g, int i) { return STREAMS ? 2 * i + g : i; };
    // whether every row sees every key of a tile
    auto whole = [&](int j_base) { return j_base + KN - 1 < sg.c && (window <= 0 || j_base > sg.c + sg.n - 1 - window); };

    if (warp == 8) tmem_alloc(smem_u32(tmem_slot), S::TMEM_COLS);
    if (tid == 0) {
        for (int i = 0; i < S::N_BARS; ++i) {
            int count = 1;
            if (i >= S::B_K_EMPTY && i < S::B_S) count = !STREAMS && rows > QM ? 2 : 1;       // the groups that read a key tile
            else if (i >= S::B_P && i < S::B_PV) count = max(1, active_warps((i - S::B_P) >> 1));
            else if (i >= S::B_Q && i < S::B_V_LAND) count = max(1, active_warps(i - S::B_Q));
            mbar_init(bar(i), count);
        }
        mbar_init_fence();
        *odd_values = 0;
    }
    for (int i = tid; i < sg.n; i += S::THREADS) parent[i] = tree_parent[sg.q_begin + i];
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const unsigned tmem = *tmem_slot;
    bool ok = true;

    constexpr int LPR = D / 8, RPI = 32 / LPR;                // lanes a row of 16-byte pieces, rows an instruction
    const int rsel = lane / LPR, sub = lane % LPR;
    const int grp = warp < 8 ? warp >> 2 : ((warp - 8) >> 1) & 1;              // group of a row warp or an issuer
    const int qt = STREAMS ? 0 : grp, n_mine = tiles_of(grp);
    const bool has_rows = warp < 8 && (warp & 3) < active_warps(grp);
    const int r = (warp & 3) * 32 + lane, row = row0 + qt * QM + r;            // a row thread's row of the tile, of the segment and head
    const bool row_valid = has_rows && row - row0 < rows;
    const size_t token = (size_t)sg.q_begin + (row_valid ? row / G : 0);
    const int h = kvh * G + (row_valid ? row % G : 0);
    const float scale_log2 = scale * LOG2E, scale_eff = softcap > 0.f ? softcap * LOG2E : scale_log2;
    unsigned line[TREE_WORDS];
    int lo_r = 0;
    float m_ref = -INFINITY, l_run = 0.f;                     // the reference maximum and the sum relative to it
    // the keys of tile j_base that this row sees, as bits
    auto visible = [&](int j_base) {
        const int at = j_base - sg.c;
        const unsigned long long nodes = (unsigned long long)line_bits(line, at) | ((unsigned long long)line_bits(line, at + 32) << 32);
        return (below(sg.c - j_base) & ~below(lo_r - j_base)) | nodes;
    };
    const unsigned lane_addr = tmem + ((unsigned)((warp & 3) * 32) << 16);
    const unsigned o_addr = lane_addr + S::O_COL + grp * D;
    // a row's maximum and sum of a group, in that group's P, which none of its products reads any more by then
    auto joined = [&](int g) { return reinterpret_cast<float2*>(sP + g * 2 * S::P_BYTES) + r; };

    if (has_rows) {
        // ================================================================== one row per thread
        if (!STREAMS || grp == 0) {
            unsigned char* tile = sQ + qt * S::Q_BYTES + (unsigned)(sub >> 3) * (QM * 128);
#pragma unroll 1
            for (int i = 0; i < 32 / RPI; ++i) {              // a row's pieces by neighbouring lanes
                const int rt = (warp & 3) * 32 + i * RPI + rsel, rr = row0 + qt * QM + rt;
                const bool there = rr - row0 < rows;
                const bf16* src = q + (there ? (size_t)(sg.q_begin + rr / G) * ld + (size_t)(kvh * G + rr % G) * D + sub * 8 : 0);
                cp16u(smem_u32(tile + sw128_offset(rt, sub & 7)), src, there);
            }
            asm volatile("cp.async.commit_group;\n" ::);
        }
        const int depth = tree_line(parent, row_valid ? row / G : 0, window, line);
        lo_r = window > 0 ? max(0, sg.c + depth - window + 1) : 0;
        if (!STREAMS || grp == 0) {
            cp_wait<0>();
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(S::B_Q + qt));
        }
        unsigned char* myPs = sP + grp * 2 * S::P_BYTES;
        for (int i = 0; i < n_mine; ++i) {
            const int j_base = (jt_begin + tile_no(grp, i)) * KN, buf = i & 1;
            ok = mbar_wait(bar(S::B_S + grp * 2 + buf), (i >> 1) & 1) && ok;
            fence_after_sync();
            unsigned a[64];
            tmem_ld32(lane_addr + (grp * 2 + buf) * KN, reinterpret_cast<unsigned(&)[32]>(a[0]));
            tmem_ld32(lane_addr + (grp * 2 + buf) * KN + 32, reinterpret_cast<unsigned(&)[32]>(a[32]));
            tmem_ld_wait();
            if (softcap > 0.f) {
                const float k = scale / softcap;
#pragma unroll
                for (int e = 0; e < 64; ++e) a[e] = __float_as_uint(fast_tanh(__uint_as_float(a[e]) * k));
            }
            float mx = -INFINITY;
            if (whole(j_base)) {
#pragma unroll
                for (int e = 0; e < 64; e += 2) mx = max3(mx, __uint_as_float(a[e]), __uint_as_float(a[e + 1]));
            } else {
                const unsigned long long vis = visible(j_base);
                const unsigned vis_lo = (unsigned)vis, vis_hi = (unsigned)(vis >> 32);
#pragma unroll
                for (int e = 0; e < 64; ++e) {
                    if (!((e < 32 ? vis_lo : vis_hi) & (1u << (e & 31)))) a[e] = 0xff800000u;
                    mx = fmaxf(mx, __uint_as_float(a[e]));
                }
            }
            mx *= scale_eff;                                  // the scale is positive
            float alpha = 1.f;
            bool moved = false;
            if (mx > m_ref + RESCALE_STEP || (m_ref == -INFINITY && mx != -INFINITY)) {
                alpha = fast_exp2(m_ref - mx);                // 0 on the first move
                m_ref = mx;
                moved = true;
            }
            const float mu = m_ref == -INFINITY ? 0.f : m_ref;
            // P(i) goes into the buffer that P V(i - 2) read; O is touched only when P V(i - 1) is done
            if (i > 1) ok = mbar_wait(bar(S::B_PV + grp * 2 + buf), ((i - 2) >> 1) & 1) && ok;
            if (i > 0 && __any_sync(0xffffffffu, moved)) {
                ok = mbar_wait(bar(S::B_PV + grp * 2 + (buf ^ 1)), ((i - 1) >> 1) & 1) && ok;
                fence_after_sync();
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    unsigned o[32];
                    tmem_ld32(o_addr + c0, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                    tmem_st32(o_addr + c0, o);
                }
                tmem_st_wait();
            }
            unsigned char* myP = myPs + buf * S::P_BYTES;
            const unsigned long long scale2 = pack2(scale_eff, scale_eff), shift2 = pack2(-mu, -mu);
            unsigned long long sum2 = pack2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
                float x0, x1;
                unpack2(fma2(pack2(__uint_as_float(a[e]), __uint_as_float(a[e + 1])), scale2, shift2), x0, x1);
                const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                sum2 = add2(sum2, pack2(p0, p1));
                a[e] = __float_as_uint(p0);
                a[e + 1] = __float_as_uint(p1);
            }
            float sum_lo, sum_hi;
            unpack2(sum2, sum_lo, sum_hi);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                uint4 v;
                v.x = pack_bf16(__uint_as_float(a[8 * c]), __uint_as_float(a[8 * c + 1]));
                v.y = pack_bf16(__uint_as_float(a[8 * c + 2]), __uint_as_float(a[8 * c + 3]));
                v.z = pack_bf16(__uint_as_float(a[8 * c + 4]), __uint_as_float(a[8 * c + 5]));
                v.w = pack_bf16(__uint_as_float(a[8 * c + 6]), __uint_as_float(a[8 * c + 7]));
                *reinterpret_cast<uint4*>(myP + sw128_offset(r, c)) = v;
            }
            l_run = l_run * alpha + (sum_lo + sum_hi);
            fence_proxy_async();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(S::B_P + grp * 2 + buf));           // S(i) is read, O is rescaled, P(i) is written
        }
        if (n_mine > 0) ok = mbar_wait(bar(S::B_PV + grp * 2 + ((n_mine - 1) & 1)), ((n_mine - 1) >> 1) & 1) && ok;
    } else if (warp >= 8 && warp < 12 && n_mine > 0 && lane == 0) {
        // ================================================================== an issuing thread: descriptors are a base plus a constant
        ok = mbar_wait(bar(S::B_Q + qt), 0) && ok;
        fence_after_sync();
        if ((warp & 1) == 0) {                                // S
            const unsigned idesc = instr_desc_bf16(QM, KN, false);
            const unsigned long long dQ = smem_desc_sw128(smem_u32(sQ) + qt * S::Q_BYTES, 0), dK = smem_desc_sw128(smem_u32(sK), 0);
            for (int i = 0; i < n_mine; ++i) {
                const int t = tile_no(grp, i), st = t % STAGES;
                ok = mbar_wait(bar(S::B_K_FULL + st), (t / STAGES) & 1) && ok;
                if (i > 1) ok = mbar_wait(bar(S::B_P + grp * 2 + (i & 1)), ((i - 2) >> 1) & 1) && ok;     // the rows have read S(i - 2)
                fence_after_sync();
                const unsigned long long k_tile = dK + (unsigned long long)(st * (S::K_BYTES >> 4));
                const unsigned d_s = tmem + (grp * 2 + (i & 1)) * KN;
#pragma unroll
                for (int d16 = 0; d16 < D / 16; ++d16)        // 64-wide slabs of the head size, four steps of 16 (32 bytes) in each
                    mma_ss(d_s, dQ + (unsigned long long)(((d16 >> 2) * (QM * 128) + (d16 & 3) * 32) >> 4),
                           k_tile + (unsigned long long)(((d16 >> 2) * (KN * 128) + (d16 & 3) * 32) >> 4), idesc, d16 > 0);
                mma_commit(bar(S::B_S + grp * 2 + (i & 1)));
                mma_commit(bar(S::B_K_EMPTY + st));
            }
        } else {                                              // P V
            const unsigned idesc = instr_desc_bf16(QM, D, true);
            const unsigned long long dP = smem_desc_sw128(smem_u32(sP) + grp * 2 * S::P_BYTES, 0);
            const unsigned long long dV = smem_desc_sw128_mn(smem_u32(sV), KN * 128, 1024u);
            const unsigned d_o = tmem + S::O_COL + grp * D;
            for (int i = 0; i < n_mine; ++i) {
                const int t = tile_no(grp, i), st = t % STAGES;
                ok = mbar_wait(bar(S::B_V_FULL + st), (t / STAGES) & 1) && ok;
                ok = mbar_wait(bar(S::B_P + grp * 2 + (i & 1)), (i >> 1) & 1) && ok;
                fence_after_sync();
                const unsigned long long v_tile = dV + (unsigned long long)(st * (S::K_BYTES >> 4)), p_tile = dP + (unsigned long long)((i & 1) * (S::P_BYTES >> 4));
#pragma unroll
                for (int k16 = 0; k16 < KN / 16; ++k16)       // 16 keys: 32 bytes along P's rows, 2048 bytes down V's
                    mma_ss(d_o, p_tile + (unsigned long long)(k16 * 2), v_tile + (unsigned long long)(k16 * 128), idesc, i > 0 || k16 > 0);
                mma_commit(bar(S::B_PV + grp * 2 + (i & 1)));
                mma_commit(bar(S::B_V_EMPTY + st));
            }
        }
    } else if (warp >= 12) {
        // ================================================================== the loaders
        const bool is_k = warp == 12;
        const bf16* pool = is_k ? kpool : vpool;
        unsigned char* ring = is_k ? sK : sV;
        const int b_full = is_k ? S::B_K_FULL : S::B_V_FULL, b_empty = is_k ? S::B_K_EMPTY : S::B_V_EMPTY;
        // Values of a tile that has landed and that some row does not see in full: rows of no key of this CTA become zero, and so do
        // values that are no numbers, which are noted.
        auto clean = [&](int t) {
            uint4* piece = reinterpret_cast<uint4*>(ring + (t % STAGES) * S::K_BYTES);
            const int j_base = (jt_begin + t) * KN;
            bool odd = false;
#pragma unroll 4
            for (int i = lane; i < (int)(S::K_BYTES / 16); i += 32) {
                uint4 v = piece[i];
                const int j = j_base + ((i >> 3) & (KN - 1));         // 8 pieces a row of 128 bytes, KN rows a slab
                const unsigned x = odd_halves(v.x), y = odd_halves(v.y), z = odd_halves(v.z), w = odd_halves(v.w);
                if (j < sg.lo || j > sg.hi) {
                    piece[i] = make_uint4(0u, 0u, 0u, 0u);
                } else if (x | y | z | w) {
                    odd = true;
                    v.x &= ~((x >> 15) * 0xffffu); v.y &= ~((y >> 15) * 0xffffu);
                    v.z &= ~((z >> 15) * 0xffffu); v.w &= ~((w >> 15) * 0xffffu);
                    piece[i] = v;
                }
            }
            if (odd) *odd_values = 1;
        };
        if (by_tma) {
            // A lane for each (page of the tile, slab): it knows the page one tile ahead and asks for its box.  A whole tile's bytes are counted
            // on the barrier that its product waits for; values that have to be looked through first land on a barrier of the loader's.
            const CUtensorMap* map = is_k ? &kmap : &vmap;
            const int box = min(pg.page_size, KN), pi = lane / S::DS, slab = lane % S::DS;
            const bool mine = pi * box < KN;
            auto in_sight = [&](int jt) { const int j = jt * KN + pi * box; return mine && j + box > sg.lo && j <= sg.hi; };
            auto ask_page = [&](int jt) { return in_sight(jt) ? bt_row[pg.block(jt * KN + pi * box)] : -1; };
            unsigned land_par = 0u;                           // the parity of each stage's next landing
            auto finish = [&](int t) {                        // values of tile t, which was not whole, have landed
                const int st = t % STAGES;
                if (whole((jt_begin + t) * KN)) return;
                ok = mbar_wait(bar(S::B_V_LAND + st), (land_par >> st) & 1u) && ok;
                land_par ^= 1u << st;
                clean(t);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(S::B_V_FULL + st));
            };
            int next = ask_page(jt_begin);
            for (int t = 0; t < n_tiles; ++t) {
                const int st = t % STAGES, page = next;
                if (t >= STAGES) ok = mbar_wait(bar(b_empty + st), (t / STAGES - 1) & 1) && ok;
                const unsigned dst = smem_u32(ring) + st * S::K_BYTES + slab * (KN * 128) + pi * box * 128;
                const unsigned boxes = __popc(__ballot_sync(0xffffffffu, page >= 0));
                const bool gone = in_sight(jt_begin + t) && page < 0;
                if (__any_sync(0xffffffffu, gone)) {          // a block that is marked as gone reads as zero
                    if (gone)
                        for (int i = 0; i < box * 8; ++i) reinterpret_cast<uint4*>(ring + (dst - smem_u32(ring)))[i] = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async();
                    __syncwarp();
                }
                const unsigned land = bar(is_k || whole((jt_begin + t) * KN) ? b_full + st : S::B_V_LAND + st);
                if (lane == 0) mbar_arrive_expect_tx(land, boxes * (unsigned)(box * 128));
                __syncwarp();
                if (page >= 0) tma::load_2d(dst, map, slab * 64, (page * Hkv + kvh) * pg.page_size + pg.row((jt_begin + t) * KN + pi * box), land);
                if (t + 1 < n_tiles) next = ask_page(jt_begin + t + 1);
                if (!is_k && t >= S::LAG) finish(t - S::LAG);
            }
            if (!is_k)
                for (int t = max(0, n_tiles - S::LAG); t < n_tiles; ++t) finish(t);
        } else {
            // The pages of rows `lane` and `lane + 32` of a tile are asked for one tile ahead.
            auto ask_pages = [&](int jt, int (&page)[2]) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int j = jt * KN + u * 32 + lane;
                    page[u] = j >= sg.lo && j <= sg.hi ? bt_row[pg.block(j)] : -1;
                }
            };
            auto announce = [&](int t) {                      // tile t has landed
                if (!is_k && !whole((jt_begin + t) * KN)) {
                    __syncwarp();
                    clean(t);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(b_full + t % STAGES));
            };
            int next_page[2];
            ask_pages(jt_begin, next_page);
            for (int t = 0; t < n_tiles; ++t) {
                const int st = t % STAGES;
                if (t >= STAGES) ok = mbar_wait(bar(b_empty + st), (t / STAGES - 1) & 1) && ok;
                const unsigned tile_smem = smem_u32(ring) + st * S::K_BYTES;
                // Lane L knows where rows L and L + 32 lie (0: not to be read); D / 8 neighbouring lanes then copy one row, so that an
                // instruction reads whole lines.
                unsigned long long where[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    where[u] = next_page[u] < 0 ? 0ull : reinterpret_cast<unsigned long long>(
                        pool + (((size_t)next_page[u] * Hkv + kvh) * pg.page_size + pg.row((jt_begin + t) * KN + u * 32 + lane)) * D);
                const unsigned slab = (unsigned)(sub >> 3) * (KN * 128), c7 = (unsigned)(sub & 7);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int i = 0; i < 32 / RPI; ++i) {
                        const int owner = i * RPI + rsel, krow = u * 32 + owner;
                        const unsigned long long w = __shfl_sync(0xffffffffu, where[u], owner);
                        const bf16* src = w ? reinterpret_cast<const bf16*>(w) + sub * 8 : pool;
                        cp16u(tile_smem + (krow >> 3) * 1024 + (krow & 7) * 128 + slab + ((c7 ^ (unsigned)(krow & 7)) << 4), src, w != 0ull);
                    }
                }
                asm volatile("cp.async.commit_group;\n" ::);
                if (t + 1 < n_tiles) ask_pages(jt_begin + t + 1, next_page);
                if (t >= S::LAG) {
                    cp_wait<S::LAG>();
                    announce(t - S::LAG);
                }
            }
            cp_wait<0>();
            for (int t = max(0, n_tiles - S::LAG); t < n_tiles; ++t) announce(t);
        }
    }
    if (STREAMS && has_rows) *joined(grp) = make_float2(m_ref, l_run);
    pdl_trigger_late();
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (has_rows) {
        // The rows leave: the finished ones, or O as it stands with the reference maximum and the sum.  Streams are joined first, either group
        // for half of the columns.
        const bool odd = *odd_values != 0, part = sg.n_split > 1;
        const size_t at = token * Hq + h, slot = (size_t)split * total_rows * Hq + at;
        float w_a = 1.f, w_b = 0.f;
        if (STREAMS && n_tiles > 1) {
            const float2 a = *joined(0), b = *joined(1);
            m_ref = fmaxf(a.x, b.x);
            const float top = m_ref == -INFINITY ? 0.f : m_ref;
            w_a = fast_exp2(a.x - top);
            w_b = fast_exp2(b.x - top);
            l_run = a.y * w_a + b.y * w_b;
        } else if (STREAMS) {
            const float2 a = *joined(0);
            m_ref = a.x;
            l_run = a.y;
        }
        const float mu = m_ref == -INFINITY ? 0.f : m_ref;
        if (part && row_valid && (!STREAMS || grp == 0)) {
            part_ml[2 * slot] = m_ref;
            part_ml[2 * slot + 1] = l_run;
        }
        float l_all = l_run;
        if (sink != nullptr && !part) l_all += exp2f(sink[h] * LOG2E - mu);
        const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
        const unsigned o_first = lane_addr + S::O_COL + (STREAMS ? 0 : grp * D);
#pragma unroll 1
        for (int c0 = STREAMS ? grp * (D / 2) : 0; c0 < (STREAMS ? (grp + 1) * (D / 2) : D); c0 += 32) {
            unsigned o[32];
            __syncwarp();
            tmem_ld32(o_first + c0, o);
            if (STREAMS && n_tiles > 1) {
                unsigned o_b[32];
                tmem_ld32(o_first + D + c0, o_b);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(__uint_as_float(o[i]), w_a, __uint_as_float(o_b[i]) * w_b));
            } else {
                tmem_ld_wait();
            }
            if (odd && row_valid) {
                // what the products left out: values that are no numbers, where this row sees their keys
                for (int t = 0; t < n_tiles; ++t) {
                    const int j_base = (jt_begin + t) * KN;
                    if (whole(j_base)) continue;
                    for (unsigned long long vis = visible(j_base); vis != 0ull; vis &= vis - 1ull) {
                        const int j = j_base + __ffsll((long long)vis) - 1, page = bt_row[pg.block(j)];
                        if (page < 0) continue;
                        const size_t key = (((size_t)page * Hkv + kvh) * pg.page_size + pg.row(j)) * D;
                        unsigned any = 0u;
#pragma unroll
                        for (int i = 0; i < 32; i += 2) any |= odd_halves(*reinterpret_cast<const unsigned*>(vpool + key + c0 + i));
                        if (any == 0u) continue;
                        float s = 0.f;
                        const bf16* qrow = q + token * ld + (size_t)h * D;
                        for (int d = 0; d < D; ++d) s = fmaf(__bfloat162float(qrow[d]), __bfloat162float(kpool[key + d]), s);
                        s = softcap > 0.f ? fast_tanh(s * (scale / softcap)) : s;
                        const float p = fast_exp2(fmaf(s, scale_eff, -mu));
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float v = __bfloat162float(vpool[key + c0 + i]);
                            if (!isfinite(v)) o[i] = __float_as_uint(fmaf(p, v, __uint_as_float(o[i])));
                        }
                    }
                }
            }
            if (part && row_valid) {
                float4* to = reinterpret_cast<float4*>(part_o + slot * D + c0);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    to[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
            } else if (row_valid) {
                uint4* to = reinterpret_cast<uint4*>(out + at * D + c0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint4 v;
                    v.x = pack_bf16(__uint_as_float(o[8 * i]) * inv, __uint_as_float(o[8 * i + 1]) * inv);
                    v.y = pack_bf16(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv);
                    v.z = pack_bf16(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv);
                    v.w = pack_bf16(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv);
                    to[i] = v;
                }
            }
        }
    }
    if (!ok) atomicExch(status, 1);
    fence_before_sync();
    __syncthreads();
    if (warp == 8) tmem_dealloc(tmem, S::TMEM_COLS);
}

// out[row, h] = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the shares of the keys, in their order: one warp a (node, head).
// grid: (nodes of the longest tree x Hq / 8, segments).
template <typename TA>
__global__ void __launch_bounds__(256)
tree_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ cu_q,
                  const int* __restrict__ seg_pos0, int total_rows, int Hq, int D, int window, int share, int max_split,
                  TA* __restrict__ out, const float* __restrict__ sink) {
    pdl_wait();
    const Segment sg(cu_q, seg_pos0, blockIdx.y, window, share, max_split);
    const int pair = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (pair >= sg.n * Hq || sg.n_split == 1) return;         // one share: its CTA wrote the row
    const int h = pair % Hq;
    const size_t at = (size_t)sg.q_begin * Hq + pair, stride = (size_t)total_rows * Hq;
    float top = -INFINITY;
    for (int s = 0; s < sg.n_split; ++s) top = fmaxf(top, part_ml[2 * (s * stride + at)]);
    const float ref = top == -INFINITY ? 0.f : top;
    float l = sink != nullptr ? exp2f(sink[h] * LOG2E - ref) : 0.f;
    float acc[TREE_MAX_D / 32];
#pragma unroll
    for (int i = 0; i < TREE_MAX_D / 32; ++i) acc[i] = 0.f;
    for (int s = 0; s < sg.n_split; ++s) {
        const size_t slot = s * stride + at;
        const float ls = part_ml[2 * slot + 1];
        if (ls == 0.f) continue;                              // a share without keys for this row left no output
        const float w = exp2f(part_ml[2 * slot] - ref);
        l += ls * w;
#pragma unroll
        for (int i = 0; i < TREE_MAX_D / 32; ++i) {
            const int d = lane + 32 * i;
            if (d < D) acc[i] += part_o[slot * D + d] * w;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < TREE_MAX_D / 32; ++i) {
        const int d = lane + 32 * i;
        if (d < D) out[at * D + d] = from_f32<TA>(acc[i] * inv);
    }
}

struct TreeCall {
    const void *q, *kpool, *vpool;
    int ld;
    const int *cu_q, *seg_pos0, *parent, *block_table;
    int bt_stride, page_size;
    void* out;
    int segments, max_nodes, total_rows, Hq, Hkv, D, pages;
    float scale;
    int window;
    float softcap;
    const float* sink;
    int splits, share;
    float* scratch;
    int* status;
    cudaStream_t st;
    float* part_ml() const { return splits > 1 ? scratch + (size_t)splits * total_rows * Hq * D : nullptr; }
};

template <typename TA>
int merge(const TreeCall& a) {
    if (a.splits <= 1) return 0;
    dim3 grid((a.max_nodes * a.Hq + 7) / 8, a.segments);
    return rb_launch_pdl(tree_merge_kernel<TA>, grid, dim3(256), 0, a.st, a.scratch, a.part_ml(), a.cu_q, a.seg_pos0, a.total_rows, a.Hq, a.D,
                         a.window, a.share, a.splits, (TA*)a.out, a.sink);
}

template <typename TA, int NC>
int simt(const TreeCall& a) {
    const size_t smem = (size_t)(SROWS + 4 * SKEYS) * (((a.D + 3) & ~3) + 4) * sizeof(float);
    static PerDevice configured;
    const int rc = configured.once([&](int) {
        return cudaFuncSetAttribute(tree_simt_kernel<TA, NC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)((SROWS + 4 * SKEYS) * (128 * NC + 4) * sizeof(float)));
    });
    if (rc) return rc;
    const int vec = sizeof(TA) == 4 && a.D % 4 == 0 && (((uintptr_t)a.kpool | (uintptr_t)a.vpool) & 15) == 0;
    dim3 grid((a.max_nodes * (a.Hq / a.Hkv) + SROWS - 1) / SROWS * a.Hkv, a.segments, a.splits);
    tree_simt_kernel<TA, NC><<<grid, 32 * SW, smem, a.st>>>(
        (const TA*)a.q, a.ld, (const TA*)a.kpool, (const TA*)a.vpool, a.cu_q, a.seg_pos0, a.parent, a.block_table, a.bt_stride, a.page_size,
        (TA*)a.out, a.scratch, a.part_ml(), a.total_rows, a.Hq, a.Hkv, a.D, a.scale, a.window, a.softcap, a.sink, a.splits > 1 ? a.share : 0, vec);
    const int e = rb_launch_status();
    return e ? e : merge<TA>(a);
}

template <int D, bool STREAMS>
int tc5_launch(const TreeCall& a) {
    typedef Shape<D, STREAMS> S;
    constexpr int ROWS = S::NQ * QM;
    static PerDevice configured;
    const int rc = configured.once([&](int) {
        return cudaFuncSetAttribute(tree_tc5_kernel<D, STREAMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
    });
    if (rc) return rc;
    // pages are whole boxes of whole groups of eight rows, and their rows can be counted in 31 bits
    const long long pool_rows = (long long)a.pages * a.Hkv * a.page_size;
    int by_tma = a.page_size % 8 == 0 && (KN % a.page_size == 0 || a.page_size % KN == 0) && pool_rows <= 0x7fffffffll;
    CUtensorMap kmap = {}, vmap = {};
    const int box = a.page_size < KN ? a.page_size : KN;
    if (by_tma && !(tma::make_map_bf16(&kmap, a.kpool, (int)pool_rows, D, D, box) && tma::make_map_bf16(&vmap, a.vpool, (int)pool_rows, D, D, box)))
        return (int)cudaErrorInvalidValue;
    dim3 grid((a.max_nodes * (a.Hq / a.Hkv) + ROWS - 1) / ROWS * a.Hkv, a.segments, a.splits);
    const int e = rb_launch_pdl(tree_tc5_kernel<D, STREAMS>, grid, dim3(S::THREADS), S::SMEM, a.st, (const bf16*)a.q, a.ld, (const bf16*)a.kpool,
                                (const bf16*)a.vpool, a.cu_q, a.seg_pos0, a.parent, a.block_table, a.bt_stride, a.page_size, (bf16*)a.out, a.scratch,
                                a.part_ml(), a.total_rows, a.Hq, a.Hkv, a.scale, a.window, a.softcap, a.sink, a.splits > 1 ? a.share : 0, a.status, by_tma, kmap, vmap);
    return e ? e : merge<bf16>(a);
}

}  // namespace

RB_EXPORT int rb_tree_max_nodes() { return TREE_MAX_NODES; }

// q: rotated queries, row stride ld.  max_nodes: the longest segment's nodes (TREE_MAX_NODES at most).  splits > 1: a segment's keys
// go to one CTA for every `share` key tiles of 64, `splits` at most; scratch then holds splits * total_rows * Hq * (D + 2) floats.
// query_tiles: 0 the CUDA cores; 1 or 2 the tensor cores with so many tiles of 128 rows a CTA (bfloat16, D 64 or 128, pools and
// queries on 16-byte boundaries, ld a multiple of 8).  *status is raised if a wait gave up.
RB_EXPORT int rb_tree_attention(const void* q, int ld, const void* kpool, const void* vpool, const int* cu_q, const int* seg_pos0,
                                const int* parent, const int* block_table, int bt_stride, int page_size, int pages, void* out, int act_dtype,
                                int segments, int max_nodes, int total_rows, int Hq, int Hkv, int D, float scale, int window,
                                float softcap, const float* sink, int splits, int share, void* scratch, int query_tiles, int* status,
                                cudaStream_t st) {
    if (segments <= 0 || max_nodes <= 0) return 0;
    if (segments > 65535 || max_nodes > TREE_MAX_NODES || D <= 0 || D > TREE_MAX_D || Hkv <= 0 || Hq % Hkv || page_size <= 0) return (int)cudaErrorInvalidValue;
    if (splits < 1 || splits > 64 || (splits > 1 && (share <= 0 || scratch == nullptr))) return (int)cudaErrorInvalidValue;
    TreeCall a = {q, kpool, vpool, ld, cu_q, seg_pos0, parent, block_table, bt_stride, page_size, out, segments, max_nodes, total_rows, Hq, Hkv,
                  D, pages, scale, window, softcap, sink, splits, share, (float*)scratch, status, st};
    if (query_tiles > 0) {
        if (act_dtype != RB_BF16 || (D != 64 && D != 128) || query_tiles > 2 || status == nullptr) return (int)cudaErrorInvalidValue;
        if ((((uintptr_t)q | (uintptr_t)kpool | (uintptr_t)vpool | (uintptr_t)out) & 15) || ld % 8) return (int)cudaErrorInvalidValue;
        if (D == 64) return query_tiles == 1 ? tc5_launch<64, true>(a) : tc5_launch<64, false>(a);
        return query_tiles == 1 ? tc5_launch<128, true>(a) : tc5_launch<128, false>(a);
    }
    if (act_dtype == RB_F32) return D <= 128 ? simt<float, 1>(a) : simt<float, 2>(a);
    return D <= 128 ? simt<bf16, 1>(a) : simt<bf16, 2>(a);
}
