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
#include "common.cuh"

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
    int segments, max_nodes, total_rows, Hq, Hkv, D;
    float scale;
    int window;
    float softcap;
    const float* sink;
    int splits, share;
    float* scratch;
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

}  // namespace

RB_EXPORT int rb_tree_max_nodes() { return TREE_MAX_NODES; }

// q: rotated queries, row stride ld.  max_nodes: the longest segment's nodes (TREE_MAX_NODES at most).  splits > 1: a segment's keys
// go to one CTA for every `share` key tiles of 64, `splits` at most; scratch then holds splits * total_rows * Hq * (D + 2) floats.
RB_EXPORT int rb_tree_attention(const void* q, int ld, const void* kpool, const void* vpool, const int* cu_q, const int* seg_pos0,
                                const int* parent, const int* block_table, int bt_stride, int page_size, void* out, int act_dtype,
                                int segments, int max_nodes, int total_rows, int Hq, int Hkv, int D, float scale, int window,
                                float softcap, const float* sink, int splits, int share, void* scratch, cudaStream_t st) {
    if (segments <= 0 || max_nodes <= 0) return 0;
    if (segments > 65535 || max_nodes > TREE_MAX_NODES || D <= 0 || D > TREE_MAX_D || Hkv <= 0 || Hq % Hkv || page_size <= 0) return (int)cudaErrorInvalidValue;
    if (splits < 1 || splits > 64 || (splits > 1 && (share <= 0 || scratch == nullptr))) return (int)cudaErrorInvalidValue;
    TreeCall a = {q, kpool, vpool, ld, cu_q, seg_pos0, parent, block_table, bt_stride, page_size, out, segments, max_nodes, total_rows, Hq, Hkv,
                  D, scale, window, softcap, sink, splits, share, (float*)scratch, st};
    if (act_dtype == RB_F32) return D <= 128 ? simt<float, 1>(a) : simt<float, 2>(a);
    return D <= 128 ? simt<bf16, 1>(a) : simt<bf16, 2>(a);
}
