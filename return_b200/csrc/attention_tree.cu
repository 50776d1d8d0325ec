// Attention of drafted trees over the paged cache: the step that checks several continuations of a request at once.
//
// A segment brings n nodes, its tree: parent[i] < i is the node before node i, the root (node 0 as a rule; any node with parent < 0) is
// the first token behind the segment's c cached ones.  The keys and values of node i already lie in slot c + i of the request's
// pages; its position is c + depth(i).  Node i sees the cached keys j < c, and of the tree itself and its ancestors.  With a
// window both must lie less than `window` positions back: j > c + depth(i) - window, depth(i) - depth(a) < window.
//   s = scale q.k   (softcap > 0: softcap tanh(s / softcap))
//   out = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink[h] - m))
// A block that the table marks as gone (-1), or whose page the pool does not have, reads as keys and values of zero; a row that sees no key
// gets zeros.
//
// Which ancestors a node has is not read from a mask: a thread walks up its parents once (the list of a segment, at most
// TREE_MAX_NODES, is in shared memory) and keeps the bits.  A parent that is not below its child ends the walk, so a list that is no
// tree gives some mask, never a hang or a read out of range.
//
// Rows are (node, query head) pairs that share a key/value head, G = Hq / Hkv heads a node: row r is node r / G, head r % G.  The
// keys of a segment are split over CTAs, one for every `share` key tiles (0: one CTA walks them all); each leaves its unnormalised
// output, maximum and sum in float32, and they are joined in the order of the shares: up to JOIN_MAX shares can be a cluster and join them
// through shared memory, others leave them in memory for tree_merge_kernel.  So the result depends on `share`, which the host works
// out from the step's lengths, and on nothing else of the launch.
#include "pairs.cuh"
#include "tc5.cuh"
#include "tma.cuh"

#define TREE_MAX_NODES 256
#define TREE_WORDS (TREE_MAX_NODES / 32)
#define TREE_MAX_D 256
#define TREE_MAX_SPLITS 64

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KEY_TILE = 64;                  // the unit of `share`

// Up to so many shares of a segment's keys can be a cluster, whose CTAs join their outputs through each other's shared memory.
constexpr int JOIN_MAX = 8;
__device__ __forceinline__ float4 peer_float4(unsigned at) {
    float4 f;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(at));
    return f;
}
__device__ __forceinline__ float2 peer_float2(unsigned at) {
    float2 f;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(at));
    return f;
}

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

// A block table's entry: the page, -1 where there is none.
__device__ __forceinline__ int page_at(const int* entry, int pages) {
    const int page = *entry;
    return (unsigned)page < (unsigned)pages ? page : -1;
}

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

// ---------------------------------------------------------------------------------------- matrix instructions of a warp, any type and head size
// A CTA of eight warps takes 32 rows and walks its keys in tiles of 64.  Scores: a warp 16 rows by 16 keys; softmax: eight lanes a row;
// outputs: a warp 16 rows by a quarter of the columns, a tile's sum made by itself and added to the running one.  While the
// scores are made the tile's values arrive, while the outputs are summed the next tile's keys.
// bfloat16: operands as they are, probabilities rounded to bfloat16, the values' type (their sum is of the unrounded ones).  float32: an operand is split into three bfloat16 parts, which hold its 24
// bits, as it is read (queries once), six of the nine products are made (the rest is below 2^-24 of a product), the largest in an accumulator
// of its own; values are multiplied by 2^16 first, so that small ones keep their bits, and the sums by 2^-16.
// A product with a value that is no number reaches every row (zero times infinity), and float32's parts cannot hold one, nor one that 2^16 takes
// beyond the numbers.  Where a float32 score is no finite number it is made again from the operands.  Where an output's sum over a tile is none,
// such values are set to zero in shared memory, the tile's sums are made again, and the values are added for the rows that see them.
// What bounds it: the chain keys - scores - softmax - values of a tile, 2.3 us (bfloat16, heads of 128) or 5.5 us (float32, where the splitting of
// operands and six products are as long as the waits), hence two CTAs an SM and keys shared out down to one tile a CTA.  Measured: one tree of 8
// nodes behind 500 tokens, 16 query and 8 key heads of 128, bfloat16 8.5 us in eight shares that join as clusters (9.5 with a merge launch, 22.2
// unsplit); float32, three trees of 13 nodes behind a window of 1,000, 25 us in 16 shares, 95 unsplit.  On the CUDA cores those took 71.
constexpr int MROWS = 32, MTHREADS = 256;
constexpr int SP = KEY_TILE + 8;              // floats of a row of scores: eight-byte reads of four rows by four lanes hit all banks
constexpr float UP = 65536.f, DOWN = 1.f / UP;

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ void ldsm(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_addr(p)));
}
__device__ __forceinline__ void ldsm_trans(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_addr(p)));
}
__device__ __forceinline__ void mma16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
struct Parts { unsigned h, m, l; };           // of two neighbouring values, the first in the low half
__device__ __forceinline__ Parts split(float x, float y) {
    Parts p;
    p.h = pack_bf16(x, y);
    x -= __uint_as_float(p.h << 16);
    y -= __uint_as_float(p.h & 0xffff0000u);
    p.m = pack_bf16(x, y);
    x -= __uint_as_float(p.m << 16);
    y -= __uint_as_float(p.m & 0xffff0000u);
    p.l = pack_bf16(x, y);
    return p;
}
// The six products of a first operand's parts (h, m, l) and a second's.
__device__ __forceinline__ void mma_parts(float (&big)[4], float (&rest)[4], const unsigned (&ah)[4], const unsigned (&am)[4], const unsigned (&al)[4],
                                          const Parts& b0, const Parts& b1) {
    mma16(big, ah, b0.h, b1.h);
    mma16(rest, ah, b0.l, b1.l);
    mma16(rest, al, b0.h, b1.h);
    mma16(rest, am, b0.m, b1.m);
    mma16(rest, ah, b0.m, b1.m);
    mma16(rest, am, b0.h, b1.h);
}
// Whether the products cannot take a value.
__device__ __forceinline__ bool is_odd(float x) { return (__float_as_uint(x) & 0x7fffffffu) >= 0x73800000u; }        // |x| >= 2^104 (times 2^16, 64 of them are still numbers), or no number
__device__ __forceinline__ bool is_odd(bf16 x) { return (__bfloat16_as_ushort(x) & 0x7f80u) == 0x7f80u; }

template <typename TA, int DP> struct MmaShape {
    static constexpr bool F32 = sizeof(TA) == 4;
    static constexpr int KPITCH = DP + 8, VPITCH = F32 ? DP + 4 : DP + 8, QPITCH = DP + 8;        // elements; reads of fragments hit all banks
    static constexpr size_t K_BYTES = (size_t)KEY_TILE * KPITCH * sizeof(TA), V_BYTES = (size_t)KEY_TILE * VPITCH * sizeof(TA),
                            Q_BYTES = (F32 ? 3 : 1) * (size_t)MROWS * QPITCH * 2, S_BYTES = (size_t)MROWS * SP * 4, P_BYTES = F32 ? 0 : (size_t)MROWS * SP * 2;
    static constexpr size_t SMEM = K_BYTES + V_BYTES + Q_BYTES + S_BYTES + P_BYTES;
};

// grid: (row blocks x kv heads, segments, splits).  DP: the head size rounded up to 32, 64, 128 or 256; what lies behind D is zero.
template <typename TA, int DP>
__global__ void __launch_bounds__(MTHREADS, DP <= 128 ? 2 : 1)
tree_mma_kernel(const TA* __restrict__ q, int ld, const TA* __restrict__ kpool, const TA* __restrict__ vpool,
                const int* __restrict__ cu_q, const int* __restrict__ seg_pos0, const int* __restrict__ tree_parent,
                const int* __restrict__ block_table, int bt_stride, int page_size, int pages, TA* __restrict__ out,
                float* __restrict__ part_o, float* __restrict__ part_ml, int total_rows, int Hq, int Hkv, int D, float scale, int window,
                float softcap, const float* __restrict__ sink, int share, int joined, int vec) {
    typedef MmaShape<TA, DP> S;
    constexpr bool F32 = S::F32;
    constexpr int PER16 = 16 / sizeof(TA);                             // elements of a 16-byte piece
    constexpr int K16 = DP / 16, NT = DP / 32;                         // steps along the head size; blocks of eight columns of a warp's quarter
    extern __shared__ __align__(16) unsigned char mma_smem[];
    TA* ks = reinterpret_cast<TA*>(mma_smem);                          // [KEY_TILE][KPITCH]
    TA* vs = reinterpret_cast<TA*>(mma_smem + S::K_BYTES);             // [KEY_TILE][VPITCH]
    bf16* qs = reinterpret_cast<bf16*>(mma_smem + S::K_BYTES + S::V_BYTES);              // [parts][MROWS][QPITCH]
    float* ss = reinterpret_cast<float*>(mma_smem + S::K_BYTES + S::V_BYTES + S::Q_BYTES);       // [MROWS][SP]: scores, then probabilities
    bf16* ps = reinterpret_cast<bf16*>(mma_smem + S::K_BYTES + S::V_BYTES + S::Q_BYTES + S::S_BYTES);     // [MROWS][SP] in bfloat16
    __shared__ int parent[TREE_MAX_NODES];
    __shared__ unsigned lines[MROWS][TREE_WORDS];
    __shared__ long long where[2][KEY_TILE];
    __shared__ int lows[MROWS];                                        // a row's first key
    __shared__ unsigned odd_keys[2];                                   // a tile's keys whose values the products cannot take
    __shared__ float s_alpha[MROWS];
    __shared__ float2 s_ml[MROWS];                                     // maximum (in units of log2) and sum
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seg = blockIdx.y, kvh = blockIdx.x % Hkv, row0 = blockIdx.x / Hkv * MROWS, sp = blockIdx.z, G = Hq / Hkv;
    const Segment sg(cu_q, seg_pos0, seg, window, share, gridDim.z);
    const int rows = min(MROWS, sg.n * G - row0);
    if (rows <= 0) return;                                             // all shares of a block of rows alike
    if (sp >= sg.n_split) {
        if (joined) { tc5::cluster_sync_all(); tc5::cluster_sync_all(); }
        return;
    }
    const int* bt = block_table + (size_t)seg * bt_stride;
    const int t0 = share > 0 ? sp * share : 0, t1 = share > 0 && sp + 1 < sg.n_split ? t0 + share : sg.tiles;      // this CTA's tiles
    auto q_row = [&](int r) { return q + (size_t)(sg.q_begin + (row0 + r) / G) * ld + (size_t)(kvh * G + (row0 + r) % G) * D; };

    // Where a tile's rows lie in a pool, -1: no key of this CTA's, or a block marked as gone.
    auto locate = [&](int jt) {
        if (tid < KEY_TILE) {
            const int j = jt * KEY_TILE + tid, page = j >= sg.lo && j <= sg.hi ? page_at(bt + j / page_size, pages) : -1;
            where[jt & 1][tid] = page < 0 ? -1 : (((long long)page * Hkv + kvh) * page_size + j % page_size) * D;
        }
    };
    // A tile's keys or values on their way: PIECES lanes a row; rows at -1 become zero.
    constexpr int PIECES = DP / PER16 < 32 ? DP / PER16 : 32;
    const int d_first = PER16 * (lane % PIECES);
    auto fetch = [&](TA* to, int pitch, const TA* pool, int jt) {
#pragma unroll 4
        for (int r = warp * (32 / PIECES) + lane / PIECES; r < KEY_TILE; r += (MTHREADS / 32) * (32 / PIECES)) {
            const long long at = where[jt & 1][r];
#pragma unroll
            for (int d = d_first; d < DP; d += PER16 * PIECES) {
                if (d >= D) continue;
                if (vec) {
                    const int bytes = at < 0 ? 0 : 16;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_addr(to + r * pitch + d)), "l"(pool + (at < 0 ? 0 : at + d)), "r"(bytes));
                } else {
#pragma unroll
                    for (int e = 0; e < PER16; ++e)
                        if (d + e < D) to[r * pitch + d + e] = at >= 0 ? pool[at + d + e] : from_f32<TA>(0.f);
                }
            }
        }
        asm volatile("cp.async.commit_group;\n" ::);
    };
    locate(sg.jt0 + t0);
    for (int i = tid; i < sg.n; i += MTHREADS) parent[i] = tree_parent[sg.q_begin + i];
    if (tid < 2) odd_keys[tid] = 0u;
    for (int i = tid; i < KEY_TILE * (DP - D); i += MTHREADS) {        // behind the head size, for good
        const int r = i / (DP - D), d = D + i % (DP - D);
        ks[r * S::KPITCH + d] = vs[r * S::VPITCH + d] = from_f32<TA>(0.f);
    }
    // Queries, split: rows that do not exist are zero.
    {
        constexpr int QR = MROWS * 32 / MTHREADS, QU = (DP + 63) / 64;
        float2 x[QR][QU];
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const int r = warp * QR + i;
            const TA* src = q_row(r < rows ? r : 0);
#pragma unroll
            for (int u = 0; u < QU; ++u) {
                const int d = 2 * lane + 64 * u;
                x[i][u] = make_float2(r < rows && d < D ? to_f32(src[d]) : 0.f, r < rows && d + 1 < D ? to_f32(src[d + 1]) : 0.f);
            }
        }
#pragma unroll
        for (int i = 0; i < QR; ++i)
#pragma unroll
            for (int u = 0; u < QU; ++u) {
                const int d = 2 * lane + 64 * u;
                if (d >= DP) continue;
                unsigned* to = reinterpret_cast<unsigned*>(qs + (warp * QR + i) * S::QPITCH + d);
                if (F32) {
                    const Parts p = split(x[i][u].x, x[i][u].y);
                    to[0] = p.h;
                    to[MROWS * S::QPITCH / 2] = p.m;
                    to[MROWS * S::QPITCH] = p.l;
                } else {
                    to[0] = pack_bf16(x[i][u].x, x[i][u].y);
                }
            }
    }
    __syncthreads();
    fetch(ks, S::KPITCH, kpool, sg.jt0 + t0);
    if (tid < MROWS) {
        unsigned line[TREE_WORDS];
        const int depth = tree_line(parent, tid < rows ? (row0 + tid) / G : 0, window, line);
        lows[tid] = tid < rows ? (window > 0 ? max(0, sg.c + depth - window + 1) : 0) : sg.hi + 1;
#pragma unroll
        for (int w = 0; w < TREE_WORDS; ++w) lines[tid][w] = tid < rows ? line[w] : 0u;
    }
    auto sees = [&](int r, int j) { return j <= sg.hi && (j < sg.c ? j >= lows[r] : (line_bits(lines[r], (j & ~31) - sg.c) >> (j & 31)) & 1u); };
    const int rt = 16 * (warp & 1), part = warp >> 1;                  // a warp's rows, and its block of keys or columns
    const int g = lane >> 2, t4 = lane & 3;
    const int r_a = rt + (lane & 7) + ((lane >> 3) & 1) * 8, c_a = 8 * (lane >> 4);      // a lane's row and column of a first operand's ldmatrix
    float m = -INFINITY, l = 0.f, o[NT][4];                            // m, l: of row 4 warp + lane / 8
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    for (int t = t0; t < t1; ++t) {
        const int jt = sg.jt0 + t, j0 = jt * KEY_TILE;
        const bool whole = j0 + KEY_TILE - 1 < sg.c && (window <= 0 || j0 > sg.c + sg.n - 1 - window);
        fetch(vs, S::VPITCH, vpool, jt);                               // the last reader passed the barrier behind the outputs
        asm volatile("cp.async.wait_group 1;\n" ::);
        __syncthreads();                                               // the keys are there
        {
            float big[2][4] = {}, rest[2][4] = {};
#pragma unroll
            for (int k = 0; k < K16; ++k) {
                unsigned ah[4], am[4], al[4];
                ldsm(ah, qs + r_a * S::QPITCH + 16 * k + c_a);
                if (F32) {
                    ldsm(am, qs + (MROWS + r_a) * S::QPITCH + 16 * k + c_a);
                    ldsm(al, qs + (2 * MROWS + r_a) * S::QPITCH + 16 * k + c_a);
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float* at = reinterpret_cast<const float*>(ks) + (16 * part + 8 * n + g) * S::KPITCH + 16 * k + 2 * t4;
                        const float2 x = *reinterpret_cast<const float2*>(at), y = *reinterpret_cast<const float2*>(at + 8);
                        mma_parts(big[n], rest[n], ah, am, al, split(x.x, x.y), split(y.x, y.y));
                    }
                } else {
                    unsigned b[4];
                    ldsm(b, ks + (16 * part + ((lane >> 4) << 3) + (lane & 7)) * S::KPITCH + 16 * k + 8 * ((lane >> 3) & 1));
                    mma16(big[0], ah, b[0], b[1]);
                    mma16(big[1], ah, b[2], b[3]);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float2*>(ss + (rt + g + 8 * h) * SP + 16 * part + 8 * n + 2 * t4) =
                        make_float2(big[n][2 * h] + rest[n][2 * h], big[n][2 * h + 1] + rest[n][2 * h + 1]);
        }
        if (t + 1 < t1) locate(jt + 1);
        __syncthreads();                                               // scores are there, the keys have been used
        if (t + 1 < t1) fetch(ks, S::KPITCH, kpool, jt + 1);
        else asm volatile("cp.async.commit_group;\n" ::);
        {
            // Softmax: eight lanes a row; lane i of them keys 4 i ..+ 3 and 32 + 4 i ..+ 3.
            const int r = 4 * warp + (lane >> 3), key0 = 4 * (lane & 7);
            float x[8];
            auto key_of = [&](int e) { return key0 + (e & 3) + 8 * (e & 4); };
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float4 f = *reinterpret_cast<const float4*>(ss + r * SP + key0 + 32 * u);
                x[4 * u] = f.x; x[4 * u + 1] = f.y; x[4 * u + 2] = f.z; x[4 * u + 3] = f.w;
            }
            if (F32) {                                                 // scores that are no finite number, from the operands
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) odd = odd || !isfinite(x[e]);
                if (odd && r < rows) {
                    const TA* query = q_row(r);
#pragma unroll 1
                    for (int e = 0; e < 8; ++e) {
                        const long long at = where[jt & 1][key_of(e)];
                        if (isfinite(x[e]) || at < 0) continue;
                        float sum = 0.f;
#pragma unroll 1
                        for (int d = 0; d < D; ++d) sum = fmaf(to_f32(query[d]), to_f32(kpool[at + d]), sum);
                        x[e] = sum;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= scale;
            if (softcap > 0.f) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = softcap * tanhf(x[e] / softcap);
            }
            unsigned vis = 0xffu;
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!sees(r, j0 + key_of(e))) { x[e] = -INFINITY; vis &= ~(1u << e); }
            }
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
#pragma unroll
            for (int w = 4; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float m_new = fmaxf(m, top), ref = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = expf(m - ref);                         // m = -inf on the first tile gives 0
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (vis >> e) & 1u ? expf(x[e] - ref) : 0.f;
            float sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
            for (int w = 4; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            l = l * alpha + sum;
            m = m_new;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                *reinterpret_cast<float4*>(ss + r * SP + key0 + 32 * u) = make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
                if (!F32)
                    *reinterpret_cast<uint2*>(ps + r * SP + key0 + 32 * u) = make_uint2(pack_bf16(x[4 * u], x[4 * u + 1]), pack_bf16(x[4 * u + 2], x[4 * u + 3]));
            }
            if ((lane & 7) == 0) s_alpha[r] = alpha;
        }
        asm volatile("cp.async.wait_group 1;\n" ::);
        __syncthreads();                                               // probabilities and values are there
        float tile[NT][4];
        bool redone = false;
        const int col0 = part * (DP / 4);                              // a warp's quarter of the columns
        while (true) {
            float rest[F32 ? NT : 1][4] = {};
#pragma unroll
            for (int n = 0; n < NT; ++n) tile[n][0] = tile[n][1] = tile[n][2] = tile[n][3] = 0.f;
#pragma unroll
            for (int k = 0; k < KEY_TILE / 16; ++k) {
                if (F32) {
                    Parts a[4];                                        // rows g and g + 8, keys 2 t4 and 2 t4 + 8
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 p = *reinterpret_cast<const float2*>(ss + (rt + g + 8 * (i & 1)) * SP + 16 * k + 2 * t4 + 8 * (i >> 1));
                        a[i] = split(p.x, p.y);
                    }
                    const unsigned ah[4] = {a[0].h, a[1].h, a[2].h, a[3].h}, am[4] = {a[0].m, a[1].m, a[2].m, a[3].m}, al[4] = {a[0].l, a[1].l, a[2].l, a[3].l};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float* at = reinterpret_cast<const float*>(vs) + (16 * k + 2 * t4) * S::VPITCH + col0 + 8 * n + g;
                        const Parts b0 = split(at[0] * UP, at[S::VPITCH] * UP), b1 = split(at[8 * S::VPITCH] * UP, at[9 * S::VPITCH] * UP);
                        mma_parts(tile[n], rest[F32 ? n : 0], ah, am, al, b0, b1);
                    }
                } else {
                    unsigned a[4];
                    ldsm(a, ps + r_a * SP + 16 * k + c_a);
                    const bf16* at = reinterpret_cast<const bf16*>(vs) + (16 * k + (lane & 7) + ((lane >> 3) & 1) * 8) * S::VPITCH + col0;
                    if (NT == 1) {                                     // one block: the other half of the four matrices is not used
                        unsigned b[4];
                        ldsm_trans(b, at);
                        mma16(tile[0], a, b[0], b[1]);
                    } else {
#pragma unroll
                        for (int n = 0; n + 1 < NT; n += 2) {
                            unsigned b[4];
                            ldsm_trans(b, at + 8 * n + c_a);
                            mma16(tile[n], a, b[0], b[1]);
                            mma16(tile[n + 1], a, b[2], b[3]);
                        }
                    }
                }
            }
            bool odd = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (F32) tile[n][e] = (tile[n][e] + rest[F32 ? n : 0][e]) * DOWN;
                    odd = odd || !isfinite(tile[n][e]);
                }
            if (redone || !__syncthreads_or(odd)) break;               // the values have been used
            for (int i = tid; i < KEY_TILE * D; i += MTHREADS) {
                TA* at = vs + (i / D) * S::VPITCH + i % D;
                if (is_odd(*at)) {
                    *at = from_f32<TA>(0.f);
                    atomicOr(&odd_keys[i / D >> 5], 1u << (i / D & 31));
                }
            }
            __syncthreads();
            redone = true;
        }
        {
            const float al0 = s_alpha[rt + g], al1 = s_alpha[rt + g + 8];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][e] = fmaf(o[n][e], e < 2 ? al0 : al1, tile[n][e]);
        }
        if (redone) {                                                  // what the products left out
            for (unsigned long long w = odd_keys[0] | ((unsigned long long)odd_keys[1] << 32); w != 0ull; w &= w - 1ull) {
                const int key = __ffsll((long long)w) - 1;
                const TA* value = vpool + max(where[jt & 1][key], 0ll);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = rt + g + 8 * (e >> 1), d = col0 + 8 * n + 2 * t4 + (e & 1);
                        if (d < D && is_odd(value[d]) && (whole || sees(r, j0 + key))) o[n][e] = fmaf(ss[r * SP + key], to_f32(value[d]), o[n][e]);
                    }
            }
            __syncthreads();
            if (tid < 2) odd_keys[tid] = 0u;
        }
    }
    pdl_trigger_late();
    if ((lane & 7) == 0) s_ml[4 * warp + (lane >> 3)] = make_float2(m * LOG2E, l);
    if (joined && sg.n_split > 1) {
        // Every share's outputs, maxima and sums lie where its keys lay; each takes a part of the (row, four columns) pairs and goes through the
        // shares in their order.
        constexpr int OP = DP + 4;
        static_assert(MROWS * OP * 4 <= S::K_BYTES, "room for the outputs");
        float* os = reinterpret_cast<float*>(mma_smem);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
                *reinterpret_cast<float2*>(os + (rt + g + 8 * hh) * OP + part * (DP / 4) + 8 * n + 2 * t4) = make_float2(o[n][2 * hh], o[n][2 * hh + 1]);
        tc5::cluster_sync_all();
        for (int i = sp * MTHREADS + tid; i < rows * (DP / 4); i += sg.n_split * MTHREADS) {
            const int r = i / (DP / 4), d = 4 * (i % (DP / 4)), row = row0 + r, h = kvh * G + row % G;
            if (d >= D) continue;
            float2 ml[JOIN_MAX];
            float4 f[JOIN_MAX];
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int u = 0; u < JOIN_MAX; ++u) {
                ml[u] = make_float2(-INFINITY, 0.f);
                if (u < sg.n_split) {
                    ml[u] = peer_float2(tc5::map_to_cta(smem_addr(s_ml + r), u));
                    f[u] = peer_float4(tc5::map_to_cta(smem_addr(os + r * OP + d), u));
                    top = fmaxf(top, ml[u].x);
                }
            }
            const float ref = top == -INFINITY ? 0.f : top;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < JOIN_MAX; ++u)
                if (ml[u].y != 0.f) {                                  // a share without keys for this row left nothing
                    const float w = exp2f(ml[u].x - ref);
                    total = fmaf(ml[u].y, w, total);
                    sum.x = fmaf(f[u].x, w, sum.x); sum.y = fmaf(f[u].y, w, sum.y);
                    sum.z = fmaf(f[u].z, w, sum.z); sum.w = fmaf(f[u].w, w, sum.w);
                }
            if (sink != nullptr) total += exp2f(sink[h] * LOG2E - ref);
            const float inv = total == 0.f ? 0.f : 1.0f / total;
            TA* to = out + ((size_t)(sg.q_begin + row / G) * Hq + h) * D + d;
            const float v[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < D) to[e] = from_f32<TA>(v[e]);
        }
        __syncwarp();
        tc5::cluster_sync_all();                                       // nobody leaves before its outputs have been read
        return;
    }
    __syncthreads();
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        const int r = rt + g + 8 * hh, row = row0 + r;
        if (r >= rows) continue;
        const int h = kvh * G + row % G;
        const size_t at = (size_t)(sg.q_begin + row / G) * Hq + h, slot = (size_t)sp * total_rows * Hq + at;
        const float2 ml = s_ml[r];
        float total = ml.y;
        if (sg.n_split > 1) {
            if (part == 0 && t4 == 0) *reinterpret_cast<float2*>(part_ml + 2 * slot) = ml;
        } else if (sink != nullptr) {
            total += ml.x == -INFINITY ? 1.f : exp2f(sink[h] * LOG2E - ml.x);
        }
        const float inv = total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = part * (DP / 4) + 8 * n + 2 * t4 + e;
                if (d >= D) continue;
                if (sg.n_split > 1) part_o[slot * D + d] = o[n][2 * hh + e];
                else out[at * D + d] = from_f32<TA>(o[n][2 * hh + e] * inv);
            }
    }
    __syncwarp();
    if (joined) { tc5::cluster_sync_all(); tc5::cluster_sync_all(); }  // beside shares that have nothing
}

// ---------------------------------------------------------------------------------------- fifth-generation tensor cores
// bfloat16, head sizes up to 256 that are multiples of 8, in shapes for 64, 128 and 256 (what lies behind the head size is zero).  A CTA (one an SM)
// owns rows of one segment and key/value head and walks its share of the keys in tiles of 64.  Two groups of four warps work side by side, so that one's waits pass while the other computes:
//   STREAMS        up to 128 rows: one query tile, the groups take the key tiles in turn.  With 64 rows or fewer the tile holds them twice, with
//                  32 four times, and of a key tile each copy's warps take a half or a quarter (their P is zero elsewhere): a row's thread has
//                  to sit on the warp of its tensor-memory lane, and this way all four have exponentials to make.  Every copy of either group
//                  has a maximum, sum and output of its own; they are joined at the end.  Heads of 256 have one group (the outputs of two do not
//                  fit into tensor memory);
//   else           up to 256 rows: a query tile of 128 rows a group, both go through every key tile.
// Per key tile and group:
//   S = Q K^T      tcgen05.mma, M = 128, N = 64, in tensor memory, two buffers a group;
//   softmax        a row a thread (its TMEM lane), no shuffles; P rounded to bfloat16 into S's own columns, since the second product's operands are of
//                  one type (the sum keeps the unrounded ones; against 64 bits outputs are off by up to 0.0023, with P in 32 bits 0.0017, where
//                  the rounding of the result alone is 0.0020).  The reference maximum moves only
//                  when the true one has outrun it by 2^8, so O is rescaled in tensor memory a few times at most;
//   O += P V       tcgen05.mma, M = 128, N = head size, P from tensor memory, V as it lies in the cache.
// Warps: four of rows a group (those without rows have nothing to do, and nobody waits for them), for each group one that issues S and one that issues
// P V (an issuing thread pays some 230 cycles a wait and 60 to 90 an instruction, so two threads share that), one that gathers K and one
// that gathers V into the 128-byte swizzle, through rings of STAGES tiles: page by page with TMA where pages are 8, 16, 32 or a multiple of 64
// rows, else row by row with cp.async.
// Barriers: each ring stage has a full and an empty one; S, P and P V have one for each of two buffers.  A barrier's next phase always needs
// all of its waiters to have passed the current one, so no parity wait can fall two phases behind.
// A key tile that some row does not see in full is looked through for values that are no numbers before the products take it: they are
// set to zero there (zero times infinity would reach every row) and added to the rows that see them at the end.
// What bounds it.  Few rows: HBM, and some 14 us around the walk (tables, tensor memory, first keys, outputs, join): 8 trees of 16 nodes behind 2,040
// tokens, 32 query and 8 key heads of 128, 25.4 us of which the walk of 69 MB takes 11; 64 trees of 8 nodes 133 us, 4.1 TB/s.  Many rows: the row
// warps, 1,390 cycles of the 1,830 a key tile of 256 rows takes (exponentials 1,024 of them, were nothing else in their way), while the tensor cores are
// busy for 45 %: 32 trees of up to 64 nodes behind 2,000 to 8,000 tokens, 64 query and 8 key heads, 322 us, 0.80 PFLOP/s, at the power limit when they
// follow each other (360 us then).  Tried there: P through shared memory 345 us; the maximum before the exponentials 335; every fourth or second pair of
// exponentials as a polynomial on the multiply-add units 335 and 348; key tiles cut into shares for the balance of the SMs costs the
// traffic of partial results, 24 us at two shares, for 8 % of balance.
using namespace tc5;

constexpr int QM = 128;                       // rows of a query tile
constexpr int KN = KEY_TILE;
constexpr float RESCALE_STEP = 8.0f;          // log2 units the true maximum may run ahead of the reference

template <int N> struct Width { static constexpr int value = N; };

template <int D, bool STREAMS> struct Shape {
    static constexpr int GROUPS = D == 256 ? 1 : 2, NQ = STREAMS ? 1 : GROUPS;       // groups of row warps; query tiles
    static constexpr int DS = D / 64;         // 64-wide slabs of the head size
    static constexpr unsigned Q_BYTES = DS * QM * 128, K_BYTES = DS * KN * 128;
    static constexpr int STAGES = D == 256 ? 2 : D == 128 ? (STREAMS ? 6 : 5) : (STREAMS ? 8 : 6);
    static constexpr int LAG = STAGES >= 4 ? 2 : 1;           // a tile is announced when this many later ones have been asked for
    static constexpr int W_ISSUE = 4 * GROUPS, W_LOAD = 6 * GROUPS, THREADS = 32 * (W_LOAD + 2);      // the first warps of the other roles
    static constexpr unsigned TMEM_COLS = 512, O_COL = GROUPS * 2 * KN;
    static constexpr int B_K_FULL = 0, B_V_FULL = STAGES, B_K_EMPTY = 2 * STAGES, B_V_EMPTY = 3 * STAGES, B_S = 4 * STAGES,
                         B_P = B_S + 2 * GROUPS, B_PV = B_P + 2 * GROUPS, B_Q = B_PV + 2 * GROUPS, B_V_LAND = B_Q + GROUPS, N_BARS = B_V_LAND + STAGES;
    static constexpr unsigned TAIL = N_BARS * 8 + 16 + TREE_MAX_NODES * 4;
    static constexpr unsigned SMEM_USED = NQ * Q_BYTES + 2 * STAGES * K_BYTES + TAIL;
    static constexpr unsigned SMEM = SMEM_USED > 120 * 1024 ? SMEM_USED : 120 * 1024;       // one CTA an SM: it takes all of the tensor memory
    static_assert(SMEM <= 227 * 1024 && O_COL + GROUPS * D <= TMEM_COLS && STAGES > LAG, "a CTA's memories");
    static_assert(2 * STAGES * K_BYTES >= GROUPS * QM * D * 4, "room for the outputs behind Q");
    static_assert(!STREAMS || GROUPS == 1 || STAGES % 2 == 0, "a ring stage belongs to one group, so that its barriers' phases come in turn");
};

// D += A B^T with A in tensor memory: a lane a row, two neighbouring values of k a column.
__device__ __forceinline__ void mma_ts(unsigned d_tmem, unsigned a_tmem, unsigned long long b_desc, unsigned idesc, bool accumulate) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"((unsigned)accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st16(unsigned taddr, const unsigned (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st8(unsigned taddr, const unsigned (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void cp16u(unsigned smem_addr, const void* gmem, bool pred) {
    const int bytes = pred ? 16 : 0;          // 0: nothing is read, the 16 bytes become zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_addr), "l"(gmem), "r"(bytes));
}
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
// Waits for the loads from tensor memory, and ties their registers to it.
__device__ __forceinline__ void tmem_ld_wait32(unsigned (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
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

// grid: (row blocks x kv heads, segments, splits).  CAP: scores are capped.  WHOLE: the head size is D, else head_size, less than D.  (The plain
// kernels are spared the registers: 32 trees behind 2,000 to 8,000 tokens are 4 % slower with a head size of its own.)
template <int D, bool STREAMS, bool CAP, bool WHOLE>
__global__ void __launch_bounds__(Shape<D, STREAMS>::THREADS, 1)
tree_tc5_kernel(const bf16* __restrict__ q, int ld, const bf16* __restrict__ kpool, const bf16* __restrict__ vpool,
                const int* __restrict__ cu_q, const int* __restrict__ seg_pos0, const int* __restrict__ tree_parent,
                const int* __restrict__ block_table, int bt_stride, int page_size, int pages, bf16* __restrict__ out,
                float* __restrict__ part_o, float* __restrict__ part_ml, int total_rows, int Hq, int Hkv, int head_size, float scale, int window,
                float softcap, const float* __restrict__ sink, int share, int joined, int* __restrict__ status, int by_tma,
                const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    const int head = WHOLE ? D : head_size;
    typedef Shape<D, STREAMS> S;
    constexpr int STAGES = S::STAGES, NQ = S::NQ, GROUPS = S::GROUPS, W_ISSUE = S::W_ISSUE, W_LOAD = S::W_LOAD;
    // The swizzled tiles need 1024-byte alignment: the kernel has no static shared memory, so its window starts at the CTA's base.
    extern __shared__ __align__(1024) unsigned char tc5_smem[];
    if ((smem_u32(tc5_smem) & 1023u) != 0u) {
        if (threadIdx.x == 0) atomicExch(status, 2);
        return;
    }
    unsigned char* sQ = tc5_smem;                             // [query tile]
    unsigned char* sK = sQ + NQ * S::Q_BYTES;                 // [stage]
    unsigned char* sV = sK + STAGES * S::K_BYTES;             // [stage]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(sV + STAGES * S::K_BYTES);
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + S::N_BARS);
    volatile int* odd_values = reinterpret_cast<int*>(tmem_slot + 1);
    int* parent = reinterpret_cast<int*>(tmem_slot + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    const int seg = blockIdx.y, kvh = blockIdx.x % Hkv, row0 = blockIdx.x / Hkv * (NQ * QM), split = blockIdx.z, G = Hq / Hkv;
    const Segment sg(cu_q, seg_pos0, seg, window, share, gridDim.z);
    const int rows = min(NQ * QM, sg.n * G - row0);
    if (rows <= 0) return;                                    // all shares of a block of rows alike
    if (split >= sg.n_split) {
        if (joined) { cluster_sync_all(); cluster_sync_all(); }
        return;
    }
    const int t0 = share > 0 ? split * share : 0, t1 = share > 0 && split + 1 < sg.n_split ? t0 + share : sg.tiles;
    const int jt_begin = sg.jt0 + t0, n_tiles = t1 - t0;      // one tile at least
    const int* bt_row = block_table + (size_t)seg * bt_stride;
    const Paging pg(page_size);
    const ByDivisor by_group(G);
    const unsigned bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    // STREAMS: the query tile holds its rows `copies` times, copy_rows rows each
    const int copy_rows = rows > 64 ? 128 : rows > 32 ? 64 : 32, copies = STREAMS ? QM / copy_rows : 1;
    // a group's rows (as warps), its key tiles, and the number of its i-th among the CTA's
    auto active_warps = [&](int g) { return STREAMS && copies > 1 ? 4 : max(0, min(4, (rows - (STREAMS ? 0 : g * QM) + 31) >> 5)); };
    auto tiles_of = [&](int g) { return STREAMS ? (n_tiles - g + GROUPS - 1) / GROUPS : active_warps(g) > 0 ? n_tiles : 0; };
    auto tile_no = [&](int g, int i) { return STREAMS ? GROUPS * i + g : i; };
    // whether every row sees every key of a tile
    auto whole = [&](int j_base) { return j_base + KN - 1 < sg.c && (window <= 0 || j_base > sg.c + sg.n - 1 - window); };

    // Everything that waits for memory is asked for before the barrier: queries, parents, the loaders' first pages.
    constexpr int LPR = D / 8, RPI = 32 / LPR;                // lanes a row of 16-byte pieces, rows an instruction
    const int rsel = lane / LPR, sub = lane % LPR;
    if (warp < W_ISSUE && (warp & 3) < active_warps(warp >> 2)) {
        constexpr int MINE = STREAMS ? 32 / GROUPS : 32;      // rows a warp asks for: STREAMS' groups share a tile
        unsigned char* tile = sQ + (STREAMS ? 0 : warp >> 2) * S::Q_BYTES + (unsigned)(sub >> 3) * (QM * 128);
#pragma unroll 4
        for (int i = 0; i < MINE / RPI; ++i) {                // a row's pieces by neighbouring lanes
            const int rt = (warp & 3) * 32 + (STREAMS ? (warp >> 2) * MINE : 0) + i * RPI + rsel, rr = row0 + (STREAMS ? rt & (copy_rows - 1) : (warp >> 2) * QM + rt);
            const bool there = rr - row0 < rows && sub * 8 < head;
            const int2 nh = by_group(rr);
            const bf16* src = q + (there ? (size_t)(sg.q_begin + nh.x) * ld + (size_t)(kvh * G + nh.y) * head + sub * 8 : 0);
            cp16u(smem_u32(tile + sw128_offset(rt, sub & 7)), src, there);
        }
    }
    asm volatile("cp.async.commit_group;\n" ::);
    for (int i = tid; i < sg.n; i += S::THREADS) parent[i] = tree_parent[sg.q_begin + i];
    const int box = min(pg.page_size, KN), pi = lane / S::DS, slab = lane % S::DS;       // a loader's lane by TMA: page of the tile, slab
    auto in_sight = [&](int jt) { const int j = jt * KN + pi * box; return pi * box < KN && j + box > sg.lo && j <= sg.hi; };
    auto ask_page = [&](int jt) { return in_sight(jt) ? page_at(bt_row + pg.block(jt * KN + pi * box), pages) : -1; };
    int next = warp >= W_LOAD && by_tma ? ask_page(jt_begin) : -1;
    if (warp == W_ISSUE) tmem_alloc(smem_u32(tmem_slot), S::TMEM_COLS);
    if (tid < S::N_BARS) {
        const int i = tid;
        int count = 1;
        if (i >= S::B_K_EMPTY && i < S::B_S) count = !STREAMS && rows > QM ? 2 : 1;           // the groups that read a key tile
        else if (i >= S::B_P && i < S::B_PV) count = max(1, active_warps((i - S::B_P) >> 1));
        else if (i >= S::B_Q && i < S::B_V_LAND) count = STREAMS ? GROUPS * active_warps(0) : max(1, active_warps(i - S::B_Q));
        mbar_init(bar(i), count);
        mbar_init_fence();
    }
    if (tid == 0) *odd_values = 0;
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const unsigned tmem = *tmem_slot;
    bool ok = true;

    const int grp = warp < W_ISSUE ? warp >> 2 : warp < W_LOAD ? (warp - W_ISSUE) >> 1 : 0;      // group of a row warp or an issuer
    const int qt = STREAMS ? 0 : grp, n_mine = tiles_of(grp);
    const bool has_rows = warp < W_ISSUE && (warp & 3) < active_warps(grp);
    // a row thread's row of the tile (its lane of tensor memory), its copy, its row in the CTA, of the segment and head
    const int r = (warp & 3) * 32 + lane, copy = STREAMS ? r / copy_rows : 0, in_cta = STREAMS ? r & (copy_rows - 1) : qt * QM + r, row = row0 + in_cta;
    const bool row_valid = has_rows && in_cta < rows;
    const int2 node_head = by_group(row_valid ? row : 0);
    const size_t token = (size_t)sg.q_begin + node_head.x;
    const int h = kvh * G + node_head.y;
    const float scale_log2 = scale * LOG2E, scale_eff = CAP ? softcap * LOG2E : scale_log2;
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

    if (has_rows) {
        // ================================================================== one row per thread, W keys of a tile
        const int depth = tree_line(parent, node_head.x, window, line);
        lo_r = window > 0 ? max(0, sg.c + depth - window + 1) : 0;
        cp_wait<0>();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(S::B_Q + qt));
        // capped scores: a polynomial where all of the warp's are well below the cap
        auto cap = [&](auto& a) {
            constexpr int N = sizeof(a) / sizeof(a[0]);
            const float k = scale / softcap;
            float far = 0.f;
#pragma unroll
            for (int e = 0; e < N; e += 2) far = max3(far, fabsf(__uint_as_float(a[e])), fabsf(__uint_as_float(a[e + 1])));
            if (!__any_sync(0xffffffffu, !(far * k <= TANH_POLY_MAX))) {
                const unsigned long long k2 = pack2(k, k);
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const unsigned long long x = mul2(pack2(__uint_as_float(a[e]), __uint_as_float(a[e + 1])), k2), u = mul2(x, x);
                    unsigned long long t = fma2(u, pack2(TANH_P4, TANH_P4), pack2(TANH_P3, TANH_P3));
                    t = fma2(u, t, pack2(TANH_P2, TANH_P2));
                    t = fma2(u, t, pack2(TANH_P1, TANH_P1));
                    float t0, t1;
                    unpack2(mul2(x, fma2(u, t, pack2(TANH_P0, TANH_P0))), t0, t1);
                    a[e] = __float_as_uint(t0);
                    a[e + 1] = __float_as_uint(t1);
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) a[e] = __float_as_uint(fast_tanh(__uint_as_float(a[e]) * k));
            }
        };
        auto walk = [&](auto width) {
            constexpr int W = decltype(width)::value;
            const int col = W == 64 ? 0 : copy * W;           // of a tile's keys
            for (int i = 0; i < n_mine; ++i) {
                const int j_base = (jt_begin + tile_no(grp, i)) * KN, buf = i & 1;
                ok = mbar_wait(bar(S::B_S + grp * 2 + buf), (i >> 1) & 1) && ok;
                fence_after_sync();
                const unsigned from = lane_addr + (grp * 2 + buf) * KN + col;
                const unsigned long long scale2 = pack2(scale_eff, scale_eff);
                unsigned w[W / 2];
                float tile_sum = 0.f;
                bool done = false;
                if (whole(j_base)) {
                    // The reference rarely moves: the exponentials are made with the last one while the maximum is looked for, and thrown away if it has
                    // been outrun.
                    const float mu = m_ref == -INFINITY ? 0.f : m_ref;
                    const unsigned long long shift2 = pack2(-mu, -mu);
                    constexpr int H = W < 32 ? W : 32;
                    unsigned half[W / H][H];
                    unsigned long long sum2[2] = {};
                    float top[2] = {-INFINITY, -INFINITY};
                    if constexpr (W == 16) {
                        tmem_ld16(from, half[0]);
                        tmem_ld_wait();
                    } else {
                        tmem_ld32(from, half[0]);
                        tmem_ld_wait32(half[0]);
                        if constexpr (W == 64) tmem_ld32(from + 32, half[1]);
                    }
#pragma unroll
                    for (int q = 0; q < W / H; ++q) {
                        if constexpr (W == 64)
                            if (q == 1) tmem_ld_wait32(half[1]);
                        if (CAP) cap(half[q]);
#pragma unroll
                        for (int e = 0; e < H; e += 2) {
                            const float s0 = __uint_as_float(half[q][e]), s1 = __uint_as_float(half[q][e + 1]);
                            const unsigned long long x = fma2(pack2(s0, s1), scale2, shift2);
                            float x0, x1;
                            unpack2(x, x0, x1);
                            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                            top[(e >> 1) & 1] = max3(top[(e >> 1) & 1], s0, s1);
                            sum2[(e >> 1) & 1] = add2(sum2[(e >> 1) & 1], pack2(p0, p1));
                            w[q * (H / 2) + (e >> 1)] = pack_bf16(p0, p1);
                        }
                    }
                    done = !__any_sync(0xffffffffu, fmaxf(top[0], top[1]) * scale_eff > m_ref + RESCALE_STEP);
                    float sum_lo, sum_hi;
                    unpack2(add2(sum2[0], sum2[1]), sum_lo, sum_hi);
                    tile_sum = sum_lo + sum_hi;
                }
                if (!done) {
                    unsigned a[W];
                    if constexpr (W == 16) {
                        tmem_ld16(from, a);
                    } else {
#pragma unroll
                        for (int c = 0; c < W; c += 32) tmem_ld32(from + c, reinterpret_cast<unsigned(&)[32]>(a[c]));
                    }
                    tmem_ld_wait();
                    if (CAP) cap(a);
                    if (!whole(j_base)) {
                        const unsigned long long vis = visible(j_base) >> col;
                        const unsigned vis_lo = (unsigned)vis, vis_hi = (unsigned)(vis >> 32);
#pragma unroll
                        for (int e = 0; e < W; ++e)
                            if (!((e < 32 ? vis_lo : vis_hi) & (1u << (e & 31)))) a[e] = 0xff800000u;
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < W; e += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) top[k] = max3(top[k], __uint_as_float(a[e + 2 * k]), __uint_as_float(a[e + 2 * k + 1]));
                    const float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]) * scale_eff;     // the scale is positive
                    float alpha = 1.f;
                    bool moved = false;
                    if (mx > m_ref + RESCALE_STEP || (m_ref == -INFINITY && mx != -INFINITY)) {
                        alpha = fast_exp2(m_ref - mx);            // 0 on the first move
                        m_ref = mx;
                        moved = true;
                    }
                    const float mu = m_ref == -INFINITY ? 0.f : m_ref;
                    // P(i) goes into the buffer that P V(i - 2) read: that was done when S(i) was issued.  O is touched only when P V(i - 1) is done.
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
                    const unsigned long long shift2 = pack2(-mu, -mu);
                    unsigned long long sum2[4] = {};
#pragma unroll
                    for (int c = 0; c < W / 8; ++c) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float x0, x1;
                            unpack2(fma2(pack2(__uint_as_float(a[8 * c + 2 * k]), __uint_as_float(a[8 * c + 2 * k + 1])), scale2, shift2), x0, x1);
                            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                            sum2[k] = add2(sum2[k], pack2(p0, p1));
                            w[4 * c + k] = pack_bf16(p0, p1);
                        }
                    }
                    float sum_lo, sum_hi;
                    unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), sum_lo, sum_hi);
                    tile_sum = sum_lo + sum_hi;
                    l_run *= alpha;
                }
                l_run += tile_sum;
                // P(i) takes the first half of S(i)'s columns; the other copies' keys are zero there
                const unsigned p_addr = lane_addr + (grp * 2 + buf) * KN;
                if constexpr (W == 64) {
                    tmem_st32(p_addr, w);
                } else if constexpr (W == 32) {
                    const unsigned none[16] = {};
                    tmem_st16(p_addr + copy * 16, w);
                    tmem_st16(p_addr + (copy ^ 1) * 16, none);
                } else {
                    const unsigned none[8] = {};
                    tmem_st8(p_addr + copy * 8, w);
#pragma unroll
                    for (int c = 1; c < 4; ++c) tmem_st8(p_addr + (copy ^ c) * 8, none);
                }
                tmem_st_wait();
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(S::B_P + grp * 2 + buf));       // S(i) is read, O is rescaled, P(i) is written
            }
        };
        if (copies == 1) walk(Width<64>());
        else if (copies == 2) walk(Width<32>());
        else walk(Width<16>());
        if (n_mine > 0) ok = mbar_wait(bar(S::B_PV + grp * 2 + ((n_mine - 1) & 1)), ((n_mine - 1) >> 1) & 1) && ok;
    } else if (warp >= W_ISSUE && warp < W_LOAD && n_mine > 0 && lane == 0) {
        // ================================================================== an issuing thread: descriptors are a base plus a constant
        ok = mbar_wait(bar(S::B_Q + qt), 0) && ok;
        fence_after_sync();
        if ((warp & 1) == 0) {                                // S
            const unsigned idesc = instr_desc_bf16(QM, KN, false);
            const unsigned long long dQ = smem_desc_sw128(smem_u32(sQ) + qt * S::Q_BYTES, 0), dK = smem_desc_sw128(smem_u32(sK), 0);
            for (int i = 0; i < n_mine; ++i) {
                const int t = tile_no(grp, i), st = t % STAGES;
                ok = mbar_wait(bar(S::B_K_FULL + st), (t / STAGES) & 1) && ok;
                if (i > 1) ok = mbar_wait(bar(S::B_PV + grp * 2 + (i & 1)), ((i - 2) >> 1) & 1) && ok;    // the rows have read S(i - 2), and P(i - 2) is free
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
            const unsigned long long dV = smem_desc_sw128_mn(smem_u32(sV), KN * 128, 1024u);
            const unsigned d_o = tmem + S::O_COL + grp * D;
            for (int i = 0; i < n_mine; ++i) {
                const int t = tile_no(grp, i), st = t % STAGES;
                ok = mbar_wait(bar(S::B_V_FULL + st), (t / STAGES) & 1) && ok;
                ok = mbar_wait(bar(S::B_P + grp * 2 + (i & 1)), (i >> 1) & 1) && ok;
                fence_after_sync();
                const unsigned long long v_tile = dV + (unsigned long long)(st * (S::K_BYTES >> 4));
                const unsigned p_tile = tmem + (grp * 2 + (i & 1)) * KN;
#pragma unroll
                for (int k16 = 0; k16 < KN / 16; ++k16)       // 16 keys: eight columns of P, 2048 bytes down V
                    mma_ts(d_o, p_tile + k16 * 8, v_tile + (unsigned long long)(k16 * 128), idesc, i > 0 || k16 > 0);
                mma_commit(bar(S::B_PV + grp * 2 + (i & 1)));
                mma_commit(bar(S::B_V_EMPTY + st));
            }
        }
    } else if (warp >= W_LOAD) {
        // ================================================================== the loaders
        const bool is_k = warp == W_LOAD;
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
                    page[u] = j >= sg.lo && j <= sg.hi ? page_at(bt_row + pg.block(j), pages) : -1;
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
                        pool + (((size_t)next_page[u] * Hkv + kvh) * pg.page_size + pg.row((jt_begin + t) * KN + u * 32 + lane)) * head);
                const unsigned slab = (unsigned)(sub >> 3) * (KN * 128), c7 = (unsigned)(sub & 7);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int i = 0; i < 32 / RPI; ++i) {
                        const int owner = i * RPI + rsel, krow = u * 32 + owner;
                        const unsigned long long w = __shfl_sync(0xffffffffu, where[u], owner);
                        const bool there = w != 0ull && sub * 8 < head;
                        const bf16* src = there ? reinterpret_cast<const bf16*>(w) + sub * 8 : pool;
                        cp16u(tile_smem + (krow >> 3) * 1024 + (krow & 7) * 128 + slab + ((c7 ^ (unsigned)(krow & 7)) << 4), src, there);
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
    // The rows leave through shared memory, where K and V lay: each (group, copy) its outputs in float32, brought to the row's common maximum,
    // a row of D by 16-byte pieces, piece p of row x at p ^ (x % 8).
    float2* stats = reinterpret_cast<float2*>(sQ);            // [group][tile row]: maximum and sum
    float* row_inv = reinterpret_cast<float*>(stats + GROUPS * QM);
    float2* row_ml = reinterpret_cast<float2*>(row_inv + NQ * QM);      // what a cluster joins
    pdl_trigger_late();
    fence_before_sync();
    __syncthreads();                                          // no product reads shared memory any more
    fence_after_sync();
    if (has_rows) stats[grp * QM + r] = make_float2(m_ref, l_run);
    __syncthreads();
    const int groups = STREAMS && n_tiles == 1 ? 1 : GROUPS;  // STREAMS: those that have had a tile
    if (has_rows && n_mine > 0) {
        float mu = m_ref == -INFINITY ? 0.f : m_ref, mine = 1.f;
        if (STREAMS) {
            float top = -INFINITY;
            for (int g = 0; g < groups; ++g)
                for (int c = 0; c < copies; ++c) top = fmaxf(top, stats[g * QM + c * copy_rows + in_cta].x);
            mu = top == -INFINITY ? 0.f : top;
            mine = fast_exp2(m_ref - mu);
            if (grp == 0 && copy == 0) {
                l_run = 0.f;
                for (int g = 0; g < groups; ++g)
                    for (int c = 0; c < copies; ++c) {
                        const float2 f = stats[g * QM + c * copy_rows + in_cta];
                        l_run += f.y * fast_exp2(f.x - mu);
                    }
                m_ref = top;
            }
        }
        if (row_valid && (!STREAMS || (grp == 0 && copy == 0))) {
            const size_t at = token * Hq + h;
            if (sg.n_split > 1) *(joined ? row_ml + in_cta : reinterpret_cast<float2*>(part_ml + 2 * ((size_t)split * total_rows * Hq + at))) = make_float2(m_ref, l_run);
            else if (sink != nullptr) l_run += exp2f(sink[h] * LOG2E - mu);
            row_inv[in_cta] = l_run == 0.f ? 0.f : 1.f / l_run;
        }
        const bool odd = *odd_values != 0 && row_valid && (!STREAMS || (grp == 0 && copy == 0));
        unsigned char* slot = sK + (size_t)(grp * QM + r) * (D * 4);
        // where key j lies in the pools, -1: on no page; and its probability beside mu, from the operands
        auto key_at = [&](int j) {
            const int page = page_at(bt_row + pg.block(j), pages);
            return page < 0 ? -1ll : (((long long)page * Hkv + kvh) * pg.page_size + pg.row(j)) * head;
        };
        auto probability = [&](long long key) {
            float s = 0.f;
            const bf16* qrow = q + token * ld + (size_t)h * head;
            for (int d = 0; d < head; ++d) s = fmaf(__bfloat162float(qrow[d]), __bfloat162float(kpool[key + d]), s);
            s = CAP ? fast_tanh(s * (scale / softcap)) : s;
            return fast_exp2(fmaf(s, scale_eff, -mu));
        };
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
            unsigned o[32];
            __syncwarp();
            tmem_ld32(o_addr + c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * mine);
            auto any_odd = [&](long long key) {               // among these columns of a value
                unsigned any = 0u;
#pragma unroll
                for (int i = 0; i < 32; i += 2)
                    if (c0 + i < head) any |= odd_halves(*reinterpret_cast<const unsigned*>(vpool + key + c0 + i));
                return any != 0u;
            };
            if (STREAMS && copies > 1 && row_valid) {
                // A value that is no number in a tile that is seen in full is multiplied by zero in the copies whose key it is not: there such columns
                // become zero, and in the copy whose key it is what the definition gives.
                float none = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) none = fmaf(__uint_as_float(o[i]), 0.f, none);
                if (!(none == 0.f)) {
                    unsigned found = 0u;
                    for (int t = 0; t < n_mine; ++t) {
                        const int j_base = (jt_begin + tile_no(grp, t)) * KN;
                        if (!whole(j_base)) continue;
                        for (int j = 0; j < KN; ++j) {
                            const long long key = key_at(j_base + j);
                            if (key < 0 || !any_odd(key)) continue;
                            const bool own = j / (KN / copies) == copy;
                            const float p = own ? probability(key) : 0.f;
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const float v = c0 + i < head ? __bfloat162float(vpool[key + c0 + i]) : 0.f;
                                if (isfinite(v)) continue;
                                if (!(found >> i & 1u)) o[i] = 0u;
                                found |= 1u << i;
                                if (own) o[i] = __float_as_uint(fmaf(p, v, __uint_as_float(o[i])));
                            }
                        }
                    }
                }
            }
            if (odd) {
                // what the products left out: values that are no numbers, where this row sees their keys
                for (int t = 0; t < n_tiles; ++t) {
                    const int j_base = (jt_begin + t) * KN;
                    if (whole(j_base)) continue;
                    for (unsigned long long vis = visible(j_base); vis != 0ull; vis &= vis - 1ull) {
                        const long long key = key_at(j_base + __ffsll((long long)vis) - 1);
                        if (key < 0 || !any_odd(key)) continue;
                        const float p = probability(key);
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float v = c0 + i < head ? __bfloat162float(vpool[key + c0 + i]) : 0.f;
                            if (!isfinite(v)) o[i] = __float_as_uint(fmaf(p, v, __uint_as_float(o[i])));
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint4*>(slot + ((((c0 >> 2) + i) ^ (r & 7)) << 4)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
    }
    if (!ok) atomicExch(status, 1);
    fence_before_sync();
    __syncthreads();
    if (warp == W_ISSUE) tmem_dealloc(tmem, S::TMEM_COLS);
    // a row's partial outputs added, whole lines written: a thread four columns
    const bool parted = sg.n_split > 1;
    const int slots = STREAMS ? groups * copies : 1;
    auto place = [&](int x, int piece) { return (unsigned)(x * (D * 4) + ((piece ^ (x & 7)) << 4)); };
#pragma unroll 2
    for (int i = tid; i < rows * (D / 4); i += S::THREADS) {
        const int x = i / (D / 4), piece = i % (D / 4);
        if (4 * piece >= head) continue;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < slots; ++c) {                     // copies of a group lie side by side, groups QM apart
            const float4 f = *reinterpret_cast<const float4*>(sK + place(STREAMS ? c * copy_rows + x : x, piece));
            sum.x += f.x; sum.y += f.y; sum.z += f.z; sum.w += f.w;
        }
        if (parted && joined) {
            *reinterpret_cast<float4*>(sK + place(x, piece)) = sum;
            continue;
        }
        const int2 nh = by_group(row0 + x);
        const size_t at = (size_t)(sg.q_begin + nh.x) * Hq + kvh * G + nh.y;
        const float inv = row_inv[x];
        if (parted) *reinterpret_cast<float4*>(part_o + ((size_t)split * total_rows * Hq + at) * head + 4 * piece) = sum;
        else *reinterpret_cast<uint2*>(out + at * head + 4 * piece) = make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv));
    }
    if (!joined) return;
    __syncwarp();
    cluster_sync_all();
    if (parted) {                                             // each share takes a part of the pairs and goes through the shares in their order
        float* weight = reinterpret_cast<float*>(row_ml + NQ * QM);       // [share][row]
        static_assert(GROUPS * QM * 8 + NQ * QM * (4 + 8 + 4 * JOIN_MAX) <= NQ * S::Q_BYTES, "room for the weights in the place of Q");
        if (tid < rows) {
            float2 ml[JOIN_MAX];
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < JOIN_MAX; ++u) {
                ml[u] = make_float2(-INFINITY, 0.f);
                if (u < sg.n_split) ml[u] = peer_float2(map_to_cta(smem_u32(row_ml + tid), u));
            }
#pragma unroll
            for (int u = 0; u < JOIN_MAX; ++u) top = fmaxf(top, ml[u].x);
            const float ref = top == -INFINITY ? 0.f : top;
            float total = sink != nullptr ? exp2f(sink[kvh * G + by_group(row0 + tid).y] * LOG2E - ref) : 0.f;
#pragma unroll
            for (int u = 0; u < JOIN_MAX; ++u) {
                ml[u].x = ml[u].y == 0.f ? 0.f : exp2f(ml[u].x - ref);     // a share without keys for this row left nothing
                total = fmaf(ml[u].y, ml[u].x, total);
            }
            const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
            for (int u = 0; u < JOIN_MAX; ++u)
                if (u < sg.n_split) weight[u * (NQ * QM) + tid] = ml[u].x * inv;
        }
        __syncthreads();
        for (int i = split * S::THREADS + tid; i < rows * (D / 4); i += sg.n_split * S::THREADS) {
            const int x = i / (D / 4), piece = i % (D / 4);
            if (4 * piece >= head) continue;
            const unsigned at_sum = smem_u32(sK + place(x, piece));
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int u0 = 0; u0 < sg.n_split; u0 += 4) {
                float4 f[4];
                float w[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    w[u] = u0 + u < sg.n_split ? weight[(u0 + u) * (NQ * QM) + x] : 0.f;
                    if (u0 + u < sg.n_split) f[u] = peer_float4(map_to_cta(at_sum, u0 + u));
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (w[u] != 0.f) {
                        sum.x = fmaf(f[u].x, w[u], sum.x); sum.y = fmaf(f[u].y, w[u], sum.y);
                        sum.z = fmaf(f[u].z, w[u], sum.z); sum.w = fmaf(f[u].w, w[u], sum.w);
                    }
            }
            const int2 nh = by_group(row0 + x);
            *reinterpret_cast<uint2*>(out + ((size_t)(sg.q_begin + nh.x) * Hq + kvh * G + nh.y) * head + 4 * piece) =
                make_uint2(pack_bf16(sum.x, sum.y), pack_bf16(sum.z, sum.w));
        }
    }
    __syncwarp();
    cluster_sync_all();                                       // nobody leaves before its outputs have been read
}

// out[row, h] = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the shares of the keys, in their order: one warp a (node, head).  All
// maxima and sums are asked for at once (a lane a share), then the shares' rows eight at a time: about two trips to memory.  Bound by the launch and
// those trips: 2.9 us behind its producer for 16 shares of 128 rows, 0.06 us a share more.
// grid: (nodes of the longest tree x Hq / 8, segments).  VEC: values of a row that lie together in a lane.
template <typename TA, int VEC>
__global__ void __launch_bounds__(256)
tree_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ cu_q,
                  const int* __restrict__ seg_pos0, int total_rows, int Hq, int D, int window, int share, int max_split,
                  TA* __restrict__ out, const float* __restrict__ sink) {
    constexpr int RUNS = TREE_MAX_D / 32 / VEC, AT_ONCE = VEC == 4 ? 8 : 2;      // VEC 4: heads up to 128
    constexpr int USED = VEC == 4 ? 1 : RUNS;
    pdl_wait();
    const Segment sg(cu_q, seg_pos0, blockIdx.y, window, share, max_split);
    const int pair = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (pair >= sg.n * Hq || sg.n_split == 1) return;         // one share: its CTA wrote the row
    const int h = pair % Hq;
    const size_t at = (size_t)sg.q_begin * Hq + pair, stride = (size_t)total_rows * Hq;
    static_assert(TREE_MAX_SPLITS <= 64, "two shares a lane");
    float2 ml[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
        ml[u] = lane + 32 * u < sg.n_split ? *reinterpret_cast<const float2*>(part_ml + 2 * ((lane + 32 * u) * stride + at)) : make_float2(-INFINITY, 0.f);
    const float top = warp_max(fmaxf(ml[0].x, ml[1].x)), ref = top == -INFINITY ? 0.f : top;
    float w[2];                                               // a share without keys for this row left no output: weight 0, nothing is read
#pragma unroll
    for (int u = 0; u < 2; ++u) w[u] = ml[u].y == 0.f ? 0.f : exp2f(ml[u].x - ref);
    float l = warp_sum(ml[0].y * w[0] + ml[1].y * w[1]);
    if (sink != nullptr) l += exp2f(sink[h] * LOG2E - ref);
    float acc[USED][VEC];
#pragma unroll
    for (int i = 0; i < USED; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[i][k] = 0.f;
    for (int s0 = 0; s0 < sg.n_split; s0 += AT_ONCE) {
        float o[AT_ONCE][USED][VEC], ws[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int s = s0 + u;
            ws[u] = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[1], s & 31);
            if (s >= sg.n_split) ws[u] = 0.f;
#pragma unroll
            for (int i = 0; i < USED; ++i) {
                const int d = VEC * (lane + 32 * i);
                const float* from = part_o + (s * stride + at) * D + d;
#pragma unroll
                for (int k = 0; k < VEC; ++k) o[u][i][k] = 0.f;
                if (ws[u] != 0.f && d < D) {
                    if (VEC == 4) {
                        const float4 f = *reinterpret_cast<const float4*>(from);
                        o[u][i][0] = f.x; o[u][i][VEC > 1 ? 1 : 0] = f.y; o[u][i][VEC > 2 ? 2 : 0] = f.z; o[u][i][VEC > 3 ? 3 : 0] = f.w;
                    } else {
                        o[u][i][0] = *from;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int i = 0; i < USED; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[i][k] = ws[u] != 0.f ? fmaf(o[u][i][k], ws[u], acc[i][k]) : acc[i][k];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < USED; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const int d = VEC * (lane + 32 * i) + k;
            if (d < D) out[at * D + d] = from_f32<TA>(acc[i][k] * inv);
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
    bool joined;
    float *scratch, *part_ml;
    int* status;
    cudaStream_t st;
};

// A launch whose shares of a block of rows are a cluster, if they join their outputs themselves.
template <typename... KArgs, typename... Args>
int launch(const TreeCall& a, void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, Args... args) {
    if (!a.joined) return rb_launch_pdl(kernel, grid, dim3(threads), smem, a.st, args...);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = a.st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = (unsigned)a.splits;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = RB_PDL_MODE == 3 ? 1 : 2;
    return (int)cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

template <typename TA>
int merge(const TreeCall& a) {
    if (a.splits <= 1 || a.joined) return 0;
    dim3 grid((a.max_nodes * a.Hq + 7) / 8, a.segments);
    return rb_launch_pdl(a.D % 4 == 0 && a.D <= 128 ? tree_merge_kernel<TA, 4> : tree_merge_kernel<TA, 1>, grid, dim3(256), 0, a.st, a.scratch, a.part_ml, a.cu_q, a.seg_pos0, a.total_rows, a.Hq, a.D,
                         a.window, a.share, a.splits, (TA*)a.out, a.sink);
}

template <typename TA, int DP>
int mma_launch(const TreeCall& a) {
    constexpr int SMEM = (int)MmaShape<TA, DP>::SMEM;
    static PerDevice configured;
    const int rc = configured.once([&](int) { return cudaFuncSetAttribute(tree_mma_kernel<TA, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
    if (rc) return rc;
    const int vec = a.D * sizeof(TA) % 16 == 0 && (((uintptr_t)a.kpool | (uintptr_t)a.vpool) & 15) == 0;
    dim3 grid((a.max_nodes * (a.Hq / a.Hkv) + MROWS - 1) / MROWS * a.Hkv, a.segments, a.splits);
    const int e = launch(a, tree_mma_kernel<TA, DP>, grid, MTHREADS, SMEM, (const TA*)a.q, a.ld, (const TA*)a.kpool,
                                (const TA*)a.vpool, a.cu_q, a.seg_pos0, a.parent, a.block_table, a.bt_stride, a.page_size, a.pages, (TA*)a.out, a.scratch,
                                a.part_ml, a.total_rows, a.Hq, a.Hkv, a.D, a.scale, a.window, a.softcap, a.sink, a.splits > 1 ? a.share : 0, (int)a.joined, vec);
    return e ? e : merge<TA>(a);
}
template <typename TA>
int mma_any(const TreeCall& a) {
    if (a.D <= 32) return mma_launch<TA, 32>(a);
    if (a.D <= 64) return mma_launch<TA, 64>(a);
    return a.D <= 128 ? mma_launch<TA, 128>(a) : mma_launch<TA, 256>(a);
}

template <int D, bool STREAMS, bool CAP, bool WHOLE>
int tc5_kernel_launch(const TreeCall& a) {
    typedef Shape<D, STREAMS> S;
    constexpr int ROWS = S::NQ * QM;
    static PerDevice configured;
    const int rc = configured.once([&](int) {
        return cudaFuncSetAttribute(tree_tc5_kernel<D, STREAMS, CAP, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
    });
    if (rc) return rc;
    // pages are whole boxes of whole groups of eight rows, and their rows can be counted in 31 bits
    const long long pool_rows = (long long)a.pages * a.Hkv * a.page_size;
    int by_tma = a.page_size % 8 == 0 && (KN % a.page_size == 0 || a.page_size % KN == 0) && pool_rows <= 0x7fffffffll;
    CUtensorMap kmap = {}, vmap = {};
    const int box = a.page_size < KN ? a.page_size : KN;
    if (by_tma && !(tma::make_map_bf16(&kmap, a.kpool, (int)pool_rows, a.D, a.D, box) && tma::make_map_bf16(&vmap, a.vpool, (int)pool_rows, a.D, a.D, box)))
        return (int)cudaErrorInvalidValue;
    dim3 grid((a.max_nodes * (a.Hq / a.Hkv) + ROWS - 1) / ROWS * a.Hkv, a.segments, a.splits);
    const int e = launch(a, tree_tc5_kernel<D, STREAMS, CAP, WHOLE>, grid, S::THREADS, S::SMEM, (const bf16*)a.q, a.ld, (const bf16*)a.kpool,
                                (const bf16*)a.vpool, a.cu_q, a.seg_pos0, a.parent, a.block_table, a.bt_stride, a.page_size, a.pages, (bf16*)a.out, a.scratch,
                                a.part_ml, a.total_rows, a.Hq, a.Hkv, a.D, a.scale, a.window, a.softcap, a.sink, a.splits > 1 ? a.share : 0, (int)a.joined, a.status, by_tma, kmap, vmap);
    return e ? e : merge<bf16>(a);
}

template <int D, bool STREAMS>
int tc5_launch(const TreeCall& a) {
    if (a.D == D) return a.softcap > 0.f ? tc5_kernel_launch<D, STREAMS, true, true>(a) : tc5_kernel_launch<D, STREAMS, false, true>(a);
    return a.softcap > 0.f ? tc5_kernel_launch<D, STREAMS, true, false>(a) : tc5_kernel_launch<D, STREAMS, false, false>(a);
}

}  // namespace

RB_EXPORT int rb_tree_max_nodes() { return TREE_MAX_NODES; }
RB_EXPORT int rb_tree_max_splits() { return TREE_MAX_SPLITS; }
RB_EXPORT int rb_tree_join_max() { return JOIN_MAX; }

// q: rotated queries, row stride ld.  max_nodes: the longest segment's nodes (TREE_MAX_NODES at most).  splits > 1: a segment's keys
// go to one CTA for every `share` key tiles of 64, `splits` at most, which are a cluster and join their outputs if `joined` (JOIN_MAX at most); else scratch holds
// splits * total_rows * Hq * D floats for their outputs, on a 16-byte boundary, and scratch_ml splits * total_rows * Hq pairs of a maximum and a sum, on one of 8.
// query_tiles: 0 the kernel for any type and head size; 1 or 2 the tcgen05 kernel with so many tiles of 128 rows a CTA (bfloat16, D and ld multiples
// of 8, one tile beyond 128; pools, queries and out on 16-byte boundaries).  *status is raised if a wait gave up.
RB_EXPORT int rb_tree_attention(const void* q, int ld, const void* kpool, const void* vpool, const int* cu_q, const int* seg_pos0,
                                const int* parent, const int* block_table, int bt_stride, int page_size, int pages, void* out, int act_dtype,
                                int segments, int max_nodes, int total_rows, int Hq, int Hkv, int D, float scale, int window,
                                float softcap, const float* sink, int splits, int share, int joined, void* scratch, void* scratch_ml, int query_tiles, int* status,
                                cudaStream_t st) {
    if (segments <= 0 || max_nodes <= 0) return 0;
    if (segments > 65535 || max_nodes > TREE_MAX_NODES || D <= 0 || D > TREE_MAX_D || Hkv <= 0 || Hq % Hkv || page_size <= 0) return (int)cudaErrorInvalidValue;
    if (splits < 1 || splits > TREE_MAX_SPLITS || (splits > 1 && (share <= 0 || (joined ? splits > JOIN_MAX : scratch == nullptr || scratch_ml == nullptr))))
        return (int)cudaErrorInvalidValue;
    if (((uintptr_t)scratch & 15) || ((uintptr_t)scratch_ml & 7)) return (int)cudaErrorInvalidValue;
    TreeCall a = {q, kpool, vpool, ld, cu_q, seg_pos0, parent, block_table, bt_stride, page_size, out, segments, max_nodes, total_rows, Hq, Hkv,
                  D, pages, scale, window, softcap, sink, splits, share, joined && splits > 1, (float*)scratch, (float*)scratch_ml, status, st};
    if (query_tiles > 0) {
        if (act_dtype != RB_BF16 || D % 8 || query_tiles > (D > 128 ? 1 : 2) || status == nullptr) return (int)cudaErrorInvalidValue;
        if ((((uintptr_t)q | (uintptr_t)kpool | (uintptr_t)vpool | (uintptr_t)out) & 15) || ld % 8) return (int)cudaErrorInvalidValue;
        if (D > 128) return tc5_launch<256, true>(a);
        if (D <= 64) return query_tiles == 1 ? tc5_launch<64, true>(a) : tc5_launch<64, false>(a);
        return query_tiles == 1 ? tc5_launch<128, true>(a) : tc5_launch<128, false>(a);
    }
    return act_dtype == RB_F32 ? mma_any<float>(a) : mma_any<bf16>(a);
}
