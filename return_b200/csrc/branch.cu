// What happens in the cache when a request is carried on along several lines: the accepted nodes of a drafted tree move up
// (tree_commit), a page's first rows are copied to another page for a second line (copy_pages), and so is a request's
// fixed-size state from slot to slot (copy_slots).
//
// A pool holds all layers of a group: [planes, pages, heads, page_size, row], planes = layers x (keys, values), or layers for a cache of
// latents (one head).  A row (a token's key of one head) is row_bytes long.  Everything here is moved as bytes, 16 at a time where rows
// and pools allow it, else two (the smallest element that is cached).
#include "pairs.cuh"

#define TREE_MAX_NODES 256
#define SLOT_TENSORS 64

namespace {

template <int W> struct Piece;
template <> struct Piece<16> { typedef uint4 type; };
template <> struct Piece<4> { typedef unsigned type; };
template <> struct Piece<2> { typedef unsigned short type; };
template <> struct Piece<1> { typedef unsigned char type; };

// ---------------------------------------------------------------------------------------- the commit of a drafted tree
// Which nodes hold: from the root (node 0) on, the child whose token is the one that was sampled behind the node, the lowest such child
// where a tree names a token twice.  One warp; path and the return value (how many nodes) are for every lane of it.
__device__ int walk_tree(const int* token, const int* parent, const int* sampled, int n, int* path, int lane) {
    int x = 0, count = 0;
    while (true) {
        if (lane == 0) path[count] = x;
        ++count;
        const int want = sampled[x];
        int best = TREE_MAX_NODES;
        for (int y0 = x + 1; y0 < n; y0 += 32) {              // a child comes behind its parent
            const int y = y0 + lane;
            const unsigned hit = __ballot_sync(0xffffffffu, y < n && parent[y] == x && token[y] == want);
            if (hit) {
                best = y0 + __ffs(hit) - 1;
                break;
            }
        }
        if (best == TREE_MAX_NODES) return count;
        x = best;                                             // x grows: the walk ends
    }
}

constexpr int COMMIT_THREADS = 256;
constexpr int MOVES_AT_ONCE = 8;

// grid: (segments, parts of the planes x heads).  Node path[i] moves from slot c + path[i] to slot c + i.  LPR lanes share a row's pieces; a
// thread keeps to its piece of a (plane, head) and goes through the moves in order, eight loads before their stores.  No store meets a row
// that is still to be read: path[k] >= k, so a later move's source lies behind every earlier move's destination.
// Bound by two trips to memory (tables, rows) where little moves: 8 nodes, 28 layers, 3.5 us.  64 requests of which six tokens hold, 36 layers of 8 key heads
// of 128, 75 MB read and written: 17.8 us from HBM, 4.2 TB/s of rows of 256 bytes that lie anywhere, and 10.7 where the rows lie in L2.
// The walk is done by every CTA for itself (a few hundred cycles); the first part writes it down.  What it takes is asked for at once, the
// part of the block table that the tree lies on with it.
template <int W>
__global__ void __launch_bounds__(COMMIT_THREADS)
tree_commit_kernel(const int* __restrict__ tokens, const int* __restrict__ tree_parent, const int* __restrict__ sampled,
                   const int* __restrict__ cu_q, const int* __restrict__ seg_pos0, const int* __restrict__ block_table, int bt_stride,
                   int page_size, unsigned char* __restrict__ pool, int planes, long long pages, int heads, int row_bytes, int lpr_log, int per_cta,
                   int* __restrict__ path_out, int* __restrict__ count_out, int* __restrict__ emitted_out, int width) {
    typedef typename Piece<W>::type P;
    __shared__ int s_token[TREE_MAX_NODES], s_parent[TREE_MAX_NODES], s_sampled[TREE_MAX_NODES], s_path[TREE_MAX_NODES];
    __shared__ int s_page[TREE_MAX_NODES + 1];                // of the blocks that the tree lies on, from its first slot's
    __shared__ int s_count;
    __shared__ long long s_src[TREE_MAX_NODES], s_dst[TREE_MAX_NODES];        // rows of head 0 in a plane, -1: nothing moves
    pdl_wait();
    const int seg = blockIdx.x, tid = threadIdx.x;
    const int q_begin = cu_q[seg], n = min(cu_q[seg + 1] - q_begin, TREE_MAX_NODES), c = seg_pos0[seg];
    const int block0 = c / page_size, blocks = pool != nullptr && n > 0 ? (c + n - 1) / page_size - block0 + 1 : 0;
    for (int i = tid; i < n; i += COMMIT_THREADS) {
        s_token[i] = tokens[q_begin + i];
        s_parent[i] = tree_parent[q_begin + i];
        s_sampled[i] = sampled[q_begin + i];
    }
    for (int i = tid; i < blocks; i += COMMIT_THREADS) s_page[i] = block_table[(size_t)seg * bt_stride + block0 + i];
    __syncthreads();
    if (tid < 32) {
        const int count = n > 0 ? walk_tree(s_token, s_parent, s_sampled, n, s_path, tid) : 0;
        if (tid == 0) s_count = count;
    }
    __syncthreads();
    const int count = s_count;
    if (blockIdx.y == 0 && path_out != nullptr) {
        for (int i = tid; i < width; i += COMMIT_THREADS) {
            const int x = i < count ? s_path[i] : -1;
            path_out[(size_t)seg * width + i] = x;
            emitted_out[(size_t)seg * width + i] = x >= 0 ? s_sampled[x] : -1;
        }
        if (tid == 0) count_out[seg] = count;
    }
    if (pool == nullptr) return;
    for (int i = tid; i < count; i += COMMIT_THREADS) {
        const int from = c + s_path[i], to = c + i;
        long long src = -1, dst = -1;
        if (from != to) {
            const int ps = s_page[from / page_size - block0], pd = s_page[to / page_size - block0];
            if (ps >= 0 && pd >= 0 && ps < pages && pd < pages) {
                src = (long long)ps * heads * page_size + from % page_size;
                dst = (long long)pd * heads * page_size + to % page_size;
            }
        }
        s_src[i] = src * row_bytes;
        s_dst[i] = dst * row_bytes;
    }
    __syncthreads();
    int first = 1;                                            // the moves begin behind the nodes that lie in place
    while (first < count && s_src[first] < 0) ++first;
    if (first >= count) return;
    const ByDivisor by_heads(heads);
    const int lpr = 1 << lpr_log, pair_end = min(planes * heads, ((int)blockIdx.y + 1) * per_cta);
    const long long plane_bytes = pages * heads * page_size * row_bytes, head_bytes = (long long)page_size * row_bytes;
    for (int pair = (int)blockIdx.y * per_cta + (tid >> lpr_log); pair < pair_end; pair += COMMIT_THREADS >> lpr_log) {
        const int2 at = by_heads(pair);                       // plane, head
        unsigned char* head = pool + at.x * plane_bytes + at.y * head_bytes;
        for (int byte = (tid & (lpr - 1)) * W; byte < row_bytes; byte += lpr * W) {
            unsigned char* base = head + byte;
            for (int i0 = first; i0 < count; i0 += MOVES_AT_ONCE) {
                P v[MOVES_AT_ONCE];
#pragma unroll
                for (int u = 0; u < MOVES_AT_ONCE; ++u)
                    if (i0 + u < count && s_src[i0 + u] >= 0) v[u] = *reinterpret_cast<const P*>(base + s_src[i0 + u]);
#pragma unroll
                for (int u = 0; u < MOVES_AT_ONCE; ++u)
                    if (i0 + u < count && s_src[i0 + u] >= 0) *reinterpret_cast<P*>(base + s_dst[i0 + u]) = v[u];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------- copies
constexpr int COPY_THREADS = 256, COPY_UNROLL = 4;

// n bytes from src to dst by the threads of a CTA, COPY_UNROLL loads of each thread before their stores.
template <int W>
__device__ __forceinline__ void copy_bytes(unsigned char* dst, const unsigned char* src, long long n, int tid) {
    typedef typename Piece<W>::type P;
    const P* s = reinterpret_cast<const P*>(src);
    P* d = reinterpret_cast<P*>(dst);
    const long long m = n / W;
    for (long long i0 = 0; i0 < m; i0 += COPY_THREADS * COPY_UNROLL) {
        P v[COPY_UNROLL];
#pragma unroll
        for (int u = 0; u < COPY_UNROLL; ++u) {
            const long long i = i0 + u * COPY_THREADS + tid;
            if (i < m) v[u] = s[i];
        }
#pragma unroll
        for (int u = 0; u < COPY_UNROLL; ++u) {
            const long long i = i0 + u * COPY_THREADS + tid;
            if (i < m) d[i] = v[u];
        }
    }
}

// The first rows[i] rows of page src[i] to page dst[i], in every plane and head.  A head's rows of a page lie together, so a (plane, head) is
// one run of bytes; a warp takes one at a time, eight loads of a lane before their stores.  Bound by HBM: 72 copies over 36 layers of 8 key heads of 128,
// 178 MB read and written, 33 us, 5.4 TB/s; four copies over 28 layers 2.4 us, the launch and a trip to memory.
// grid: (copies, parts of the planes x heads).
template <int W>
__global__ void __launch_bounds__(COPY_THREADS)
copy_pages_kernel(unsigned char* __restrict__ pool, const int* __restrict__ src, const int* __restrict__ dst, const int* __restrict__ rows,
                  int planes, int pages, int heads, int page_size, int row_bytes, int per_cta) {
    typedef typename Piece<W>::type P;
    constexpr int AT_ONCE = 8;
    pdl_wait();
    const int i = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int from = src[i], to = dst[i], n = min(rows[i], page_size);
    if (from < 0 || to < 0 || from >= pages || to >= pages || from == to || n <= 0) return;
    const int pair_end = min(planes * heads, ((int)blockIdx.y + 1) * per_cta);
    const int bytes = n * row_bytes;                          // of one (plane, head)
    const long long run = (long long)page_size * row_bytes, page = run * heads, plane = page * pages, step = (to - from) * page;
    const ByDivisor by_heads(heads);
    for (int pair = (int)blockIdx.y * per_cta + warp; pair < pair_end; pair += COPY_THREADS / 32) {
        const int2 at = by_heads(pair);                       // plane, head
        unsigned char* head = pool + at.x * plane + at.y * run + from * page;
        for (int b0 = lane * W; b0 < bytes; b0 += 32 * W * AT_ONCE) {
            P v[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
                if (b0 + u * 32 * W < bytes) v[u] = *reinterpret_cast<const P*>(head + b0 + u * 32 * W);
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
                if (b0 + u * 32 * W < bytes) *reinterpret_cast<P*>(head + step + b0 + u * 32 * W) = v[u];
        }
    }
}

struct SlotTensors {
    unsigned char* at[SLOT_TENSORS];
    long long row_bytes[SLOT_TENSORS];
};
constexpr long long SLOT_CHUNK = 32768;       // bytes of a row that a CTA copies

// Row src[i] to row dst[i] of every tensor.  grid: (pieces of the longest row, tensors, copies).  Bound by HBM: 32 copies in eight tensors of 1 MB a row
// 80 us, the rate of a plain copy; three copies of 0.5 MB 6.3 us, 4.1 where they lie in L2.
__global__ void __launch_bounds__(COPY_THREADS)
copy_slots_kernel(const SlotTensors t, const int* __restrict__ src, const int* __restrict__ dst, int slots) {
    const int from = src[blockIdx.z], to = dst[blockIdx.z];
    if (from < 0 || to < 0 || from >= slots || to >= slots || from == to) return;
    const long long row = t.row_bytes[blockIdx.y], begin = blockIdx.x * SLOT_CHUNK, n = min(SLOT_CHUNK, row - begin);
    if (n <= 0) return;
    unsigned char* base = t.at[blockIdx.y];
    const unsigned char* s = base + from * row + begin;
    unsigned char* d = base + to * row + begin;
    const unsigned long long low = (unsigned long long)base | (unsigned long long)row;
    if ((low & 15) == 0) copy_bytes<16>(d, s, n, threadIdx.x);
    else if ((low & 3) == 0) copy_bytes<4>(d, s, n, threadIdx.x);
    else copy_bytes<1>(d, s, n, threadIdx.x);
}

// How many (plane, head) pairs a CTA takes: so many that `first` x parts CTAs give every SM `per_sm`, which is as many as it holds, a multiple of `unit`.
int pairs_per_cta(int first, int pairs, int unit, int per_sm) {
    const int want = rb_num_sms() * per_sm;
    const long long parts = first >= want ? 1 : want / first;
    long long per = (pairs + parts - 1) / parts;
    per = (per + unit - 1) / unit * unit;
    return (int)(per < unit ? unit : per);
}

}  // namespace

RB_EXPORT int rb_slot_tensors() { return SLOT_TENSORS; }
RB_EXPORT int rb_commit_max_nodes() { return TREE_MAX_NODES; }

// pool null: the walk alone.  path_out null: no walk is written down (a second group's cache of the same step).
RB_EXPORT int rb_tree_commit(const int* tokens, const int* parent, const int* sampled, const int* cu_q, const int* seg_pos0, int segments,
                             const int* block_table, int bt_stride, int page_size, void* pool, int planes, int pages, int heads,
                             int row_bytes, int* path_out, int* count_out, int* emitted_out, int width, cudaStream_t st) {
    if (segments <= 0) return 0;
    if (pool != nullptr && (planes <= 0 || heads <= 0 || page_size <= 0 || row_bytes <= 0 || row_bytes % 2)) return (int)cudaErrorInvalidValue;
    const bool wide = ((uintptr_t)pool & 15) == 0 && row_bytes % 16 == 0;
    const int pairs = pool != nullptr ? planes * heads : 1, W = wide ? 16 : 2;
    int lpr_log = 0;                                          // lanes that share a row
    while ((W << lpr_log) < row_bytes && lpr_log < 5) ++lpr_log;
    const int per_cta = pairs_per_cta(segments, pairs, COMMIT_THREADS >> lpr_log, 4);
    dim3 grid(segments, (pairs + per_cta - 1) / per_cta);
    if (grid.y > 65535 || pairs > (1 << 22)) return (int)cudaErrorInvalidValue;      // what ByDivisor takes
    auto kernel = wide ? tree_commit_kernel<16> : tree_commit_kernel<2>;
    return rb_launch_pdl(kernel, grid, dim3(COMMIT_THREADS), 0, st, tokens, parent, sampled, cu_q, seg_pos0, block_table, bt_stride, page_size,
                         (unsigned char*)pool, planes, (long long)pages, heads, row_bytes, lpr_log, per_cta, path_out, count_out, emitted_out, width);
}

RB_EXPORT int rb_copy_pages(void* pool, const int* src, const int* dst, const int* rows, int copies, int planes, int pages, int heads,
                            int page_size, int row_bytes, cudaStream_t st) {
    if (copies <= 0) return 0;
    if (planes <= 0 || heads <= 0 || page_size <= 0 || row_bytes <= 0 || row_bytes % 2) return (int)cudaErrorInvalidValue;
    const bool wide = ((uintptr_t)pool & 15) == 0 && row_bytes % 16 == 0;
    if ((long long)page_size * row_bytes > (1ll << 30) || planes * (long long)heads > (1 << 22)) return (int)cudaErrorInvalidValue;
    const int per_cta = pairs_per_cta(copies, planes * heads, COPY_THREADS / 32, 4);
    dim3 grid(copies, (planes * heads + per_cta - 1) / per_cta);
    if (grid.y > 65535) return (int)cudaErrorInvalidValue;
    auto kernel = wide ? copy_pages_kernel<16> : copy_pages_kernel<2>;
    return rb_launch_pdl(kernel, grid, dim3(COPY_THREADS), 0, st, (unsigned char*)pool, src, dst, rows, planes, pages, heads, page_size, row_bytes, per_cta);
}

// tensors: host array of `count` addresses and then `count` row lengths in bytes.
RB_EXPORT int rb_copy_slots(const long long* tensors, int count, const int* src, const int* dst, int copies, int slots, cudaStream_t st) {
    if (copies <= 0) return 0;
    if (copies > 65535) return (int)cudaErrorInvalidValue;
    for (int t0 = 0; t0 < count; t0 += SLOT_TENSORS) {
        SlotTensors t = {};
        const int n = count - t0 < SLOT_TENSORS ? count - t0 : SLOT_TENSORS;
        long long longest = 0;
        for (int i = 0; i < n; ++i) {
            t.at[i] = (unsigned char*)tensors[t0 + i];
            t.row_bytes[i] = tensors[count + t0 + i];
            if (t.row_bytes[i] > longest) longest = t.row_bytes[i];
        }
        if (longest <= 0) continue;
        dim3 grid((unsigned)((longest + SLOT_CHUNK - 1) / SLOT_CHUNK), n, copies);
        copy_slots_kernel<<<grid, COPY_THREADS, 0, st>>>(t, src, dst, slots);
        const int e = rb_launch_status();
        if (e) return e;
    }
    return 0;
}
