// Embedding lookup with scaling and the gradient of the table.
//
//   z[i, :] = scale * table[t_i, :]          grad[v, :] (+)= scale * sum over i with t_i = v of dz[i, :]
//
// A token below 0 is padding: its row of z is zero. A token at or beyond the table's end gives a row of NaN: nothing is
// read out of range and the mistake stays visible. Neither takes part in the gradient.
//
// The lookup is a copy of rows, bound by HBM (or by L2, where tokens repeat). The gradient adds up rows that stand
// anywhere: with atomics its value would depend on their order, and the frequent tokens of a text (one in sixteen is the
// commonest) would queue up on a few addresses. So the (token, position) pairs are sorted first, stably, which puts the
// rows of a token next to each other in the order of their positions; the sorted list is cut into chunks of equal
// length, a group of threads walks a chunk and writes every run that ends inside it, and a run that crosses a chunk's
// end leaves partial sums, which a last launch folds in order. The result is the same bits on every run. Sums are held
// in float (double for double data) and rounded once, after scaling and, where asked for, adding what grad holds.
//
// The sort is a least-significant-digit radix sort with digits of up to 9 bits: two passes up to a table of 2^18 rows.
// Up to 65536 tokens one cluster of CTAs does all passes in one launch, the counts travelling through distributed
// shared memory; the other CTAs of that launch write the zeros of the table meanwhile. Longer lists take three launches
// per pass.
#include "../../include/nd4j_b200.h"
#include <cooperative_groups.h>
#include "device_utils.cuh"
#include "entry_checks.h"

namespace cg = cooperative_groups;

namespace nd4jb200 {
namespace {

// ---- the order of the tokens -------------------------------------------------------------------------------------
constexpr int kOrdThreads = 1024;
constexpr int kOrdWarps = kOrdThreads / 32;
constexpr int kOrdKeys = 8;                                   // per thread
constexpr int kOrdTile = kOrdThreads * kOrdKeys;
constexpr int kOrdBits = 9;
constexpr int kOrdBins = 1 << kOrdBits;
constexpr int kOrdCluster = 8;

struct OrderArgs {
    const LL *tokens;
    unsigned *key[2], *pos[2];       // ping-pong; `result` says which pair holds the sorted list
    unsigned n;
    unsigned vocab;                  // key of a token that takes no part: sorts behind all others
    int bits;                        // per digit
    int passes;
    unsigned *hist;                  // long lists: [tile][kOrdBins]
    unsigned tiles;
    // table rows to be zeroed beside the sort (one-launch form)
    void *zero;
    LL zeroRows, zeroRow, zeroCol;   // rows, and element strides
    LL cols;
    int zeroWords;                   // 128-bit words per row, 0: element by element
    int sortCtas;
};

struct OrderShared {
    unsigned short count[kOrdWarps][kOrdBins];   // per warp and digit: keys so far, then the tile-local start
    unsigned total[kOrdBins];                    // the tile's keys per digit (read by the other CTAs of a cluster)
    unsigned base[kOrdBins];                     // where the tile's first key of the digit goes, less its local start
    unsigned warpSums[kOrdWarps];
};

ND_D unsigned order_key(const OrderArgs &a, LL token) { return token >= 0 && token < (LL) a.vocab ? (unsigned) token : a.vocab; }

// Warp w holds the tile's keys [w * 256, w * 256 + 256), round r of it the next 32: "earlier" is (warp, round, lane).
ND_D unsigned order_index(unsigned tile, int r) {
    return tile * kOrdTile + (threadIdx.x >> 5) * (32 * kOrdKeys) + r * 32 + (threadIdx.x & 31);
}
ND_D void order_read(const OrderArgs &a, int pass, unsigned tile, unsigned (&key)[kOrdKeys], unsigned (&pos)[kOrdKeys]) {
#pragma unroll
    for (int r = 0; r < kOrdKeys; r++) {
        const unsigned i = order_index(tile, r);
        key[r] = pos[r] = 0;
        if (i < a.n) {
            if (pass == 0) { key[r] = order_key(a, a.tokens[i]); pos[r] = i; }
            // written by other SMs in the pass before: from L2, where they meet
            else { key[r] = __ldcg(a.key[(pass - 1) & 1] + i); pos[r] = __ldcg(a.pos[(pass - 1) & 1] + i); }
        }
    }
}

// Exclusive prefix sum over the CTA's threads.
ND_D unsigned order_scan(unsigned v, unsigned *warpSums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += t;
    }
    if (lane == 31) warpSums[warp] = inc;
    __syncthreads();
    unsigned w = warpSums[lane], before = w;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += t;
    }
    before = __shfl_sync(0xffffffffu, before - w, warp);
    __syncthreads();
    return before + inc - v;
}

// Rank of every key among the warp's earlier keys of its digit, and the tile's counts. Afterwards count[w][d] is the
// number of the tile's keys of digit d in the warps before w, total[d] that of the tile.
ND_D void order_rank(const OrderArgs &a, int pass, unsigned tile, const unsigned (&key)[kOrdKeys], unsigned (&rank)[kOrdKeys],
                     OrderShared &s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned *words = reinterpret_cast<unsigned *>(&s.count[0][0]);
    for (int i = threadIdx.x; i < kOrdWarps * kOrdBins / 2; i += kOrdThreads) words[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kOrdKeys; r++) {
        const bool valid = order_index(tile, r) < a.n;
        const unsigned d = valid ? (key[r] >> (pass * a.bits)) & ((1u << a.bits) - 1u) : 0xffffffffu;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const unsigned earlier = __popc(peers & ((1u << lane) - 1u));
        unsigned before = 0;
        if (valid) before = s.count[warp][d];
        __syncwarp();
        if (valid && earlier == 0) s.count[warp][d] = (unsigned short) (before + __popc(peers));
        __syncwarp();
        rank[r] = before + earlier;
    }
    __syncthreads();
    if (threadIdx.x < kOrdBins) {
        unsigned run = 0;
#pragma unroll 8
        for (int w = 0; w < kOrdWarps; w++) {
            const unsigned c = s.count[w][threadIdx.x];
            s.count[w][threadIdx.x] = (unsigned short) run;
            run += c;
        }
        s.total[threadIdx.x] = run;
    }
    __syncthreads();
}

ND_D void order_write(const OrderArgs &a, int pass, unsigned tile, const unsigned (&key)[kOrdKeys], const unsigned (&pos)[kOrdKeys],
                      const unsigned (&rank)[kOrdKeys], const OrderShared &s) {
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int r = 0; r < kOrdKeys; r++) {
        if (order_index(tile, r) < a.n) {
            const unsigned d = (key[r] >> (pass * a.bits)) & ((1u << a.bits) - 1u);
            const unsigned to = s.base[d] + s.count[warp][d] + rank[r];
            __stcg(a.key[pass & 1] + to, key[r]);
            __stcg(a.pos[pass & 1] + to, pos[r]);
        }
    }
}

// One element of T that is zero in every type.
template <class T> ND_D void zero_rows(const OrderArgs &a, LL first, LL step) {
    T *z = static_cast<T *>(a.zero);
    if (a.zeroWords > 0 && a.zeroRow == a.cols) {              // one run
        const LL words = a.zeroRows * a.zeroWords;
        uint4 *p = reinterpret_cast<uint4 *>(z);
        for (LL i = first; i < words; i += step) __stcs(p + i, make_uint4(0, 0, 0, 0));
        return;
    }
    const LL perRow = a.zeroWords > 0 ? a.zeroWords : a.cols;
    for (LL i = first; i < a.zeroRows * perRow; i += step) {
        const LL row = i / perRow, c = i - row * perRow;
        if (a.zeroWords > 0) *reinterpret_cast<uint4 *>(z + row * a.zeroRow + c * Elem<T>::kVec) = make_uint4(0, 0, 0, 0);
        else z[row * a.zeroRow + c * a.zeroCol] = Elem<T>::from_c(0);
    }
}

// All passes in one launch. The first `sortCtas` CTAs (one cluster) sort a tile each, the others zero the table.
template <class T>
__global__ void __launch_bounds__(kOrdThreads) k_order_cluster(const OrderArgs a) {
    grid_dependency_sync();
    __shared__ OrderShared s;
    if (blockIdx.x >= (unsigned) a.sortCtas) {
        if (a.zero) zero_rows<T>(a, (LL) (blockIdx.x - a.sortCtas) * kOrdThreads + threadIdx.x, (LL) (gridDim.x - a.sortCtas) * kOrdThreads);
        return;
    }
    cg::cluster_group cl = cg::this_cluster();
    const unsigned tile = blockIdx.x, ctas = (unsigned) a.sortCtas;
    for (int pass = 0; pass < a.passes; pass++) {
        unsigned key[kOrdKeys], pos[kOrdKeys], rank[kOrdKeys];
        order_read(a, pass, tile, key, pos);
        order_rank(a, pass, tile, key, rank, s);
        cl.sync();                                            // every CTA's totals stand
        unsigned before = 0, all = 0;
        if (threadIdx.x < kOrdBins) {
            for (unsigned q = 0; q < ctas; q++) {
                const unsigned c = cl.map_shared_rank(s.total, q)[threadIdx.x];
                if (q < tile) before += c;
                all += c;
            }
        }
        const unsigned start = order_scan(all, s.warpSums);
        if (threadIdx.x < kOrdBins) s.base[threadIdx.x] = start + before;
        __syncthreads();
        order_write(a, pass, tile, key, pos, rank, s);
        cl.sync();                                            // keys written, and nobody reads the totals any more
    }
}

__global__ void __launch_bounds__(kOrdThreads) k_order_count(const OrderArgs a, int pass) {
    grid_dependency_sync();
    __shared__ OrderShared s;
    for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        unsigned key[kOrdKeys], pos[kOrdKeys], rank[kOrdKeys];
        order_read(a, pass, tile, key, pos);
        order_rank(a, pass, tile, key, rank, s);
        if (threadIdx.x < kOrdBins) a.hist[(LL) tile * kOrdBins + threadIdx.x] = s.total[threadIdx.x];
        __syncthreads();
    }
}

// hist[tile][d] becomes where the tile's keys of digit d begin.
__global__ void __launch_bounds__(kOrdThreads) k_order_starts(const OrderArgs a) {
    grid_dependency_sync();
    __shared__ unsigned warpSums[kOrdWarps];
    unsigned run = 0;
    const bool live = threadIdx.x < kOrdBins;
    if (live) for (unsigned t = 0; t < a.tiles; t++) run += a.hist[(LL) t * kOrdBins + threadIdx.x];
    unsigned at = order_scan(live ? run : 0, warpSums);
    if (live) {
        for (unsigned t = 0; t < a.tiles; t++) {
            unsigned &h = a.hist[(LL) t * kOrdBins + threadIdx.x];
            const unsigned c = h;
            h = at;
            at += c;
        }
    }
}

__global__ void __launch_bounds__(kOrdThreads) k_order_scatter(const OrderArgs a, int pass) {
    grid_dependency_sync();
    __shared__ OrderShared s;
    for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        unsigned key[kOrdKeys], pos[kOrdKeys], rank[kOrdKeys];
        order_read(a, pass, tile, key, pos);
        order_rank(a, pass, tile, key, rank, s);
        if (threadIdx.x < kOrdBins) s.base[threadIdx.x] = a.hist[(LL) tile * kOrdBins + threadIdx.x];
        __syncthreads();
        order_write(a, pass, tile, key, pos, rank, s);
        __syncthreads();
    }
}

template <class T> __global__ void __launch_bounds__(kOrdThreads) k_zero_rows(const OrderArgs a) {
    grid_dependency_sync();
    zero_rows<T>(a, (LL) blockIdx.x * kOrdThreads + threadIdx.x, (LL) gridDim.x * kOrdThreads);
}

// ---- lookup ------------------------------------------------------------------------------------------------------
constexpr int kEmbThreads = 256;
constexpr int kEmbRows = 4;                  // rows a group of threads has in flight

struct EmbArgs {
    const void *src;                         // lookup: the table; gradient: dz
    void *dst;                               // lookup: z; gradient: grad
    const LL *tokens;
    LL n, vocab, cols;
    LL srcRow, srcCol, dstRow, dstCol;
    double scale;
    int words;                               // runs of V values per row
    int group;                               // threads per row (a power of two from 8 to 256)
    // gradient
    const unsigned *key, *pos;
    unsigned chunk;                          // sorted entries per group of threads
    unsigned chunks;
    void *partials;                          // [chunk][2][cols] wide values: head, tail
    int accumulate;
};

template <class T, int V> struct EmbRun {
    T v[V];
    ND_D void load(const T *p) {
        if constexpr (V == 1) v[0] = *p;
        else *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
    }
    ND_D void store(T *p) const {
        if constexpr (V == 1) *p = v[0];
        else *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(v);
    }
};
template <class T, int V> struct alignas(V == 1 ? sizeof(T) : 16) EmbWord : EmbRun<T, V> {};

template <class T, int V>
__global__ void __launch_bounds__(kEmbThreads) k_embedding(const EmbArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    const int groups = kEmbThreads / a.group, g = threadIdx.x / a.group, t = threadIdx.x - g * a.group;
    const T *table = static_cast<const T *>(a.src);
    T *z = static_cast<T *>(a.dst);
    const C scale = (C) a.scale;
    for (LL i0 = ((LL) blockIdx.x * groups + g) * kEmbRows; i0 < a.n; i0 += (LL) gridDim.x * groups * kEmbRows) {
        LL token[kEmbRows];
#pragma unroll
        for (int r = 0; r < kEmbRows; r++) token[r] = i0 + r < a.n ? a.tokens[i0 + r] : -1;
        for (int w = t; w < a.words; w += a.group) {
            EmbWord<T, V> v[kEmbRows];
#pragma unroll
            for (int r = 0; r < kEmbRows; r++)
                if (token[r] >= 0 && token[r] < a.vocab) v[r].load(table + token[r] * a.srcRow + (LL) w * V * a.srcCol);
#pragma unroll
            for (int r = 0; r < kEmbRows; r++) {
                if (i0 + r >= a.n) break;
#pragma unroll
                for (int k = 0; k < V; k++) {
                    if (token[r] < 0) v[r].v[k] = Elem<T>::from_c(C(0));
                    else if (token[r] >= a.vocab) v[r].v[k] = Elem<T>::from_c((C) NAN);
                    else v[r].v[k] = Elem<T>::from_c(Elem<T>::to_c(v[r].v[k]) * scale);
                }
                v[r].store(z + (i0 + r) * a.dstRow + (LL) w * V * a.dstCol);
            }
        }
    }
}

// ---- gradient ----------------------------------------------------------------------------------------------------
template <class T, int V, class C> ND_D void emb_finish(const EmbArgs &a, unsigned row, int w, const C (&sum)[V]) {
    T *g = static_cast<T *>(a.dst) + (LL) row * a.dstRow + (LL) w * V * a.dstCol;
    EmbWord<T, V> o;
    if (a.accumulate) o.load(g);
#pragma unroll
    for (int k = 0; k < V; k++) {
        const C v = sum[k] * (C) a.scale;
        o.v[k] = Elem<T>::from_c(a.accumulate ? Elem<T>::to_c(o.v[k]) + v : v);
    }
    o.store(g);
}
template <int V, class C> ND_D void emb_partial(const EmbArgs &a, unsigned chunk, int which, int w, const C (&sum)[V]) {
    C *p = static_cast<C *>(a.partials) + ((LL) chunk * 2 + which) * a.cols + (LL) w * V;
#pragma unroll
    for (int k = 0; k < V; k++) p[k] = sum[k];
}

// A group of threads walks a chunk of the sorted list, each thread one run of V columns. Four rows are in flight.
template <class T, int V>
__global__ void __launch_bounds__(kEmbThreads) k_embedding_sums(const EmbArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    const int groups = kEmbThreads / a.group, g = threadIdx.x / a.group, t = threadIdx.x - g * a.group;
    const unsigned chunk = blockIdx.x * groups + g;
    const T *dz = static_cast<const T *>(a.src);
    if (chunk >= a.chunks) return;
    const unsigned n = (unsigned) a.n, vocab = (unsigned) a.vocab;
    const unsigned first = chunk * a.chunk, last = n - first < a.chunk ? n : first + a.chunk;
    const unsigned before = first > 0 ? a.key[first - 1] : 0xffffffffu;      // no key: vocab is below 2^31
    for (int w = t + (int) blockIdx.y * a.group; w < a.words; w += a.group * (int) gridDim.y) {
        C sum[V];
#pragma unroll
        for (int k = 0; k < V; k++) sum[k] = C(0);
        unsigned key = a.key[first];
        bool head = key == before;                              // the run began in an earlier chunk
        for (unsigned i = first; i < last && key < vocab; i += 4) {
            EmbWord<T, V> v[4];
            unsigned next[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (i + q < last) {
                    if (a.key[i + q] < vocab) v[q].load(dz + (LL) a.pos[i + q] * a.srcRow + (LL) w * V * a.srcCol);
                    next[q] = i + q + 1 < n ? a.key[i + q + 1] : vocab;
                }
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (i + q >= last || key >= vocab) break;
#pragma unroll
                for (int k = 0; k < V; k++) sum[k] += Elem<T>::to_c(v[q].v[k]);
                if (next[q] != key || i + q + 1 == last) {
                    // the run ends here, or the chunk does
                    if (head) emb_partial<V>(a, chunk, 0, w, sum);
                    else if (next[q] != key) emb_finish<T, V>(a, key, w, sum);
                    else emb_partial<V>(a, chunk, 1, w, sum);
                    head = false;
                    key = next[q];
#pragma unroll
                    for (int k = 0; k < V; k++) sum[k] = C(0);
                }
            }
        }
    }
}

// Runs that cross chunks: the CTA of the chunk that such a run begins in adds up the tail there and the heads of the
// chunks it reaches, eight at a time, the eight sums in order.
template <class T>
__global__ void __launch_bounds__(256) k_embedding_join(const EmbArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    __shared__ C part[8][32];
    const unsigned chunk = blockIdx.x, n = (unsigned) a.n;
    const unsigned end = (chunk + 1) * a.chunk;                 // there is a next chunk: the grid leaves out the last one
    const unsigned key = a.key[end - 1];
    if (key >= (unsigned) a.vocab || a.key[end] != key) return;                                 // no run crosses
    const unsigned first = chunk * a.chunk;
    if (first > 0 && a.key[first] == key && a.key[first - 1] == key) return;                    // began earlier
    // the chunks the run reaches: up to the one that holds its last entry, found by bisection
    unsigned lo = end, hi = n - 1;
    while (lo < hi) {
        const unsigned mid = lo + (hi - lo + 1) / 2;
        if (a.key[mid] == key) lo = mid; else hi = mid - 1;
    }
    const unsigned reach = lo / a.chunk;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const C *p = static_cast<const C *>(a.partials);
    for (LL c0 = (LL) blockIdx.y * 32; c0 < a.cols; c0 += (LL) gridDim.y * 32) {
        const LL c = c0 + lane;
        C s = C(0);
        if (c < a.cols) {
            if (warp == 0) s = p[((LL) chunk * 2 + 1) * a.cols + c];
            for (unsigned q = chunk + 1 + warp; q <= reach; q += 8) s += p[(LL) q * 2 * a.cols + c];
        }
        __syncthreads();
        part[warp][lane] = s;
        __syncthreads();
        if (warp == 0 && c < a.cols) {
            for (int q = 1; q < 8; q++) s += part[q][lane];
            T *g = static_cast<T *>(a.dst) + (LL) key * a.dstRow + c * a.dstCol;
            s *= (C) a.scale;
            Elem<T>::store(g, a.accumulate ? Elem<T>::load(g) + s : s);
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------
int group_for(LL words) {
    int g = 8;
    while (g < kEmbThreads && g < words) g *= 2;
    return g;
}

template <class T> Status emb_lookup(EmbArgs &a, bool words, cudaStream_t st) {
    constexpr int V = Elem<T>::kVec;
    a.words = (int) (words ? a.cols / V : a.cols);
    a.group = group_for(a.words);
    const LL blocks = ceil_div(a.n, (LL) kEmbThreads / a.group * kEmbRows);
    const dim3 grid((unsigned) (blocks < 0x7fffffffLL ? blocks : 0x7fffffffLL));
    if (words) launch_kernel(k_embedding<T, V>, grid, dim3(kEmbThreads), st, a);
    else launch_kernel(k_embedding<T, 1>, grid, dim3(kEmbThreads), st, a);
    ND_CUDA(cudaGetLastError());
    return kOk;
}

template <class T> Status launch_order_cluster(const OrderArgs &o, unsigned grid, unsigned cluster, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(kOrdThreads); cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_tuning[kTuneOverlapLaunch] ? 2 : 1;
    cudaLaunchKernelEx(&cfg, k_order_cluster<T>, o);
    count_launch();
    return kOk;
}

// Sorts the tokens (and zeroes the table when `o.zero` is set); *result says which pair of lists holds the outcome.
template <class T> Status order_tokens(OrderArgs &o, int *result, cudaStream_t st) {
    int width = 1;
    while (width < 32 && (o.vocab >> width) != 0) width++;               // keys go up to vocab itself
    o.passes = (int) ceil_div(width, kOrdBits);
    o.bits = (int) ceil_div(width, o.passes);
    o.tiles = (unsigned) ceil_div(o.n, kOrdTile);
    *result = (o.passes - 1) & 1;
    const unsigned zeroCtas = o.zero ? (unsigned) kNumSMs : 0u;
    if (o.tiles <= (unsigned) kOrdCluster) {
        unsigned cluster = 1;
        while (cluster < o.tiles) cluster *= 2;
        o.sortCtas = (int) cluster;
        return launch_order_cluster<T>(o, cluster + zeroCtas / cluster * cluster, cluster, st);
    }
    if (o.zero) launch_kernel(k_zero_rows<T>, dim3(zeroCtas * 2), dim3(kOrdThreads), st, o);
    const unsigned grid = o.tiles < (unsigned) kNumSMs * 2 ? o.tiles : (unsigned) kNumSMs * 2;
    for (int pass = 0; pass < o.passes; pass++) {
        launch_kernel(k_order_count, dim3(grid), dim3(kOrdThreads), st, o, pass);
        launch_kernel(k_order_starts, dim3(1), dim3(kOrdThreads), st, o);
        launch_kernel(k_order_scatter, dim3(grid), dim3(kOrdThreads), st, o, pass);
    }
    return kOk;
}

template <class T> Status emb_gradient(EmbArgs &a, OrderArgs &o, bool words, cudaStream_t st) {
    typedef typename Elem<T>::C C;
    constexpr int V = Elem<T>::kVec;
    if (a.n == 0) {
        if (o.zero) launch_kernel(k_zero_rows<T>, dim3((unsigned) kNumSMs * 2), dim3(kOrdThreads), st, o);
        ND_CUDA(cudaGetLastError());
        return kOk;
    }
    a.words = (int) (words ? a.cols / V : a.cols);
    a.group = group_for(a.words);
    const LL slices = ceil_div(a.words, a.group);
    // Longer chunks mean fewer partial sums, shorter ones more CTAs: the longest of 8 .. 64 that still gives every SM
    // eight CTAs, as far as there are that many rows.
    LL chunk = 64;
    while (chunk > 8 && ceil_div(a.n, chunk) * slices * a.group / kEmbThreads < (LL) kNumSMs * 8) chunk /= 2;
    a.chunk = (unsigned) chunk;
    a.chunks = (unsigned) ceil_div(a.n, chunk);
    const size_t list = round_up((size_t) a.n * sizeof(unsigned), 256);
    const size_t hist = round_up((size_t) ceil_div(a.n, kOrdTile) * kOrdBins * sizeof(unsigned), 256);
    Scratch scratch(st);
    ND_TRY(scratch.alloc(4 * list + hist + (size_t) a.chunks * 2 * (size_t) a.cols * sizeof(C)));
    for (int k = 0; k < 2; k++) { o.key[k] = scratch.at<unsigned>(2 * k * list); o.pos[k] = scratch.at<unsigned>((2 * k + 1) * list); }
    o.hist = scratch.at<unsigned>(4 * list);
    a.partials = scratch.at<void>(4 * list + hist);
    int result = 0;
    ND_TRY(order_tokens<T>(o, &result, st));
    a.key = o.key[result]; a.pos = o.pos[result];
    const dim3 grid((unsigned) ceil_div(a.chunks, kEmbThreads / a.group), (unsigned) (slices < 65535 ? slices : 65535));
    if (words) launch_kernel(k_embedding_sums<T, V>, grid, dim3(kEmbThreads), st, a);
    else launch_kernel(k_embedding_sums<T, 1>, grid, dim3(kEmbThreads), st, a);
    if (a.chunks > 1) {
        const LL slabs = ceil_div(a.cols, 32);
        launch_kernel(k_embedding_join<T>, dim3(a.chunks - 1, (unsigned) (slabs < 64 ? slabs : 64)), dim3(256), st, a);
    }
    ND_CUDA(cudaGetLastError());
    return kOk;
}

// Shape checks that lookup and gradient share: `table` is [vocab, cols], `rows` is [n, cols].
Status emb_shapes(const char *what, const ShapeDesc &table, const ShapeDesc &rows) {
    if (table.rank != 2 || rows.rank != 2) return bad_arg(std::string(what) + ": the table and the rows must be of rank 2");
    if (table.shape[1] != rows.shape[1]) return bad_arg(std::string(what) + ": the table and the rows differ in width");
    if (table.shape[0] >= 0x7fffffffLL || table.shape[1] >= 0x7fffffffLL || rows.shape[0] > 1LL << 30) {
        set_error(std::string(what) + ": at most 2^31 - 2 table rows, columns and 2^30 tokens are served");
        return kTooLarge;
    }
    return kOk;
}
bool emb_words(const ShapeDesc &d, const void *p, LL V) {
    return d.shape[1] % V == 0 && d.stride[1] == 1 && (d.shape[0] < 2 || d.stride[0] % V == 0) && aligned16(p);
}
Status emb_scale(int dtype, double scale) {
    if (!std::isfinite(dtype == kF64 ? scale : (double) (float) scale)) return bad_arg("embedding: scale must be finite");
    return kOk;
}

Status emb_lookup_entry(void *stream, int dtype, const void *table, const Nd4jLong *tableShapeInfo, const Nd4jLong *tokens,
                        double scale, void *z, const Nd4jLong *zShapeInfo) {
    ND_TRY(require_dtype(dtype));
    ND_TRY(emb_scale(dtype, scale));
    ShapeDesc td, zd;
    ND_TRY(parse_shape(tableShapeInfo, "tableShapeInfo", &td));
    ND_TRY(parse_shape(zShapeInfo, "zShapeInfo", &zd));
    ND_TRY(emb_shapes("embedding", td, zd));
    if (zd.length == 0) return kOk;
    ND_TRY(require(tokens, "tokens")); ND_TRY(require(z, "z"));
    if (td.length > 0) ND_TRY(require(table, "table"));
    const size_t elem = size_of_dtype(dtype);
    ND_TRY(require_aligned(table, elem, "table")); ND_TRY(require_aligned(z, elem, "z")); ND_TRY(require_aligned(tokens, 8, "tokens"));
    ND_TRY(check_written(zd, "z"));
    const Span sz = span_of(z, zd, elem);
    ND_TRY(check_apart(sz, "z", span_of(table, td, elem), "table"));
    ND_TRY(check_apart(sz, "z", span_of(tokens, zd.shape[0], 8), "tokens"));
    EmbArgs a = {};
    a.src = table; a.dst = z; a.tokens = tokens; a.n = zd.shape[0]; a.vocab = td.shape[0]; a.cols = zd.shape[1];
    a.srcRow = td.stride[0]; a.srcCol = td.stride[1]; a.dstRow = zd.stride[0]; a.dstCol = zd.stride[1];
    a.scale = scale;
    const LL V = 16 / (LL) elem;
    const bool words = emb_words(td, table, V) && emb_words(zd, z, V);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kF32: return emb_lookup<float>(a, words, st);
        case kF64: return emb_lookup<double>(a, words, st);
        default: return emb_lookup<__half>(a, words, st);
    }
}

Status emb_gradient_entry(void *stream, int dtype, const Nd4jLong *tokens, double scale, const void *dz,
                          const Nd4jLong *dzShapeInfo, void *grad, const Nd4jLong *gradShapeInfo, int accumulate) {
    ND_TRY(require_dtype(dtype));
    ND_TRY(emb_scale(dtype, scale));
    ShapeDesc gd, dd;
    ND_TRY(parse_shape(gradShapeInfo, "gradShapeInfo", &gd));
    ND_TRY(parse_shape(dzShapeInfo, "dzShapeInfo", &dd));
    ND_TRY(emb_shapes("embedding gradient", gd, dd));
    if (gd.length == 0) return kOk;
    ND_TRY(require(grad, "grad"));
    const size_t elem = size_of_dtype(dtype);
    ND_TRY(require_aligned(grad, elem, "grad"));
    ND_TRY(check_written(gd, "grad"));
    if (dd.length > 0) {
        ND_TRY(require(tokens, "tokens")); ND_TRY(require(dz, "dz"));
        ND_TRY(require_aligned(dz, elem, "dz")); ND_TRY(require_aligned(tokens, 8, "tokens"));
        const Span sg = span_of(grad, gd, elem);
        ND_TRY(check_apart(sg, "grad", span_of(dz, dd, elem), "dz"));
        ND_TRY(check_apart(sg, "grad", span_of(tokens, dd.shape[0], 8), "tokens"));
    }
    EmbArgs a = {};
    a.src = dz; a.dst = grad; a.tokens = tokens; a.n = dd.shape[0]; a.vocab = gd.shape[0]; a.cols = gd.shape[1];
    a.srcRow = dd.stride[0]; a.srcCol = dd.stride[1]; a.dstRow = gd.stride[0]; a.dstCol = gd.stride[1];
    a.scale = scale; a.accumulate = accumulate != 0;
    const LL V = 16 / (LL) elem;
    const bool gradWords = emb_words(gd, grad, V);
    const bool words = gradWords && emb_words(dd, dz, V);
    OrderArgs o = {};
    o.tokens = tokens; o.n = (unsigned) a.n; o.vocab = (unsigned) a.vocab;
    o.zero = accumulate ? nullptr : grad;
    o.zeroRows = gd.shape[0]; o.zeroRow = gd.stride[0]; o.zeroCol = gd.stride[1]; o.cols = gd.shape[1];
    o.zeroWords = gradWords ? (int) (a.cols / V) : 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kF32: return emb_gradient<float>(a, o, words, st);
        case kF64: return emb_gradient<double>(a, o, words, st);
        default: return emb_gradient<__half>(a, o, words, st);
    }
}

}  // namespace
}  // namespace nd4jb200

using namespace nd4jb200;

#pragma GCC visibility push(default)
extern "C" {

int nd4jb200_exec_embedding(void *stream, int dtype, const void *table, const Nd4jLong *tableShapeInfo, const Nd4jLong *tokens,
                            double scale, void *z, const Nd4jLong *zShapeInfo) {
    return c_entry([&] { return emb_lookup_entry(stream, dtype, table, tableShapeInfo, tokens, scale, z, zShapeInfo); });
}

int nd4jb200_exec_embedding_grad(void *stream, int dtype, const Nd4jLong *tokens, double scale, const void *dz,
                                 const Nd4jLong *dzShapeInfo, void *grad, const Nd4jLong *gradShapeInfo, int accumulate) {
    return c_entry([&] { return emb_gradient_entry(stream, dtype, tokens, scale, dz, dzShapeInfo, grad, gradShapeInfo, accumulate); });
}

}  // extern "C"
#pragma GCC visibility pop
