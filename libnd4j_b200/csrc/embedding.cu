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
// end leaves partial sums, one for each chunk, which a last launch adds up: every eighth of them, then the eight sums.
// That order follows from the sizes, the layouts and the tokens alone, so the result is the same bits on every run. Sums
// are held in float (double for double data) and rounded once, after scaling and, where asked for, adding what grad holds.
//
// The sort is a least-significant-digit radix sort with digits of up to 9 bits: two passes up to a table of 2^18 rows.
// Up to 65536 tokens one cluster of CTAs does all passes in one launch, the counts and the keys travelling through
// distributed shared memory; the other CTAs of that launch write the zeros of the table meanwhile. Longer lists take
// three launches per pass.
//
// Measured: lookup of 32768 rows of 2048 halves, 41 us = 6.6 TB/s; gradient of 16384 rows of 1024 floats over a table of
// 50000 rows: 35 us for the zeros (5.8 TB/s) with the sort (13 us alone) beside them, 17 us for the sums, 9 for the joins.
#include "../../include/nd4j_b200.h"
#include <cooperative_groups.h>
#include "device_utils.cuh"
#include "entry_checks.h"

namespace cg = cooperative_groups;

namespace nd4jb200 {
namespace {

// ---- the order of the tokens -------------------------------------------------------------------------------------
constexpr int kOrdThreads = 512;
constexpr int kOrdWarps = kOrdThreads / 32;
constexpr int kOrdMaxKeys = 16;                               // per thread
constexpr int kOrdBits = 9;
constexpr int kOrdBins = 1 << kOrdBits;                       // one per thread
constexpr int kOrdCluster = 8;
static_assert(kOrdBins == kOrdThreads, "thread d looks after digit d");

struct OrderArgs {
    const LL *tokens;
    unsigned *key[2], *pos[2];       // ping-pong lists; one launch: the sorted list goes to the first
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
    unsigned base[kOrdBins];                     // where the tile's first key of the digit goes
    unsigned warpSums[kOrdWarps];
};

ND_D unsigned order_key(const OrderArgs &a, LL token) { return token >= 0 && token < (LL) a.vocab ? (unsigned) token : a.vocab; }

// Warp w holds keys [w * 32 * KPT, ...) of the tile, round r of it the next 32: "earlier" is (warp, round, lane).
template <int KPT> ND_D unsigned order_local(int r) { return (threadIdx.x >> 5) * (32 * KPT) + r * 32 + (threadIdx.x & 31); }

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
    unsigned before = 0;
#pragma unroll
    for (int w = 0; w < kOrdWarps; w++) before += w < warp ? warpSums[w] : 0u;
    __syncthreads();
    return before + inc - v;
}

// Rank of every key among the warp's earlier keys of its digit, and the tile's counts; `live` of the tile's keys exist.
// The lanes that share a digit are found with one ballot per bit of it (match.any takes a step per distinct value: a
// tile of 4096 keys took 14 us per pass with it). Afterwards count[w][d] is the number of the tile's keys of digit d in
// the warps before w, total[d] that of the tile.
template <int KPT>
ND_D void order_rank(const unsigned (&key)[KPT], unsigned (&rank)[KPT], int shift, int bits, unsigned live, OrderShared &s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint4 *words = reinterpret_cast<uint4 *>(&s.count[0][0]);
#pragma unroll
    for (int i = 0; i < kOrdWarps * kOrdBins / 8 / kOrdThreads; i++) words[i * kOrdThreads + threadIdx.x] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const unsigned below = (1u << lane) - 1u, mask = (1u << bits) - 1u;
#pragma unroll
    for (int r = 0; r < KPT; r++) {
        const bool valid = order_local<KPT>(r) < live;
        const unsigned d = (key[r] >> shift) & mask;
        unsigned peers = __ballot_sync(0xffffffffu, valid);
#pragma unroll
        for (int b = 0; b < kOrdBits; b++) {                  // bits beyond `bits` are 0 in every lane
            const bool bit = (d >> b) & 1u;
            const unsigned has = __ballot_sync(0xffffffffu, bit);
            peers &= bit ? has : ~has;
        }
        const unsigned earlier = __popc(peers & below);
        const unsigned before = s.count[warp][d];
        __syncwarp();
        if (valid && earlier == 0) s.count[warp][d] = (unsigned short) (before + __popc(peers));
        __syncwarp();
        rank[r] = before + earlier;
    }
    __syncthreads();
    unsigned c[kOrdWarps], run = 0;
#pragma unroll
    for (int w = 0; w < kOrdWarps; w++) c[w] = s.count[w][threadIdx.x];
#pragma unroll
    for (int w = 0; w < kOrdWarps; w++) { s.count[w][threadIdx.x] = (unsigned short) run; run += c[w]; }
    s.total[threadIdx.x] = run;
    __syncthreads();
}

// Zeroes the table's rows; `first` and `step` deal the work to the threads (at least 16 of them).
template <class T> ND_D void zero_rows(const OrderArgs &a, LL first, LL step) {
    T *z = static_cast<T *>(a.zero);
    if (a.zeroCol == 1 && a.zeroRow == a.cols) {                // one run: whole words but for its two ends
        const LL n = a.zeroRows * a.cols;
        LL head = (LL) (((16 - (reinterpret_cast<unsigned long long>(z) & 15)) & 15) / sizeof(T));
        if (head > n) head = n;
        const LL words = (n - head) / Elem<T>::kVec, tail = n - head - words * Elem<T>::kVec;
        uint4 *p = reinterpret_cast<uint4 *>(z + head);
        if (first < head) z[first] = Elem<T>::from_c(0);
        if (first < tail) z[n - tail + first] = Elem<T>::from_c(0);
        LL i = first;
        for (; i + 3 * step < words; i += 4 * step) {
#pragma unroll
            for (int j = 0; j < 4; j++) __stcs(p + i + j * step, make_uint4(0, 0, 0, 0));
        }
        for (; i < words; i += step) __stcs(p + i, make_uint4(0, 0, 0, 0));
        return;
    }
    const LL perRow = a.zeroWords > 0 ? a.zeroWords : a.cols;
    for (LL i = first; i < a.zeroRows * perRow; i += step) {
        const LL row = i / perRow, c = i - row * perRow;
        if (a.zeroWords > 0) *reinterpret_cast<uint4 *>(z + row * a.zeroRow + c * Elem<T>::kVec) = make_uint4(0, 0, 0, 0);
        else z[row * a.zeroRow + c * a.zeroCol] = Elem<T>::from_c(0);
    }
}

// All passes in one launch. The first `sortCtas` CTAs (one cluster) sort a tile of kOrdThreads * KPT keys each, the
// others zero the table. Between the passes keys and positions go straight into the shared memory of the CTA whose tile
// they belong to next: every CTA has its keys in registers when the totals have been exchanged, so one buffer serves.
template <class T, int KPT>
__global__ void __launch_bounds__(kOrdThreads) k_order_cluster(const OrderArgs a) {
    grid_dependency_sync();
    extern __shared__ unsigned ord_smem[];                    // keys, then positions, of the tile
    __shared__ __align__(16) OrderShared s;
    constexpr unsigned TILE = kOrdThreads * KPT;
    if (blockIdx.x >= (unsigned) a.sortCtas) {
        if (a.zero) zero_rows<T>(a, (LL) (blockIdx.x - a.sortCtas) * kOrdThreads + threadIdx.x, (LL) (gridDim.x - a.sortCtas) * kOrdThreads);
        return;
    }
    cg::cluster_group cl = cg::this_cluster();
    const unsigned tile = blockIdx.x, ctas = (unsigned) a.sortCtas;
    const unsigned live = a.n > tile * TILE ? a.n - tile * TILE : 0u;      // of this tile's keys: all are in front
    unsigned key[KPT], pos[KPT], rank[KPT];
#pragma unroll
    for (int r = 0; r < KPT; r++) {
        const unsigned i = tile * TILE + order_local<KPT>(r);
        key[r] = i < a.n ? order_key(a, a.tokens[i]) : 0u;
        pos[r] = i;
    }
    for (int pass = 0; pass < a.passes; pass++) {
        const int shift = pass * a.bits;
        order_rank<KPT>(key, rank, shift, a.bits, live, s);
        cl.sync();                                            // every CTA's totals stand, every CTA has read its keys
        unsigned before = 0, all = 0;
#pragma unroll 8
        for (unsigned q = 0; q < ctas; q++) {
            const unsigned c = cl.map_shared_rank(s.total, q)[threadIdx.x];
            before += q < tile ? c : 0u;
            all += c;
        }
        s.base[threadIdx.x] = order_scan(all, s.warpSums) + before;
        __syncthreads();
        const bool last = pass + 1 == a.passes;
#pragma unroll
        for (int r = 0; r < KPT; r++) {
            if (order_local<KPT>(r) < live) {
                const unsigned d = (key[r] >> shift) & ((1u << a.bits) - 1u);
                const unsigned to = s.base[d] + s.count[threadIdx.x >> 5][d] + rank[r];
                if (last) { a.key[0][to] = key[r]; a.pos[0][to] = pos[r]; }
                else {
                    unsigned *there = cl.map_shared_rank(ord_smem, to / TILE);
                    there[to % TILE] = key[r];
                    there[TILE + to % TILE] = pos[r];
                }
            }
        }
        cl.sync();                                            // keys stand, and nobody reads the totals any more
        if (!last) {
#pragma unroll
            for (int r = 0; r < KPT; r++) { key[r] = ord_smem[order_local<KPT>(r)]; pos[r] = ord_smem[TILE + order_local<KPT>(r)]; }
        }
    }
}

template <int KPT> ND_D void order_read(const OrderArgs &a, int pass, unsigned tile, unsigned (&key)[KPT], unsigned (&pos)[KPT]) {
    const unsigned *fromKey = a.key[(pass - 1) & 1], *fromPos = a.pos[(pass - 1) & 1];
#pragma unroll
    for (int r = 0; r < KPT; r++) {
        const unsigned i = tile * (kOrdThreads * KPT) + order_local<KPT>(r);
        key[r] = pos[r] = 0;
        if (i < a.n) {
            key[r] = pass == 0 ? order_key(a, a.tokens[i]) : fromKey[i];
            pos[r] = pass == 0 ? i : fromPos[i];
        }
    }
}

__global__ void __launch_bounds__(kOrdThreads) k_order_count(const OrderArgs a, int pass) {
    grid_dependency_sync();
    __shared__ __align__(16) OrderShared s;
    constexpr unsigned TILE = kOrdThreads * kOrdMaxKeys;
    for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        unsigned key[kOrdMaxKeys], pos[kOrdMaxKeys], rank[kOrdMaxKeys];
        order_read<kOrdMaxKeys>(a, pass, tile, key, pos);
        order_rank<kOrdMaxKeys>(key, rank, pass * a.bits, a.bits, a.n - tile * TILE, s);
        a.hist[(LL) tile * kOrdBins + threadIdx.x] = s.total[threadIdx.x];
        __syncthreads();
    }
}

// hist[tile][d] becomes where the tile's keys of digit d begin.
__global__ void __launch_bounds__(kOrdThreads) k_order_starts(const OrderArgs a) {
    grid_dependency_sync();
    __shared__ unsigned warpSums[kOrdWarps];
    unsigned run = 0;
#pragma unroll 8
    for (unsigned t = 0; t < a.tiles; t++) run += a.hist[(LL) t * kOrdBins + threadIdx.x];
    unsigned at = order_scan(run, warpSums);
    unsigned t = 0;
    for (; t + 8 <= a.tiles; t += 8) {
        unsigned c[8];
#pragma unroll
        for (int k = 0; k < 8; k++) c[k] = a.hist[(LL) (t + k) * kOrdBins + threadIdx.x];
#pragma unroll
        for (int k = 0; k < 8; k++) { a.hist[(LL) (t + k) * kOrdBins + threadIdx.x] = at; at += c[k]; }
    }
    for (; t < a.tiles; t++) {
        const unsigned c = a.hist[(LL) t * kOrdBins + threadIdx.x];
        a.hist[(LL) t * kOrdBins + threadIdx.x] = at;
        at += c;
    }
}

__global__ void __launch_bounds__(kOrdThreads) k_order_scatter(const OrderArgs a, int pass) {
    grid_dependency_sync();
    __shared__ __align__(16) OrderShared s;
    constexpr unsigned TILE = kOrdThreads * kOrdMaxKeys;
    unsigned *toKey = a.key[pass & 1], *toPos = a.pos[pass & 1];
    for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        unsigned key[kOrdMaxKeys], pos[kOrdMaxKeys], rank[kOrdMaxKeys];
        const unsigned live = a.n - tile * TILE;
        order_read<kOrdMaxKeys>(a, pass, tile, key, pos);
        order_rank<kOrdMaxKeys>(key, rank, pass * a.bits, a.bits, live, s);
        s.base[threadIdx.x] = a.hist[(LL) tile * kOrdBins + threadIdx.x];
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kOrdMaxKeys; r++) {
            if (order_local<kOrdMaxKeys>(r) < live) {
                const unsigned d = (key[r] >> (pass * a.bits)) & ((1u << a.bits) - 1u);
                const unsigned to = s.base[d] + s.count[threadIdx.x >> 5][d] + rank[r];
                toKey[to] = key[r];
                toPos[to] = pos[r];
            }
        }
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
    unsigned words;                          // runs of V values per row: below 2^31, so that a loop's last step still fits
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
__global__ void __launch_bounds__(kEmbThreads, 6) k_embedding(const EmbArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    const int groups = kEmbThreads / a.group, g = threadIdx.x / a.group, t = threadIdx.x - g * a.group;
    const T *table = static_cast<const T *>(a.src);
    T *z = static_cast<T *>(a.dst);
    const C scale = (C) a.scale;
    for (LL i0 = ((LL) blockIdx.x * groups + g) * kEmbRows; i0 < a.n; i0 += (LL) gridDim.x * groups * kEmbRows) {
        int row[kEmbRows];
        bool in[kEmbRows];
        C other[kEmbRows];
#pragma unroll
        for (int r = 0; r < kEmbRows; r++) {
            const LL token = i0 + r < a.n ? a.tokens[i0 + r] : -1;
            in[r] = token >= 0 && token < a.vocab;
            row[r] = in[r] ? (int) token : 0;
            other[r] = token < 0 ? C(0) : (C) NAN;
        }
        for (unsigned w = t; w < a.words; w += a.group) {
            EmbWord<T, V> v[kEmbRows];
#pragma unroll
            for (int r = 0; r < kEmbRows; r++)
                if (in[r]) v[r].load(table + row[r] * a.srcRow + (LL) w * V * a.srcCol);
#pragma unroll
            for (int r = 0; r < kEmbRows; r++) {
                if (i0 + r >= a.n) break;
#pragma unroll
                for (int k = 0; k < V; k++) v[r].v[k] = Elem<T>::from_c(in[r] ? Elem<T>::to_c(v[r].v[k]) * scale : other[r]);
                v[r].store(z + (i0 + r) * a.dstRow + (LL) w * V * a.dstCol);
            }
        }
    }
}

// ---- gradient ----------------------------------------------------------------------------------------------------
template <class T, int V, class C> ND_D void emb_finish(const EmbArgs &a, unsigned row, unsigned w, const C (&sum)[V]) {
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
template <int V, class C> ND_D void emb_partial(const EmbArgs &a, unsigned chunk, int which, unsigned w, const C (&sum)[V]) {
    C *p = static_cast<C *>(a.partials) + ((LL) chunk * 2 + which) * a.cols + (LL) w * V;
#pragma unroll
    for (int k = 0; k < V; k++) p[k] = sum[k];
}

// A group of threads walks a chunk of the sorted list, each thread one run of V columns. The chunk's keys and positions
// are fetched first, so that the rows themselves can be read without waiting for one another, eight at a time.
constexpr int kEmbMaxChunk = 64;
template <class T, int V>
__global__ void __launch_bounds__(kEmbThreads, 4) k_embedding_sums(const EmbArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    constexpr int R = 8;
    extern __shared__ unsigned emb_smem[];                      // per group: keys of one entry before .. one behind, positions
    const int groups = kEmbThreads / a.group, g = threadIdx.x / a.group, t = threadIdx.x - g * a.group;
    const unsigned chunk = blockIdx.x * groups + g, n = (unsigned) a.n, vocab = (unsigned) a.vocab;
    unsigned *key = emb_smem + g * (2 * kEmbMaxChunk + 2) + 1, *pos = key + kEmbMaxChunk + 1;
    const unsigned first = chunk < a.chunks ? chunk * a.chunk : n;
    const int len = n - first < a.chunk ? (int) (n - first) : (int) a.chunk;
    for (int i = t - 1; i <= len; i += a.group) {
        const bool in = i < 0 ? first > 0 : first + i < n;
        key[i] = in ? a.key[first + i] : (i < 0 ? 0xffffffffu : vocab);        // no token has these
        if (i >= 0 && i < len) pos[i] = a.pos[first + i];
    }
    __syncthreads();
    const T *dz = static_cast<const T *>(a.src);
    for (unsigned w = t + blockIdx.y * a.group; w < a.words; w += a.group * gridDim.y) {
        C sum[V];
#pragma unroll
        for (int k = 0; k < V; k++) sum[k] = C(0);
        bool head = key[0] == key[-1];                          // the run began in an earlier chunk
        for (int i = 0; i < len && key[i] < vocab; i += R) {
            EmbWord<T, V> v[R];
#pragma unroll
            for (int q = 0; q < R; q++)
                if (i + q < len && key[i + q] < vocab) v[q].load(dz + (LL) pos[i + q] * a.srcRow + (LL) w * V * a.srcCol);
#pragma unroll
            for (int q = 0; q < R; q++) {
                if (i + q >= len || key[i + q] >= vocab) break;
#pragma unroll
                for (int k = 0; k < V; k++) sum[k] += Elem<T>::to_c(v[q].v[k]);
                const bool ends = key[i + q + 1] != key[i + q];
                if (ends || i + q + 1 == len) {
                    // the run ends here, or the chunk does
                    if (head) emb_partial<V>(a, chunk, 0, w, sum);
                    else if (ends) emb_finish<T, V>(a, key[i + q], w, sum);
                    else emb_partial<V>(a, chunk, 1, w, sum);
                    head = false;
#pragma unroll
                    for (int k = 0; k < V; k++) sum[k] = C(0);
                }
            }
        }
    }
}

// Runs that cross chunks: the CTA of the chunk that such a run begins in adds up the tail there and the heads of the
// chunks it reaches, warp w every eighth of them, then the warps' eight sums. Most chunks have no such run and their CTA ends at once.
template <class T>
__global__ void __launch_bounds__(256) k_embedding_join(const EmbArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    constexpr int W = 4;                                        // columns per lane
    __shared__ C part[8][32 * W];
    const unsigned chunk = blockIdx.x;
    const unsigned end = (chunk + 1) * a.chunk;                 // there is a next chunk: the grid leaves out the last one
    const unsigned first = chunk * a.chunk;
    const unsigned key = a.key[end - 1], after = a.key[end], start = a.key[first], before = first > 0 ? a.key[first - 1] : 0xffffffffu;
    if (key >= (unsigned) a.vocab || after != key) return;      // no run crosses
    if (start == key && before == key) return;                  // it began earlier
    // the chunks the run reaches are those that begin with its key: 256 of them are looked at in one step
    unsigned reach = chunk;
    for (;;) {
        const LL q = (LL) reach + 1 + threadIdx.x;
        const int more = __syncthreads_count(q < a.chunks && a.key[q * a.chunk] == key);
        reach += more;
        if (more < 256) break;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const C *p = static_cast<const C *>(a.partials);
    for (LL c0 = (LL) blockIdx.y * 32 * W; c0 < a.cols; c0 += (LL) gridDim.y * 32 * W) {
        C s[W];
#pragma unroll
        for (int k = 0; k < W; k++) s[k] = C(0);
        if (warp == 0) {
#pragma unroll
            for (int k = 0; k < W; k++) if (c0 + k * 32 + lane < a.cols) s[k] = p[((LL) chunk * 2 + 1) * a.cols + c0 + k * 32 + lane];
        }
        for (unsigned q = chunk + 1 + warp; q <= reach; q += 32) {          // four of the warp's chunks in flight
            C v[4][W];
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int k = 0; k < W; k++)
                    v[u][k] = q + 8 * u <= reach && c0 + k * 32 + lane < a.cols ? p[(LL) (q + 8 * u) * 2 * a.cols + c0 + k * 32 + lane] : C(0);
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int k = 0; k < W; k++) s[k] += v[u][k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < W; k++) part[warp][k * 32 + lane] = s[k];
        __syncthreads();
        const LL c = c0 + threadIdx.x;
        if (threadIdx.x < 32 * W && c < a.cols) {
            C sum = part[0][threadIdx.x];
#pragma unroll
            for (int q = 1; q < 8; q++) sum += part[q][threadIdx.x];
            T *g = static_cast<T *>(a.dst) + (LL) key * a.dstRow + c * a.dstCol;
            sum *= (C) a.scale;
            Elem<T>::store(g, a.accumulate ? Elem<T>::load(g) + sum : sum);
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
    a.words = (unsigned) (words ? a.cols / V : a.cols);
    a.group = group_for(a.words);
    const LL blocks = ceil_div(a.n, (LL) kEmbThreads / a.group * kEmbRows);
    const dim3 grid((unsigned) (blocks < 0x7fffffffLL ? blocks : 0x7fffffffLL));
    if (words) launch_kernel(k_embedding<T, V>, grid, dim3(kEmbThreads), st, a);
    else launch_kernel(k_embedding<T, 1>, grid, dim3(kEmbThreads), st, a);
    ND_CUDA(cudaGetLastError());
    return kOk;
}

template <class T, int KPT> Status launch_order_cluster(const OrderArgs &o, unsigned grid, unsigned cluster, cudaStream_t st) {
    const size_t smem = o.passes > 1 ? 2 * sizeof(unsigned) * kOrdThreads * KPT : 0;
    static std::atomic<unsigned long long> asked{0};
    ND_TRY(allow_shared(reinterpret_cast<const void *>(k_order_cluster<T, KPT>), smem + sizeof(OrderShared), asked));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(kOrdThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_tuning[kTuneOverlapLaunch] ? 2 : 1;
    cudaLaunchKernelEx(&cfg, k_order_cluster<T, KPT>, o);
    count_launch();
    return kOk;
}

// Sorts the tokens (and zeroes the table when `o.zero` is set); *result says which pair of lists holds the outcome.
template <class T> Status order_tokens(OrderArgs &o, int *result, cudaStream_t st) {
    int width = 1;
    while (width < 32 && (o.vocab >> width) != 0) width++;               // keys go up to vocab itself
    o.passes = (int) ceil_div(width, kOrdBits);
    o.bits = (int) ceil_div(width, o.passes);
    const unsigned zeroCtas = o.zero ? (unsigned) kNumSMs * 3 : 0u;
    // One cluster, of as many CTAs as the tokens fill with the fewest keys per thread that let eight CTAs hold them
    // all: the time goes with the keys per thread.
    for (int kpt = 1; kpt <= kOrdMaxKeys; kpt *= 2) {
        const LL tile = (LL) kOrdThreads * kpt;
        if (o.n > tile * kOrdCluster) continue;
        unsigned cluster = 1;
        while (cluster * tile < o.n) cluster *= 2;
        o.sortCtas = (int) cluster;
        *result = 0;
        const unsigned grid = cluster + zeroCtas / cluster * cluster;
        switch (kpt) {
            case 1: return launch_order_cluster<T, 1>(o, grid, cluster, st);
            case 2: return launch_order_cluster<T, 2>(o, grid, cluster, st);
            case 4: return launch_order_cluster<T, 4>(o, grid, cluster, st);
            case 8: return launch_order_cluster<T, 8>(o, grid, cluster, st);
            default: return launch_order_cluster<T, 16>(o, grid, cluster, st);
        }
    }
    *result = (o.passes - 1) & 1;
    o.tiles = (unsigned) ceil_div(o.n, kOrdThreads * kOrdMaxKeys);
    if (o.zero) launch_kernel(k_zero_rows<T>, dim3((unsigned) kNumSMs * 4), dim3(kOrdThreads), st, o);
    const unsigned grid = o.tiles < (unsigned) kNumSMs * 2 ? o.tiles : (unsigned) kNumSMs * 2;
    for (int pass = 0; pass < o.passes; pass++) {
        launch_kernel(k_order_count, dim3(grid), dim3(kOrdThreads), st, o, pass);
        launch_kernel(k_order_starts, dim3(1), dim3(kOrdThreads), st, o);
        launch_kernel(k_order_scatter, dim3(grid), dim3(kOrdThreads), st, o, pass);
    }
    return kOk;
}

template <class T, int V> void launch_sums(const EmbArgs &a, dim3 grid, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(kEmbThreads); cfg.stream = st;
    cfg.dynamicSmemBytes = sizeof(unsigned) * (2 * kEmbMaxChunk + 2) * (kEmbThreads / a.group);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_tuning[kTuneOverlapLaunch] ? 1 : 0;
    cudaLaunchKernelEx(&cfg, k_embedding_sums<T, V>, a);
    count_launch();
}

template <class T> Status emb_gradient(EmbArgs &a, OrderArgs &o, bool words, cudaStream_t st) {
    typedef typename Elem<T>::C C;
    constexpr int V = Elem<T>::kVec;
    if (a.n == 0) {
        if (o.zero) launch_kernel(k_zero_rows<T>, dim3((unsigned) kNumSMs * 2), dim3(kOrdThreads), st, o);
        ND_CUDA(cudaGetLastError());
        return kOk;
    }
    a.words = (unsigned) (words ? a.cols / V : a.cols);
    a.group = group_for(a.words);
    const LL slices = ceil_div(a.words, a.group);
    // Longer chunks mean fewer partial sums, shorter ones more CTAs: the longest of 8 .. 64 that still gives every SM
    // three CTAs, as far as there are that many rows.
    LL chunk = kEmbMaxChunk;
    while (chunk > 8 && ceil_div(a.n, chunk) * slices * a.group / kEmbThreads < (LL) kNumSMs * 3) chunk /= 2;
    a.chunk = (unsigned) chunk;
    a.chunks = (unsigned) ceil_div(a.n, chunk);
    const size_t list = round_up((size_t) a.n * sizeof(unsigned), 256);
    const size_t hist = round_up((size_t) ceil_div(a.n, kOrdThreads * kOrdMaxKeys) * kOrdBins * sizeof(unsigned), 256);
    Scratch scratch(st);
    ND_TRY(scratch.alloc(4 * list + hist + (size_t) a.chunks * 2 * (size_t) a.cols * sizeof(C)));
    for (int k = 0; k < 2; k++) { o.key[k] = scratch.at<unsigned>(2 * k * list); o.pos[k] = scratch.at<unsigned>((2 * k + 1) * list); }
    o.hist = scratch.at<unsigned>(4 * list);
    a.partials = scratch.at<void>(4 * list + hist);
    int result = 0;
    ND_TRY(order_tokens<T>(o, &result, st));
    a.key = o.key[result]; a.pos = o.pos[result];
    const dim3 grid((unsigned) ceil_div(a.chunks, kEmbThreads / a.group), (unsigned) (slices < 65535 ? slices : 65535));
    if (words) launch_sums<T, V>(a, grid, st);
    else launch_sums<T, 1>(a, grid, st);
    if (a.chunks > 1) {
        const LL slabs = ceil_div(a.cols, 128);
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
