// Log probabilities of given tokens under rows of logits, with the entropy of every row and its best alternatives, and
// the gradient of log probabilities and entropies. With c the scale (an inverse temperature) and m a row's maximum:
//
//   d_j = c (x_j - m),  s = sum_j exp(d_j),  u = sum_j d_j exp(d_j)
//   log p_j = d_j - log s,   logProb = log p_t,   entropy = -sum_j p_j log p_j = log s - u / s
//   dx_j = c ( g (delta_jt - p_j) - h p_j (log p_j + entropy) )      for upstream gradients g, h
//
// LogSoftMax followed by a gather writes the whole matrix to pick one value of each row, and an entropy takes three
// more sweeps. Here a row is read once, as fast as HBM delivers it, each thread carrying the running maximum of what it
// has seen and the two sums relative to it, rescaled in the rare step that moves the maximum; nothing but the results
// is written. Sums are held in float for float and half data, in double for double. Measured: 4096 rows of 32768 floats,
// 82 us = 6.5 TB/s a call among others, 94 with cold caches (HBM); 8192 rows of 50001 halves with entropy, 154 us = 5.3
// TB/s with cold caches (HBM and, at 0.7, the exponentials).
//
// Exponentials are powers of two (one special-function instruction, relative error 2^-22), so c carries the factor log2(e).
// Half data: the distance from the reference point is one fused multiply-add, x c - R. R is the rounded m c; every term is
// relative to the same R, so its rounding cancels as long as it is a small exponent itself, which it is up to
// 65504 c = 2^24 (half a unit in R's last place: 1/2). Larger scales, and float data at any, subtract first, (x - m) c: a
// rounding of m c that passes 126 would leave nothing of the maximum's own term, and a float of the type's lowest value, the
// usual mask, would overflow when multiplied. Masked entries (-inf) contribute nothing, a row of nothing else has log
// probability -inf, entropy 0 and gradient 0; a row with a NaN or +inf answers NaN.
//
// Few rows: the CTAs of a cluster of up to 8 share a row and join their sums through distributed shared memory, so that
// eight rows of a large vocabulary still keep 64 SMs reading.
//
// Best alternatives need no second sweep: each thread already knows the largest value of its slice and, with a batch
// number kept beside it, where it stands. The k-th best of these is a lower bound for the k-th best of all; only the
// slices of the k threads at or above it are read again (k / 256 of the row, mostly from L2), what reaches the bound is
// collected and ranked by counting. Equal values are ordered by index. Should the collection overflow, or the row hold a
// NaN (which ranks first), the best are taken one by one.
#include "../../include/nd4j_b200.h"
#include <cfloat>
#include <cooperative_groups.h>
#include "device_utils.cuh"
#include "entry_checks.h"

namespace cg = cooperative_groups;

namespace nd4jb200 {
namespace {

// Threads per CTA. 256 with six CTAs per SM keep their loads overlapping one another's sums (4096 rows of 32768 floats:
// 94 us; 512 threads, three CTAs: 94; two, the next batch fetched ahead: 107; 8192 rows of 50001 halves: 152, 182, 205).
// A warp of its own takes a row of up to 512 words (8192 rows of 1000 floats: 37 us with 256 threads).
constexpr int kLpThreads = 256;
constexpr int kLpShortWords = 512;
template <class T> constexpr int lp_ctas(int threads) { return threads == 32 ? 24 : (sizeof(T) == 8 ? 4 : 6); }
constexpr int kLpBatch = 4;                 // 128-bit words a thread has in flight
constexpr int kLpMaxTop = 64;
constexpr int kLpList = 1024;               // collected candidates, at most
constexpr int kLpNone = 0x7fffffff;

// Exponent arithmetic of one element type. A reference point stands for a maximum; dist() is an element's exponent
// relative to it, gap() that of another reference point. FAR: half data at a scale that its fused form does not serve.
template <class T, bool FAR = false> struct LpMath;
template <> struct LpMath<__half, false> {
    typedef float C;
    static constexpr float kFloor = -65504.f;       // reference of a row without values: the lowest finite one
    static constexpr double kUnit = 1.4426950408889634;          // log2(e): exponents are of base two
    static ND_D float ref(float m, float c) { return fmaxf(m, kFloor) * c; }
    static ND_D float dist(float x, float r, float c) { return fmaf(x, c, -r); }
    static ND_D float gap(float a, float b, float) { return a - b; }
    static ND_D float off(float m, float r, float c) { return fmaf(-m, c, r); }         // exponent of the reference over the maximum's
};
template <> struct LpMath<float, false> {
    typedef float C;
    static constexpr float kFloor = -FLT_MAX;
    static constexpr double kUnit = 1.4426950408889634;
    static ND_D float ref(float m, float) { return fmaxf(m, kFloor); }
    static ND_D float dist(float x, float r, float c) { return (x - r) * c; }
    static ND_D float gap(float a, float b, float c) { return (a - b) * c; }
    static ND_D float off(float, float, float) { return 0.f; }
};
template <> struct LpMath<__half, true> : LpMath<float, false> {};
template <> struct LpMath<double, false> {
    typedef double C;
    static constexpr double kFloor = -DBL_MAX;
    static constexpr double kUnit = 1.0;
    static ND_D double ref(double m, double) { return fmax(m, kFloor); }
    static ND_D double dist(double x, double r, double c) { return (x - r) * c; }
    static ND_D double gap(double a, double b, double c) { return (a - b) * c; }
    static ND_D double off(double, double, double) { return 0.0; }
};
// the larger of two, a number before a NaN
ND_D float lp_max(float a, float b) { return fmaxf(a, b); }
ND_D double lp_max(double a, double b) { return fmax(a, b); }
ND_D float lp_exp(float d) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d)); return r; }
ND_D double lp_exp(double d) { return exp(d); }
ND_D float lp_log(float s) { return log2f(s); }
ND_D double lp_log(double s) { return log(s); }
// an exponent that is finite, for products with a power that has become 0
ND_D float lp_finite(float d) { return fmaxf(d, -1000.f); }
ND_D double lp_finite(double d) { return fmax(d, -10000.0); }

struct LpArgs {
    const void *x;
    LL rows, row, col;               // element strides
    int vocab;
    const LL *tokens;                // may be null (forward): no token is asked for
    double scale;
    void *logProbs, *entropy, *rowMax, *logSum;      // wide values, each may be null (forward)
    int k;
    LL *topTokens;
    void *topLogProbs;
    int cluster;
    // gradient
    const void *gLogProbs, *gEntropy;
    void *dx;
    LL dRow, dCol;
    int chunks;                      // CTAs per row
};

// How a row's elements are dealt to threads: `head` elements up to the first 16-byte boundary, then words of V, then
// the rest. (V = 1, any stride: all of them are words.)
template <class T, int V> struct LpRow {
    const T *x;
    LL col;
    int head, words, tail;
    ND_D LpRow(const LpArgs &a, LL r) {
        x = static_cast<const T *>(a.x) + r * a.row;
        col = a.col;
        head = 0;
        if (V > 1) {
            head = (int) (((16 - (reinterpret_cast<unsigned long long>(x) & 15)) & 15) / sizeof(T));
            if (head > a.vocab) head = a.vocab;
        }
        words = (a.vocab - head) / V;
        tail = a.vocab - head - words * V;
    }
    ND_D int index(int word) const { return head + word * V; }
    ND_D T at(int i) const { return x[V > 1 ? (LL) i : (LL) i * col]; }
    ND_D void load(int word, T (&v)[V]) const {
        if constexpr (V == 1) v[0] = x[(LL) word * col];
        else *reinterpret_cast<uint4 *>(v) = __ldcs(reinterpret_cast<const uint4 *>(x + index(word)));
    }
    // The elements of the slice of thread `slot` in a row shared by `span` threads: (index, value) handed to `f`, ascending.
    template <class F> ND_D void each(int slot, int span, F f) const {
        if (V > 1 && slot < head) f(slot, Elem<T>::to_c(at(slot)));
        for (int w = slot; w < words; w += span) {
            alignas(16) T v[V];
            load(w, v);
#pragma unroll
            for (int k = 0; k < V; k++) f(index(w) + k, Elem<T>::to_c(v[k]));
        }
        if (V > 1 && slot < tail) f(index(words) + slot, Elem<T>::to_c(at(index(words) + slot)));
    }
};

// Largest of the words of a batch.
template <class T, int V, int N> ND_D typename LpMath<T>::C lp_batch_max(const T (&v)[N][V]) {
    typedef typename LpMath<T>::C C;
    if constexpr (sizeof(T) == 2 && V > 1) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&v[0][0]);
        __half2 m = h[0];
#pragma unroll
        for (int j = 1; j < N * V / 2; j++) m = __hmax2(m, h[j]);
        const float lo = __low2float(m), hi = __high2float(m);
        return lp_max(lp_max(lo, hi), -C(INFINITY));                // all NaN: nothing
    } else {
        C m = -C(INFINITY);
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int k = 0; k < V; k++) m = lp_max(m, Elem<T>::to_c(v[j][k]));
        return m;
    }
}

// Moves sums from one reference point to another. A reference far below leaves a power of 0: its sum must not meet an
// infinite gap.
template <class M, bool ENT> ND_D void lp_move(typename M::C &s, typename M::C &u, typename M::C from, typename M::C to,
                                               typename M::C c) {
    typedef typename M::C C;
    const C g = M::gap(from, to, c), f = lp_exp(g);
    if (ENT) u = f == C(0) ? C(0) : f * fma(lp_finite(g), s, u);
    s *= f;
}

// A candidate as a key that orders like (value, lower index first): the value's bits made order-preserving, a NaN above
// all, -0 as +0; then the complement of the index. Comparing keys takes two instructions, which the ranking by counting
// below lives on. The least key stands for "none": -inf never becomes a candidate.
template <class C> struct LpKey;
template <> struct LpKey<float> {
    unsigned long long k;
    static ND_D LpKey none() { return LpKey{0ull}; }
    static ND_D LpKey of(float v, int i) {
        const unsigned b = __float_as_uint(v + 0.f);
        const unsigned o = v != v ? 0xffffffffu : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
        return LpKey{((unsigned long long) o << 32) | (0xffffffffu - (unsigned) i)};
    }
    ND_D int index() const { return (int) (0xffffffffu - (unsigned) k); }
    ND_D float value() const {
        const unsigned o = (unsigned) (k >> 32);
        return o == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
    }
    ND_D bool above(const LpKey &o) const { return k > o.k; }
    ND_D bool same(const LpKey &o) const { return k == o.k; }
    // the greatest of the warp
    ND_D LpKey warp_best() const {
        const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned) (k >> 32));
        const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned) (k >> 32) == hi ? (unsigned) k : 0u);
        return LpKey{((unsigned long long) hi << 32) | lo};
    }
};
template <> struct LpKey<double> {
    unsigned long long k;
    unsigned i;                                   // complement of the index
    static ND_D LpKey none() { return LpKey{0ull, 0u}; }
    static ND_D LpKey of(double v, int i) {
        const unsigned long long b = (unsigned long long) __double_as_longlong(v + 0.0);
        const unsigned long long o = v != v ? ~0ull : b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
        return LpKey{o, 0xffffffffu - (unsigned) i};
    }
    ND_D int index() const { return (int) (0xffffffffu - i); }
    ND_D double value() const {
        return __longlong_as_double(k == ~0ull ? 0x7fffffffffffffffll : (long long) (k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
    }
    ND_D bool above(const LpKey &o) const { return k > o.k || (k == o.k && i > o.i); }
    ND_D bool same(const LpKey &o) const { return k == o.k && i == o.i; }
    ND_D LpKey warp_best() const {
        LpKey b = *this;
        for (int m = 16; m > 0; m >>= 1) {
            const LpKey o = {__shfl_xor_sync(0xffffffffu, b.k, m), __shfl_xor_sync(0xffffffffu, b.i, m)};
            if (o.above(b)) b = o;
        }
        return b;
    }
};

template <class C> struct LpSum { C ref, s, u; };

template <class C, int LT> struct LpShared {
    static constexpr int kLpWarps = LT / 32;
    C sums[kLpWarps], sumsU[kLpWarps], tops[kLpWarps];
    C ctaMax, ctaS, ctaU;                    // read by the other CTAs of a cluster
    LpKey<C> warpBest[kLpWarps];
    LpKey<C> list[kLpList];                  // candidates
    LpKey<C> best[kLpMaxTop];                // this CTA's best, in order (read by the leading CTA of a cluster)
    int slots[kLpMaxTop];
    int counts[8];
    int count, numBest;
};

// How many of the n keys of a list in shared memory are above `mine`.
template <class C> ND_D int lp_rank(const LpKey<C> *list, int n, const LpKey<C> &mine) {
    int above = 0, q = 0;
    for (; q + 8 <= n; q += 8) {
#pragma unroll
        for (int e = 0; e < 8; e++) above += list[q + e].above(mine);
    }
    for (; q < n; q++) above += list[q].above(mine);
    return above;
}

// The k best of the CTA's part of a row into s.best, their number into s.numBest. `mine`: the thread's own best (none:
// nothing above -inf). `odd`: the row holds a NaN or +inf.
template <class T, int V, int LT>
ND_D void lp_select(const LpRow<T, V> &row, const LpKey<typename LpMath<T>::C> &mine, bool odd, int k, int rank, int span,
                    LpShared<typename LpMath<T>::C, LT> &s) {
    constexpr int kLpWarps = LT / 32;
    typedef typename LpMath<T>::C C;
    typedef LpKey<C> Key;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slot = rank * LT + threadIdx.x;
    const Key none = Key::none();
    bool slow = odd;
    if (!odd) {
        // a first bound: of every warp the r-th best, of these the least; at least r * kLpWarps >= k threads reach it
        const int rounds = (k + kLpWarps - 1) / kLpWarps;
        Key left = mine, bound = none;
        for (int q = 0; q < rounds; q++) {
            bound = left.warp_best();
            if (bound.same(left)) left = none;
        }
        if (lane == 0) s.warpBest[warp] = bound;
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kLpWarps; w++) if (bound.above(s.warpBest[w])) bound = s.warpBest[w];
        // (a warp with fewer values gives none: then every thread with a value counts)
        const bool source = mine.above(none) && !bound.above(mine);
        if (source) s.list[atomicAdd(&s.count, 1)] = mine;
        __syncthreads();
        // the k-th best of them exactly
        const int n0 = s.count;
        const int place = source ? lp_rank(s.list, n0, mine) : k;
        __syncthreads();
        if (place < k) s.slots[place] = threadIdx.x;
        if (place == k - 1) s.warpBest[0] = mine;
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        const int numSlots = n0 < k ? n0 : k;
        const Key least = n0 < k ? none : s.warpBest[0];
        // what reaches it, from the slices of those threads; every word of them is a thread's
        auto offer = [&](int j, C w) {
            const Key key = Key::of(w, j);
            if (w > -C(INFINITY) && !least.above(key)) {
                const int p = atomicAdd(&s.count, 1);
                if (p < kLpList) s.list[p] = key;
            }
        };
        const int perSlot = (row.words + span - 1) / span + 1;          // the first: elements beside the words
        for (int item = threadIdx.x; item < numSlots * perSlot; item += LT) {
            const int q = item / perSlot, e = item - q * perSlot;
            const int owner = rank * LT + s.slots[q];
            if (e == 0) {
                if (V > 1 && owner < row.head) offer(owner, Elem<T>::to_c(row.at(owner)));
                if (V > 1 && owner < row.tail) offer(row.index(row.words) + owner, Elem<T>::to_c(row.at(row.index(row.words) + owner)));
            } else if (owner + (e - 1) * span < row.words) {
                const int w = owner + (e - 1) * span;
                alignas(16) T x[V];
                row.load(w, x);
#pragma unroll
                for (int f = 0; f < V; f++) offer(row.index(w) + f, Elem<T>::to_c(x[f]));
            }
        }
        __syncthreads();
        const int n = s.count;
        slow = n > kLpList;
        if (!slow) {
            for (int q = threadIdx.x; q < n; q += LT) {
                const Key key = s.list[q];
                const int at = lp_rank(s.list, n, key);
                if (at < k) s.best[at] = key;
            }
            if (threadIdx.x == 0) s.numBest = n < k ? n : k;
        }
        __syncthreads();
    }
    if (!slow) return;
    // one by one: the best of the threads' bests is taken, its owner looks for its next
    Key pop = none, next = none;
    bool first = true;
    auto look = [&]() {
        next = none;
        row.each(slot, span, [&](int j, C w) {
            if (!(w > -C(INFINITY)) && w == w) return;
            const Key key = Key::of(w, j);
            if ((first || pop.above(key)) && key.above(next)) next = key;
        });
    };
    look();
    first = false;
    int taken = 0;
    for (; taken < k; taken++) {
        Key b = next.warp_best();
        if (lane == 0) s.warpBest[warp] = b;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kLpWarps; w++) if (s.warpBest[w].above(b)) b = s.warpBest[w];
        __syncthreads();
        if (!b.above(none)) break;
        if (threadIdx.x == 0) s.best[taken] = b;
        pop = b;
        if (next.same(b)) look();
    }
    if (threadIdx.x == 0) s.numBest = taken;
    __syncthreads();
}

template <class T, int V, bool ENT, bool TOP, int LT, bool FAR>
__global__ void __launch_bounds__(LT, lp_ctas<T>(LT)) k_token_log_probs(const LpArgs a) {
    grid_dependency_sync();
    typedef LpMath<T, FAR> M;
    typedef typename M::C C;
    constexpr int kLpWarps = LT / 32;
    __shared__ LpShared<C, LT> s;
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = a.cluster, rank = ctas > 1 ? (int) cl.block_rank() : 0;
    const int span = ctas * LT, slot = rank * LT + threadIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const C c = (C) (a.scale * M::kUnit), back = (C) (1.0 / M::kUnit);
    const C nan = (C) NAN;
    for (LL r = blockIdx.x / ctas; r < a.rows; r += gridDim.x / ctas) {
        const LL token = a.tokens ? a.tokens[r] : 0;
        if (token < 0) {                                        // padding: nothing is read
            if (rank == 0) {
                if (threadIdx.x == 0) {
                    if (a.logProbs) static_cast<C *>(a.logProbs)[r] = C(0);
                    if (a.entropy) static_cast<C *>(a.entropy)[r] = C(0);
                    if (a.rowMax) static_cast<C *>(a.rowMax)[r] = C(0);
                    if (a.logSum) static_cast<C *>(a.logSum)[r] = C(0);
                }
                for (int q = threadIdx.x; TOP && q < a.k; q += LT) {
                    a.topTokens[r * a.k + q] = -1;
                    static_cast<C *>(a.topLogProbs)[r * a.k + q] = C(0);
                }
            }
            continue;
        }
        const LpRow<T, V> row(a, r);
        C top = -C(INFINITY);
        int batch = kLpNone;                                    // where `top` was met: a word, or -1 head, -2 tail
        C ref = M::ref(top, c), sum = C(0), sumU = C(0);
        auto meet = [&](C bm, int where) {
            if (bm > top) {
                const C to = M::ref(bm, c);
                if (to > ref) { lp_move<M, ENT>(sum, sumU, ref, to, c); ref = to; }
                top = bm;
                batch = where;
            }
        };
        auto add = [&](C x, C &s0, C &u0) {
            const C d = M::dist(x, ref, c), e = lp_exp(d);
            s0 += e;
            if (ENT) u0 = fma(e, lp_finite(d), u0);
        };
        auto fetch = [&](int w, T (&v)[kLpBatch][V]) {
            if (w + (kLpBatch - 1) * span < row.words) {
#pragma unroll
                for (int j = 0; j < kLpBatch; j++) row.load(w + j * span, v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < kLpBatch; j++) {
                    if (w + j * span < row.words) row.load(w + j * span, v[j]);
                    else {
#pragma unroll
                        for (int k = 0; k < V; k++) v[j][k] = Elem<T>::from_c(-C(INFINITY));
                    }
                }
            }
        };
        if (V > 1 && slot < row.head) { const C x = Elem<T>::to_c(row.at(slot)); meet(x, -1); add(x, sum, sumU); }
        alignas(16) T v[kLpBatch][V];
        for (int w = slot; w < row.words; w += kLpBatch * span) {
            fetch(w, v);
            meet(lp_batch_max<T, V, kLpBatch>(v), w);
            C s1 = C(0), u1 = C(0);                             // two chains of additions
#pragma unroll
            for (int j = 0; j < kLpBatch; j += 2)
#pragma unroll
                for (int k = 0; k < V; k++) {
                    add(Elem<T>::to_c(v[j][k]), sum, sumU);
                    add(Elem<T>::to_c(v[j + 1][k]), s1, u1);
                }
            sum += s1;
            if (ENT) sumU += u1;
        }
        if (V > 1 && slot < row.tail) { const C x = Elem<T>::to_c(row.at(row.index(row.words) + slot)); meet(x, -2); add(x, sum, sumU); }

        // over the warp, the CTA, the cluster: first the maximum, then the sums relative to it; every thread gets both
        C m = top;
        for (int o = 16; o > 0; o >>= 1) m = lp_max(m, __shfl_xor_sync(0xffffffffu, m, o));
        __syncthreads();                                        // the shared block may still serve the row before
        if (lane == 0) s.tops[warp] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kLpWarps; w++) m = lp_max(m, s.tops[w]);
        LpSum<C> all = {M::ref(m, c), sum, sumU};
        lp_move<M, ENT>(all.s, all.u, ref, all.ref, c);
        for (int o = 16; o > 0; o >>= 1) {
            all.s += __shfl_xor_sync(0xffffffffu, all.s, o);
            if (ENT) all.u += __shfl_xor_sync(0xffffffffu, all.u, o);
        }
        if (lane == 0) { s.sums[warp] = all.s; s.sumsU[warp] = all.u; }
        __syncthreads();
        all.s = all.u = C(0);
#pragma unroll
        for (int w = 0; w < kLpWarps; w++) { all.s += s.sums[w]; if (ENT) all.u += s.sumsU[w]; }
        if (ctas > 1) {
            if (threadIdx.x == 0) { s.ctaMax = m; s.ctaS = all.s; s.ctaU = all.u; }
            cl.sync();
            // eight independent reads of the other CTAs' shared memory, then the arithmetic
            C qm[8], qs[8], qu[8];
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const LpShared<C, LT> *o = cl.map_shared_rank(&s, q < ctas ? q : 0);
                qm[q] = o->ctaMax;
                qs[q] = o->ctaS;
                qu[q] = ENT ? o->ctaU : C(0);
            }
#pragma unroll
            for (int q = 0; q < 8; q++) m = lp_max(m, qm[q]);
            all.ref = M::ref(m, c);
            all.s = all.u = C(0);
#pragma unroll
            for (int q = 0; q < 8; q++) {
                if (q < ctas) {
                    lp_move<M, ENT>(qs[q], qu[q], M::ref(qm[q], c), all.ref, c);
                    all.s += qs[q];
                    all.u += qu[q];
                }
            }
            cl.sync();
        }
        const bool odd = !(all.s == all.s);
        const C logS = lp_log(all.s);                           // in the exponents' base, relative to all.ref
        const C logSum = (logS + M::off(m, all.ref, c)) * back; // log of the sum relative to the maximum
        // in natural units: a log probability near the type's lowest value is still finite
        auto log_p = [&](C x) { return all.s > C(0) || odd ? (x - m) * (C) a.scale - logSum : -C(INFINITY); };
        if (rank == 0 && threadIdx.x == 0) {
            const bool empty = all.s == C(0);
            if (a.logProbs) {
                C lp = nan;
                if (token < a.vocab) lp = log_p(Elem<T>::load(row.x + (V > 1 ? token : token * row.col)));
                static_cast<C *>(a.logProbs)[r] = lp;
            }
            if (ENT) static_cast<C *>(a.entropy)[r] = empty ? C(0) : (logS - all.u / all.s) * back;
            if (a.rowMax) static_cast<C *>(a.rowMax)[r] = odd ? nan : m;
            if (a.logSum) static_cast<C *>(a.logSum)[r] = empty ? -C(INFINITY) : logSum;
        }
        if (TOP) {
            // where the thread's own best stands
            int mine = kLpNone;
            if (batch == -1) mine = slot;
            else if (batch == -2) mine = row.index(row.words) + slot;
            else if (batch != kLpNone) {
                fetch(batch, v);
#pragma unroll
                for (int j = kLpBatch - 1; j >= 0; j--)
#pragma unroll
                    for (int k = V - 1; k >= 0; k--) if (Elem<T>::to_c(v[j][k]) == top) mine = row.index(batch + j * span) + k;
            }
            typedef LpKey<C> Key;
            lp_select<T, V, LT>(row, mine == kLpNone ? Key::none() : Key::of(top, mine), odd, a.k, rank, span, s);
            if (ctas > 1) {
                cl.sync();
                if (rank == 0) {
                    // the CTAs' lists, at most 8 * 64 entries, ranked once more
                    if (threadIdx.x < ctas) s.counts[threadIdx.x] = cl.map_shared_rank(&s, threadIdx.x)->numBest;
                    __syncthreads();
                    int n = 0;
                    for (int q = 0; q < ctas; q++) {
                        for (int e = threadIdx.x; e < s.counts[q]; e += LT) s.list[n + e] = cl.map_shared_rank(&s, q)->best[e];
                        n += s.counts[q];
                    }
                    __syncthreads();
                    for (int e = threadIdx.x; e < n; e += LT) {
                        const Key key = s.list[e];
                        const int at = lp_rank(s.list, n, key);
                        if (at < a.k) s.best[at] = key;
                    }
                    if (threadIdx.x == 0) s.numBest = n < a.k ? n : a.k;
                    __syncthreads();
                }
            }
            if (rank == 0) {
                const int n = s.numBest;
                for (int q = threadIdx.x; q < n; q += LT) {
                    a.topTokens[r * a.k + q] = s.best[q].index();
                    static_cast<C *>(a.topLogProbs)[r * a.k + q] = odd ? nan : log_p(s.best[q].value());
                }
                // fewer values than asked for: masked entries follow, the first of them first
                if (n < a.k && warp == 0) {
                    int have = n;
                    for (int j0 = 0; j0 < a.vocab && have < a.k; j0 += 32) {
                        const int j = j0 + lane;
                        const bool masked = j < a.vocab && Elem<T>::to_c(row.at(j)) == -C(INFINITY);
                        const unsigned ballot = __ballot_sync(0xffffffffu, masked);
                        const int at = have + __popc(ballot & ((1u << lane) - 1u));
                        if (masked && at < a.k) {
                            a.topTokens[r * a.k + at] = j;
                            static_cast<C *>(a.topLogProbs)[r * a.k + at] = odd ? nan : -C(INFINITY);
                        }
                        have += __popc(ballot);
                    }
                }
            }
            if (ctas > 1) cl.sync();                            // the leading CTA has read the others' lists
        }
    }
}

// ---- gradient ----------------------------------------------------------------------------------------------------
// Reads a word, writes a word. What costs beside the traffic is the wait for a row's values before anything can be
// computed, so small CTAs, many per SM, each with all its words in flight from the start (8192 rows of 50001 halves: 291 us
// with 256 threads of 4 words that waited for the row's values first, 272 so, 307 where the maximum is loaded only for
// tokens inside the row; 4096 rows of 32768 floats with entropy: 182, 168).
constexpr int kLpGradThreads = 128;
template <class T> constexpr int kLpGradWords = sizeof(T) == 2 ? 8 : 4;       // per thread
template <class T> constexpr int kLpGradCtas = sizeof(T) == 2 ? 8 : 10;

template <class T, int V, bool ENT, bool FAR>
__global__ void __launch_bounds__(kLpGradThreads, kLpGradCtas<T>) k_token_log_probs_grad(const LpArgs a) {
    grid_dependency_sync();
    typedef LpMath<T, FAR> M;
    typedef typename M::C C;
    constexpr int W = kLpGradWords<T>;
    const C c = (C) (a.scale * M::kUnit), unit = (C) M::kUnit, back = (C) (1.0 / M::kUnit);
    const LL units = a.rows * a.chunks;
    for (LL b = blockIdx.x; b < units; b += gridDim.x) {
        const LL r = b / a.chunks;
        const int chunk = (int) (b - r * a.chunks);
        const LpRow<T, V> row(a, r);
        T *dx = static_cast<T *>(a.dx) + r * a.dRow;
        // the words are asked for before the row's values are known, padding or not: the two waits become one
        const int first = chunk * (kLpGradThreads * W) + threadIdx.x;
        alignas(16) T v[W][V];
#pragma unroll
        for (int j = 0; j < W; j++)
            if (first + j * kLpGradThreads < row.words) row.load(first + j * kLpGradThreads, v[j]);
        const LL token = a.tokens[r];
        C m = static_cast<const C *>(a.rowMax)[r];                // loaded for any token: it must not wait for that one
        const C logSum = static_cast<const C *>(a.logSum)[r];
        const C g = (C) a.scale * (a.gLogProbs ? static_cast<const C *>(a.gLogProbs)[r] : C(0));
        const C h = ENT ? (C) a.scale * static_cast<const C *>(a.gEntropy)[r] : C(0);
        if (token >= a.vocab) m = (C) NAN;                        // a row of NaN of any row, as where it holds a NaN
        const bool none = token < 0 || m == -C(INFINITY);         // padding, or a row without a value: zeros
        const C ref = M::ref(m, c), shift = logSum * unit - M::off(m, ref, c);
        C A = ENT ? -(g + h * static_cast<const C *>(a.entropy)[r]) : -g;
        const C B = ENT ? -h * back : C(0);
        if (m != m) A = (C) NAN;
        auto one = [&](C x) -> C {
            const C lp = M::dist(x, ref, c) - shift, p = lp_exp(lp);
            return ENT ? p * fma(B, lp_finite(lp), A) : p * A;
        };
        const bool aligned = V > 1 && (reinterpret_cast<unsigned long long>(dx + row.head) & 15) == 0;
#pragma unroll
        for (int j = 0; j < W; j++) {
            const int w = first + j * kLpGradThreads;
            if (w >= row.words) break;
            const int i = row.index(w);
            const LL at = none ? -1 : token - i;
#pragma unroll
            for (int k = 0; k < V; k++) {
                C d = none ? C(0) : one(Elem<T>::to_c(v[j][k]));
                if (at == k) d += g;
                v[j][k] = Elem<T>::from_c(d);
            }
            if (V == 1) dx[(LL) i * a.dCol] = v[j][0];
            else if (aligned) __stcs(reinterpret_cast<uint4 *>(dx + i), *reinterpret_cast<const uint4 *>(v[j]));
            else {
#pragma unroll
                for (int k = 0; k < V; k++) dx[i + k] = v[j][k];
            }
        }
        if (V > 1 && chunk == 0 && threadIdx.x < 2 * V) {       // the elements before and behind the words
            const int k = threadIdx.x % V;
            const bool headSide = threadIdx.x < V;
            if (k < (headSide ? row.head : row.tail)) {
                const int i = headSide ? k : row.index(row.words) + k;
                C d = none ? C(0) : one(Elem<T>::to_c(row.at(i)));
                if (!none && token == i) d += g;
                dx[i] = Elem<T>::from_c(d);
            }
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------
template <class K> void launch_log_probs(K kernel, const LpArgs &a, unsigned grid, int threads, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3((unsigned) threads); cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned) a.cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = g_tuning[kTuneOverlapLaunch] ? attr : attr + 1;
    cfg.numAttrs = g_tuning[kTuneOverlapLaunch] ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, a);
    count_launch();
}

// Half data leaves the fused form once the rounding of the largest 65504 c exceeds half an exponent (scale above 177). The
// other form takes an instruction more per element: 8192 rows of 50001 halves, 160 us against 154; their gradient 324
// against 272.
bool lp_far(const LpArgs &a) { return a.scale * LpMath<__half>::kUnit * 65504.0 > 16777216.0; }

template <class T, int V, int LT, bool FAR> void lp_forward_kernels(const LpArgs &a, unsigned grid, cudaStream_t st) {
    if (a.k > 0) {
        if (a.entropy) launch_log_probs(k_token_log_probs<T, V, true, true, LT, FAR>, a, grid, LT, st);
        else launch_log_probs(k_token_log_probs<T, V, false, true, LT, FAR>, a, grid, LT, st);
    } else {
        if (a.entropy) launch_log_probs(k_token_log_probs<T, V, true, false, LT, FAR>, a, grid, LT, st);
        else launch_log_probs(k_token_log_probs<T, V, false, false, LT, FAR>, a, grid, LT, st);
    }
}

template <class T, bool FAR> Status lp_forward(LpArgs &a, cudaStream_t st) {
    constexpr int V = Elem<T>::kVec;
    // Rows that would leave SMs idle are shared by a cluster, as long as every CTA keeps at least one batch.
    a.cluster = 1;
    const LL run = a.col == 1 ? V : 1;
    const LL perCta = (LL) kLpThreads * kLpBatch * run;
    const bool shortRows = a.col == 1 && a.vocab <= kLpShortWords * run;
    while (!shortRows && a.cluster < 8 && a.rows * a.cluster * 2 <= kNumSMs * 2 && a.vocab >= a.cluster * 2 * perCta) a.cluster *= 2;
    LL grid = a.rows * a.cluster;
    if (grid > 0x7fffffff / 8 * 8) grid = 0x7fffffff / 8 * 8;
    if (a.col == 1) {
        if (shortRows) lp_forward_kernels<T, V, 32, FAR>(a, (unsigned) grid, st);
        else lp_forward_kernels<T, V, kLpThreads, FAR>(a, (unsigned) grid, st);
    } else {
        lp_forward_kernels<T, 1, kLpThreads, FAR>(a, (unsigned) grid, st);
    }
    ND_CUDA(cudaGetLastError());
    return kOk;
}

template <class T, bool FAR> Status lp_gradient(LpArgs &a, cudaStream_t st) {
    constexpr int V = Elem<T>::kVec;
    const bool unit = a.col == 1 && a.dCol == 1;
    a.chunks = (int) ceil_div(ceil_div(a.vocab, unit ? V : 1), (LL) kLpGradThreads * kLpGradWords<T>);
    const LL units = a.rows * a.chunks;
    const dim3 grid((unsigned) (units < 0x7fffffffLL ? units : 0x7fffffffLL));
    const dim3 block(kLpGradThreads);
    if (unit) {
        if (a.gEntropy) launch_kernel(k_token_log_probs_grad<T, V, true, FAR>, grid, block, st, a);
        else launch_kernel(k_token_log_probs_grad<T, V, false, FAR>, grid, block, st, a);
    } else {
        if (a.gEntropy) launch_kernel(k_token_log_probs_grad<T, 1, true, FAR>, grid, block, st, a);
        else launch_kernel(k_token_log_probs_grad<T, 1, false, FAR>, grid, block, st, a);
    }
    ND_CUDA(cudaGetLastError());
    return kOk;
}

Status lp_shape(const char *what, const ShapeDesc &d) {
    if (d.rank != 2) return bad_arg(std::string(what) + ": the logits must be of rank 2, one row for each token");
    if (d.shape[1] < 1 && d.shape[0] > 0) return bad_arg(std::string(what) + ": rows without entries");
    if (d.shape[1] > (1LL << 30)) {
        set_error(std::string(what) + ": rows of more than 2^30 entries are not served");
        return kTooLarge;
    }
    return kOk;
}
Status lp_scale(int dtype, double scale) {
    // the largest difference of two halves, times the scale, has to stay a finite float
    const double s = dtype == kF64 ? scale : (double) (float) scale;
    if (!(s > 0 && scale <= 1e30)) return bad_arg("log probabilities: scale must be positive and at most 1e30");
    return kOk;
}

struct LpOut { const void *p; const char *name; size_t size; LL n; };

Status lp_forward_entry(void *stream, int dtype, const void *logits, const Nd4jLong *logitsShapeInfo, const Nd4jLong *tokens,
                        double scale, void *logProbs, void *entropy, void *rowMax, void *logSum, int k, Nd4jLong *topTokens,
                        void *topLogProbs) {
    ND_TRY(require_dtype(dtype));
    ND_TRY(lp_scale(dtype, scale));
    ShapeDesc d;
    ND_TRY(parse_shape(logitsShapeInfo, "logitsShapeInfo", &d));
    ND_TRY(lp_shape("log probabilities", d));
    if (k < 0 || k > kLpMaxTop) return bad_arg("log probabilities: k must lie between 0 and 64");
    if (d.shape[0] == 0) return kOk;
    if (k > d.shape[1]) return bad_arg("log probabilities: k exceeds the number of entries of a row");
    const size_t elem = size_of_dtype(dtype), wide = size_of_wide(dtype);
    ND_TRY(require(logits, "logits"));
    ND_TRY(require_aligned(logits, elem, "logits"));
    if (logProbs) ND_TRY(require(tokens, "tokens"));
    if (k > 0) { ND_TRY(require(topTokens, "topTokens")); ND_TRY(require(topLogProbs, "topLogProbs")); }
    const LL rows = d.shape[0];
    const LpOut outs[] = {{logProbs, "logProbs", wide, rows}, {entropy, "entropy", wide, rows}, {rowMax, "rowMax", wide, rows},
                          {logSum, "logSum", wide, rows}, {k > 0 ? topTokens : nullptr, "topTokens", 8, rows * k},
                          {k > 0 ? topLogProbs : nullptr, "topLogProbs", wide, rows * k}};
    const Span sx = span_of(logits, d, elem), st = span_of(tokens, tokens ? rows : 0, 8);
    bool any = false;
    for (int i = 0; i < 6; i++) {
        if (!outs[i].p) continue;
        any = true;
        ND_TRY(require_aligned(outs[i].p, outs[i].size, outs[i].name));
        const Span so = span_of(outs[i].p, outs[i].n, outs[i].size);
        ND_TRY(check_apart(so, outs[i].name, sx, "logits"));
        ND_TRY(check_apart(so, outs[i].name, st, "tokens"));
        for (int j = 0; j < i; j++)
            if (outs[j].p) ND_TRY(check_apart(so, outs[i].name, span_of(outs[j].p, outs[j].n, outs[j].size), outs[j].name));
    }
    if (!any) return bad_arg("log probabilities: no result is asked for");
    ND_TRY(require_aligned(tokens, 8, "tokens"));
    LpArgs a = {};
    a.x = logits; a.rows = rows; a.row = d.stride[0]; a.col = d.shape[1] > 1 ? d.stride[1] : 1; a.vocab = (int) d.shape[1];
    a.tokens = tokens; a.scale = dtype == kF64 ? scale : (double) (float) scale;
    a.logProbs = logProbs; a.entropy = entropy; a.rowMax = rowMax; a.logSum = logSum;
    a.k = k; a.topTokens = topTokens; a.topLogProbs = topLogProbs;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kF32: return lp_forward<float, false>(a, cs);
        case kF64: return lp_forward<double, false>(a, cs);
        default: return lp_far(a) ? lp_forward<__half, true>(a, cs) : lp_forward<__half, false>(a, cs);
    }
}

Status lp_gradient_entry(void *stream, int dtype, const void *logits, const Nd4jLong *logitsShapeInfo, const Nd4jLong *tokens,
                         double scale, const void *rowMax, const void *logSum, const void *entropy, const void *gLogProbs,
                         const void *gEntropy, void *dLogits, const Nd4jLong *dLogitsShapeInfo) {
    ND_TRY(require_dtype(dtype));
    ND_TRY(lp_scale(dtype, scale));
    ShapeDesc d, o;
    ND_TRY(parse_shape(logitsShapeInfo, "logitsShapeInfo", &d));
    ND_TRY(parse_shape(dLogitsShapeInfo, "dLogitsShapeInfo", &o));
    ND_TRY(lp_shape("log probabilities gradient", d));
    if (!equal_shape(d, o)) return bad_arg("log probabilities gradient: logits and dLogits differ in shape");
    if (d.shape[0] == 0) return kOk;
    const size_t elem = size_of_dtype(dtype), wide = size_of_wide(dtype);
    ND_TRY(require(logits, "logits")); ND_TRY(require(tokens, "tokens")); ND_TRY(require(rowMax, "rowMax"));
    ND_TRY(require(logSum, "logSum")); ND_TRY(require(dLogits, "dLogits"));
    if (!gLogProbs && !gEntropy) return bad_arg("log probabilities gradient: no upstream gradient is given");
    if (gEntropy) ND_TRY(require(entropy, "entropy"));
    ND_TRY(require_aligned(logits, elem, "logits")); ND_TRY(require_aligned(dLogits, elem, "dLogits"));
    ND_TRY(require_aligned(tokens, 8, "tokens"));
    ND_TRY(check_written(o, "dLogits"));
    ND_TRY(check_alias(dLogits, o, "dLogits", logits, d, "logits", elem));
    const LL rows = d.shape[0];
    const Span so = span_of(dLogits, o, elem);
    ND_TRY(check_apart(so, "dLogits", span_of(tokens, rows, 8), "tokens"));
    const LpOut ins[] = {{rowMax, "rowMax", wide, rows}, {logSum, "logSum", wide, rows}, {gEntropy ? entropy : nullptr, "entropy", wide, rows},
                         {gLogProbs, "gLogProbs", wide, rows}, {gEntropy, "gEntropy", wide, rows}};
    for (const LpOut &in : ins) {
        if (!in.p) continue;
        ND_TRY(require_aligned(in.p, in.size, in.name));
        ND_TRY(check_apart(so, "dLogits", span_of(in.p, in.n, in.size), in.name));
    }
    LpArgs a = {};
    a.x = logits; a.rows = rows; a.row = d.stride[0]; a.col = d.shape[1] > 1 ? d.stride[1] : 1; a.vocab = (int) d.shape[1];
    a.tokens = tokens; a.scale = dtype == kF64 ? scale : (double) (float) scale;
    a.rowMax = const_cast<void *>(rowMax); a.logSum = const_cast<void *>(logSum); a.entropy = const_cast<void *>(entropy);
    a.gLogProbs = gLogProbs; a.gEntropy = gEntropy;
    a.dx = dLogits; a.dRow = o.stride[0]; a.dCol = o.shape[1] > 1 ? o.stride[1] : 1;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kF32: return lp_gradient<float, false>(a, cs);
        case kF64: return lp_gradient<double, false>(a, cs);
        default: return lp_far(a) ? lp_gradient<__half, true>(a, cs) : lp_gradient<__half, false>(a, cs);
    }
}

}  // namespace
}  // namespace nd4jb200

using namespace nd4jb200;

#pragma GCC visibility push(default)
extern "C" {

int nd4jb200_exec_token_log_probs(void *stream, int dtype, const void *logits, const Nd4jLong *logitsShapeInfo,
                                  const Nd4jLong *tokens, double scale, void *logProbs, void *entropy, void *rowMax,
                                  void *logSum, int k, Nd4jLong *topTokens, void *topLogProbs) {
    return c_entry([&] { return lp_forward_entry(stream, dtype, logits, logitsShapeInfo, tokens, scale, logProbs, entropy, rowMax,
                                                 logSum, k, topTokens, topLogProbs); });
}

int nd4jb200_exec_token_log_probs_grad(void *stream, int dtype, const void *logits, const Nd4jLong *logitsShapeInfo,
                                       const Nd4jLong *tokens, double scale, const void *rowMax, const void *logSum,
                                       const void *entropy, const void *gLogProbs, const void *gEntropy, void *dLogits,
                                       const Nd4jLong *dLogitsShapeInfo) {
    return c_entry([&] { return lp_gradient_entry(stream, dtype, logits, logitsShapeInfo, tokens, scale, rowMax, logSum, entropy,
                                                  gLogProbs, gEntropy, dLogits, dLogitsShapeInfo); });
}

}  // extern "C"
#pragma GCC visibility pop
