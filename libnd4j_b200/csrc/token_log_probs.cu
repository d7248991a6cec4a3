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
// is written. Sums are held in float for float and half data, in double for double.
//
// Exponentials are powers of two (one special-function instruction), so c carries the factor log2(e). Half data: the
// distance from the reference point is one fused multiply-add, x c - R; R is the rounded m c, and since every term is
// relative to the same R its rounding cancels exactly. Float data subtracts first: a value of the type's lowest, the
// usual mask, would overflow when multiplied. Masked entries (-inf) contribute nothing, a row of nothing else has log
// probability -inf, entropy 0 and gradient 0; a row with a NaN or +inf answers NaN.
//
// Few rows: the CTAs of a cluster of up to 8 share a row and join their sums through distributed shared memory, so that
// eight rows of a large vocabulary still keep 64 SMs reading.
//
// Best alternatives need no second sweep: each thread already knows the largest value of its slice and, with a batch
// number kept beside it, where it stands. The k-th best of these is a lower bound for the k-th best of all; only the
// slices of the k threads at or above it are read again (k / 512 of the row, mostly from L2), what reaches the bound is
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

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpBatch = 4;                 // 128-bit words a thread has in flight
constexpr int kLpMaxTop = 64;
constexpr int kLpList = 1024;               // collected candidates, at most
constexpr int kLpNone = 0x7fffffff;

// Exponent arithmetic of one element type. A reference point stands for a maximum; dist() is an element's exponent
// relative to it, gap() that of another reference point.
template <class T> struct LpMath;
template <> struct LpMath<__half> {
    typedef float C;
    static constexpr float kFloor = -65504.f;       // reference of a row without values: the lowest finite one
    static constexpr double kUnit = 1.4426950408889634;          // log2(e): exponents are of base two
    static ND_D float ref(float m, float c) { return fmaxf(m, kFloor) * c; }
    static ND_D float dist(float x, float r, float c) { return fmaf(x, c, -r); }
    static ND_D float gap(float a, float b, float) { return a - b; }
    static ND_D float off(float m, float r, float c) { return fmaf(-m, c, r); }         // exponent of the reference over the maximum's
};
template <> struct LpMath<float> {
    typedef float C;
    static constexpr float kFloor = -FLT_MAX;
    static constexpr double kUnit = 1.4426950408889634;
    static ND_D float ref(float m, float) { return fmaxf(m, kFloor); }
    static ND_D float dist(float x, float r, float c) { return (x - r) * c; }
    static ND_D float gap(float a, float b, float c) { return (a - b) * c; }
    static ND_D float off(float, float, float) { return 0.f; }
};
template <> struct LpMath<double> {
    typedef double C;
    static constexpr double kFloor = -DBL_MAX;
    static constexpr double kUnit = 1.0;
    static ND_D double ref(double m, double) { return fmax(m, kFloor); }
    static ND_D double dist(double x, double r, double c) { return (x - r) * c; }
    static ND_D double gap(double a, double b, double c) { return (a - b) * c; }
    static ND_D double off(double, double, double) { return 0.0; }
};
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
    // Element f of the slice of thread `slot` in a row shared by `span` threads: (index, value) handed to `f`, ascending.
    template <class F> ND_D void each(int slot, int span, int firstWord, int wordStep, F f) const {
        if (V > 1 && firstWord == 0 && slot < head) f(slot, Elem<T>::to_c(at(slot)));
        for (int w = slot + firstWord * span; w < words; w += wordStep * span) {
            alignas(16) T v[V];
            load(w, v);
#pragma unroll
            for (int k = 0; k < V; k++) f(index(w) + k, Elem<T>::to_c(v[k]));
        }
        if (V > 1 && firstWord == 0 && slot < tail) f(index(words) + slot, Elem<T>::to_c(at(index(words) + slot)));
    }
};

template <class C> struct LpSum { C ref, s, u; };

template <class T, bool ENT> ND_D LpSum<typename LpMath<T>::C> lp_join(const LpSum<typename LpMath<T>::C> &a,
                                                                       const LpSum<typename LpMath<T>::C> &b, typename LpMath<T>::C c) {
    typedef LpMath<T> M;
    typedef typename M::C C;
    LpSum<C> r;
    r.ref = a.ref > b.ref ? a.ref : b.ref;
    const C ga = M::gap(a.ref, r.ref, c), gb = M::gap(b.ref, r.ref, c);
    const C fa = lp_exp(ga), fb = lp_exp(gb);
    r.s = a.s * fa + b.s * fb;
    r.u = C(0);
    // a reference far below leaves a power of 0: its sum must not meet an infinite gap
    if (ENT) r.u = (fa == C(0) ? C(0) : fa * (a.u + lp_finite(ga) * a.s)) + (fb == C(0) ? C(0) : fb * (b.u + lp_finite(gb) * b.s));
    return r;
}

// Order of candidates: larger first, then the lower index; a NaN before all values.
template <class C> ND_D bool lp_better(C v, int i, C w, int j) {
    const bool nv = v != v, nw = w != w;
    if (nv || nw) return nv && nw ? i < j : nv;
    return v > w || (v == w && i < j);
}
template <class C> ND_D void lp_warp_best(C &v, int &i) {
    for (int m = 16; m > 0; m >>= 1) {
        const C w = __shfl_xor_sync(0xffffffffu, v, m);
        const int j = __shfl_xor_sync(0xffffffffu, i, m);
        if (j != kLpNone && (i == kLpNone || lp_better(w, j, v, i))) { v = w; i = j; }
    }
}

template <class C> struct LpShared {
    LpSum<C> sums[kLpWarps];
    LpSum<C> ctaSum;                         // read by the other CTAs of a cluster
    C warpV[kLpWarps]; int warpI[kLpWarps];
    C listV[kLpList]; int listI[kLpList];    // candidates
    C bestV[kLpMaxTop]; int bestI[kLpMaxTop];   // this CTA's best, in order (read by the leading CTA of a cluster)
    int slots[kLpMaxTop];
    int count, best, numSlots;
};

// The k best of the CTA's part of a row into s.bestV / bestI, their number into s.best. (v, i): the thread's own best
// (i = kLpNone: nothing above -inf). `odd`: the row holds a NaN or +inf.
template <class T, int V>
ND_D void lp_select(const LpRow<T, V> &row, typename LpMath<T>::C v, int i, bool odd, int k, int rank, int span, LpShared<typename LpMath<T>::C> &s) {
    typedef typename LpMath<T>::C C;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slot = rank * kLpThreads + threadIdx.x;
    if (threadIdx.x == 0) s.count = s.best = s.numSlots = 0;
    __syncthreads();
    bool slow = odd;
    if (!odd) {
        // a first bound: of every warp the r-th best, of these the least; at least r * kLpWarps >= k threads reach it
        const int rounds = (k + kLpWarps - 1) / kLpWarps;
        C bv = v; int bi = i;
        bool out = false;
        for (int q = 0; q < rounds; q++) {
            bv = v; bi = out ? kLpNone : i;
            lp_warp_best(bv, bi);
            if (bi == i) out = true;
        }
        if (lane == 0) { s.warpV[warp] = bv; s.warpI[warp] = bi; }
        __syncthreads();
        bool all = false;                      // some warp has fewer: every thread with a value counts
        bv = s.warpV[0]; bi = s.warpI[0];
        for (int w = 0; w < kLpWarps; w++) {
            if (s.warpI[w] == kLpNone) all = true;
            else if (lp_better(bv, bi, s.warpV[w], s.warpI[w])) { bv = s.warpV[w]; bi = s.warpI[w]; }
        }
        const bool source = i != kLpNone && (all || !lp_better(bv, bi, v, i));
        int at = 0;
        if (source) { at = atomicAdd(&s.count, 1); s.listV[at] = v; s.listI[at] = i; }
        __syncthreads();
        // the k-th best of them exactly
        const int n0 = s.count;
        int place = 0;
        if (source) {
            for (int q = 0; q < n0; q++) if (lp_better(s.listV[q], s.listI[q], v, i)) place++;
            if (place < k) s.slots[place] = threadIdx.x;
            if (place == k - 1) { s.warpV[0] = v; s.warpI[0] = i; }
        }
        __syncthreads();
        const int numSlots = n0 < k ? n0 : k;
        const bool bounded = n0 >= k;
        const C tv = s.warpV[0]; const int ti = s.warpI[0];
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        // what reaches it, from the slices of those threads; a slice is read by a warp
        for (int q = warp; q < numSlots; q += kLpWarps) {
            const int owner = rank * kLpThreads + s.slots[q];
            row.each(owner, span, lane, 32, [&](int j, C w) {
                if (w > -C(INFINITY) && (!bounded || !lp_better(tv, ti, w, j))) {
                    const int p = atomicAdd(&s.count, 1);
                    if (p < kLpList) { s.listV[p] = w; s.listI[p] = j; }
                }
            });
        }
        __syncthreads();
        const int n = s.count;
        slow = n > kLpList;
        if (!slow) {
            for (int q = threadIdx.x; q < n; q += kLpThreads) {
                const C w = s.listV[q]; const int j = s.listI[q];
                int before = 0;
                for (int o = 0; o < n && before < k; o++) if (lp_better(s.listV[o], s.listI[o], w, j)) before++;
                if (before < k) { s.bestV[before] = w; s.bestI[before] = j; }
            }
            if (threadIdx.x == 0) s.best = n < k ? n : k;
        }
        __syncthreads();
    }
    if (!slow) return;
    // one by one: the best of the threads' bests is taken, its owner looks for its next
    C popV = C(0); int popI = kLpNone;
    C bv = C(0); int bi = kLpNone;
    auto look = [&]() {
        bi = kLpNone;
        row.each(slot, span, 0, 1, [&](int j, C w) {
            const bool real = w > -C(INFINITY) || w != w;
            if (real && (popI == kLpNone || lp_better(popV, popI, w, j)) && (bi == kLpNone || lp_better(w, j, bv, bi))) { bv = w; bi = j; }
        });
    };
    look();
    int taken = 0;
    for (; taken < k; taken++) {
        C wv = bv; int wi = bi;
        lp_warp_best(wv, wi);
        if (lane == 0) { s.warpV[warp] = wv; s.warpI[warp] = wi; }
        __syncthreads();
        wv = s.warpV[0]; wi = s.warpI[0];
        for (int w = 1; w < kLpWarps; w++)
            if (s.warpI[w] != kLpNone && (wi == kLpNone || lp_better(s.warpV[w], s.warpI[w], wv, wi))) { wv = s.warpV[w]; wi = s.warpI[w]; }
        __syncthreads();
        if (wi == kLpNone) break;
        if (threadIdx.x == 0) { s.bestV[taken] = wv; s.bestI[taken] = wi; }
        popV = wv; popI = wi;
        if (bi == wi) look();
    }
    if (threadIdx.x == 0) s.best = taken;
    __syncthreads();
}

template <class T, int V, bool ENT, bool TOP>
__global__ void __launch_bounds__(kLpThreads) k_token_log_probs(const LpArgs a) {
    grid_dependency_sync();
    typedef LpMath<T> M;
    typedef typename M::C C;
    __shared__ LpShared<C> s;
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = a.cluster, rank = ctas > 1 ? (int) cl.block_rank() : 0;
    const int span = ctas * kLpThreads, slot = rank * kLpThreads + threadIdx.x;
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
                if (TOP && threadIdx.x < a.k) {
                    a.topTokens[r * a.k + threadIdx.x] = -1;
                    static_cast<C *>(a.topLogProbs)[r * a.k + threadIdx.x] = C(0);
                }
            }
            continue;
        }
        const LpRow<T, V> row(a, r);
        C top = -C(INFINITY);
        int batch = kLpNone;                                    // where `top` was met: a word, or -1 head, -2 tail
        LpSum<C> sum = {M::ref(top, c), C(0), C(0)};
        auto meet = [&](C bm, int where) {
            if (bm > top) {
                const C ref = M::ref(bm, c);
                const LpSum<C> moved = {ref, C(0), C(0)};
                if (ref > sum.ref) sum = lp_join<T, ENT>(sum, moved, c);
                top = bm;
                batch = where;
            }
        };
        auto add = [&](C x) {
            const C d = M::dist(x, sum.ref, c), e = lp_exp(d);
            sum.s += e;
            if (ENT) sum.u = fma(e, lp_finite(d), sum.u);
        };
        if (V > 1 && slot < row.head) { const C x = Elem<T>::to_c(row.at(slot)); meet(x, -1); add(x); }
        for (int w = slot; w < row.words; w += kLpBatch * span) {
            alignas(16) T v[kLpBatch][V];
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
            C bm = -C(INFINITY);
#pragma unroll
            for (int j = 0; j < kLpBatch; j++)
#pragma unroll
                for (int k = 0; k < V; k++) { const C x = Elem<T>::to_c(v[j][k]); bm = x > bm ? x : bm; }
            meet(bm, w);
#pragma unroll
            for (int j = 0; j < kLpBatch; j++)
#pragma unroll
                for (int k = 0; k < V; k++) add(Elem<T>::to_c(v[j][k]));
        }
        if (V > 1 && slot < row.tail) { const C x = Elem<T>::to_c(row.at(row.index(row.words) + slot)); meet(x, -2); add(x); }

        // over the warp, the CTA, the cluster: every thread ends with the row's sums and maximum
        LpSum<C> all = sum;
        C m = top;
        for (int o = 16; o > 0; o >>= 1) {
            LpSum<C> b;
            b.ref = __shfl_xor_sync(0xffffffffu, all.ref, o);
            b.s = __shfl_xor_sync(0xffffffffu, all.s, o);
            if (ENT) b.u = __shfl_xor_sync(0xffffffffu, all.u, o);
            // the lower lane's state on the left, so that both sides round alike
            all = (lane & o) == 0 ? lp_join<T, ENT>(all, b, c) : lp_join<T, ENT>(b, all, c);
            const C mo = __shfl_xor_sync(0xffffffffu, m, o);
            m = mo > m ? mo : m;
        }
        __syncthreads();                                        // the shared block may still serve the row before
        if (lane == 0) { s.sums[warp] = all; s.warpV[warp] = m; }
        __syncthreads();
        all = s.sums[0];
        m = s.warpV[0];
        for (int w = 1; w < kLpWarps; w++) { all = lp_join<T, ENT>(all, s.sums[w], c); m = s.warpV[w] > m ? s.warpV[w] : m; }
        if (ctas > 1) {
            if (threadIdx.x == 0) { s.ctaSum = all; s.bestV[0] = m; }
            cl.sync();
            for (int q = 0; q < ctas; q++) {
                const LpShared<C> *o = cl.map_shared_rank(&s, q);
                const LpSum<C> b = o->ctaSum;
                const C mo = o->bestV[0];
                all = q == 0 ? b : lp_join<T, ENT>(all, b, c);
                m = mo > m ? mo : m;
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
                for (int j = kLpBatch - 1; j >= 0; j--) {
                    if (batch + j * span < row.words) {
                        alignas(16) T v[V];
                        row.load(batch + j * span, v);
#pragma unroll
                        for (int k = V - 1; k >= 0; k--) if (Elem<T>::to_c(v[k]) == top) mine = row.index(batch + j * span) + k;
                    }
                }
            }
            lp_select<T, V>(row, top, mine, odd, a.k, rank, span, s);
            if (ctas > 1) {
                cl.sync();
                if (rank == 0) {
                    // the CTAs' lists, at most 8 * 64 entries, ranked once more
                    __shared__ int counts[8];
                    if (threadIdx.x < ctas) counts[threadIdx.x] = cl.map_shared_rank(&s, threadIdx.x)->best;
                    __syncthreads();
                    const int q = threadIdx.x / kLpMaxTop, e = threadIdx.x - q * kLpMaxTop;
                    int first = 0, n = 0;
                    for (int o = 0; o < ctas; o++) { if (o < q) first += counts[o]; n += counts[o]; }
                    const bool have = q < ctas && e < counts[q];
                    if (have) {
                        const LpShared<C> *o = cl.map_shared_rank(&s, q);
                        s.listV[first + e] = o->bestV[e];
                        s.listI[first + e] = o->bestI[e];
                    }
                    __syncthreads();
                    int before = 0;
                    C w = C(0); int j = 0;
                    if (have) {
                        w = s.listV[first + e]; j = s.listI[first + e];
                        for (int o = 0; o < n; o++) if (lp_better(s.listV[o], s.listI[o], w, j)) before++;
                    }
                    __syncthreads();
                    if (have && before < a.k) { s.bestV[before] = w; s.bestI[before] = j; }
                    if (threadIdx.x == 0) s.best = n < a.k ? n : a.k;
                    __syncthreads();
                }
            }
            if (rank == 0) {
                const int n = s.best;
                for (int q = threadIdx.x; q < n; q += kLpThreads) {
                    a.topTokens[r * a.k + q] = s.bestI[q];
                    static_cast<C *>(a.topLogProbs)[r * a.k + q] = odd ? nan : log_p(s.bestV[q]);
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
constexpr int kLpGradThreads = 256;
constexpr int kLpGradWords = 4;              // words in flight per thread, all a CTA does

template <class T, int V, bool ENT>
__global__ void __launch_bounds__(kLpGradThreads) k_token_log_probs_grad(const LpArgs a) {
    grid_dependency_sync();
    typedef LpMath<T> M;
    typedef typename M::C C;
    const C c = (C) (a.scale * M::kUnit), unit = (C) M::kUnit, back = (C) (1.0 / M::kUnit);
    const LL units = a.rows * a.chunks;
    for (LL b = blockIdx.x; b < units; b += gridDim.x) {
        const LL r = b / a.chunks;
        const int chunk = (int) (b - r * a.chunks);
        const LpRow<T, V> row(a, r);
        T *dx = static_cast<T *>(a.dx) + r * a.dRow;
        const LL token = a.tokens[r];
        const C m = static_cast<const C *>(a.rowMax)[r], logSum = static_cast<const C *>(a.logSum)[r];
        const C g = (C) a.scale * (a.gLogProbs ? static_cast<const C *>(a.gLogProbs)[r] : C(0));
        const C h = ENT ? (C) a.scale * static_cast<const C *>(a.gEntropy)[r] : C(0);
        const bool none = token < 0 || m == -C(INFINITY);         // padding, or a row without a value: zeros
        const C ref = M::ref(m, c), shift = logSum * unit - M::off(m, ref, c);
        C A = ENT ? -(g + h * static_cast<const C *>(a.entropy)[r]) : -g;
        const C B = ENT ? -h * back : C(0);
        if (token >= a.vocab || m != m) A = (C) NAN;
        auto one = [&](C x) -> C {
            const C lp = M::dist(x, ref, c) - shift, p = lp_exp(lp);
            return ENT ? p * fma(B, lp_finite(lp), A) : p * A;
        };
        const int first = chunk * (kLpGradThreads * kLpGradWords) + threadIdx.x;
        alignas(16) T v[kLpGradWords][V];
        if (!none) {
#pragma unroll
            for (int j = 0; j < kLpGradWords; j++)
                if (first + j * kLpGradThreads < row.words) row.load(first + j * kLpGradThreads, v[j]);
        }
        const bool aligned = V > 1 && (reinterpret_cast<unsigned long long>(dx + row.head) & 15) == 0;
#pragma unroll
        for (int j = 0; j < kLpGradWords; j++) {
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
template <class K> void launch_log_probs(K kernel, const LpArgs &a, unsigned grid, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(kLpThreads); cfg.stream = st;
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

template <class T, int V> void lp_forward_kernels(const LpArgs &a, unsigned grid, cudaStream_t st) {
    if (a.k > 0) {
        if (a.entropy) launch_log_probs(k_token_log_probs<T, V, true, true>, a, grid, st);
        else launch_log_probs(k_token_log_probs<T, V, false, true>, a, grid, st);
    } else {
        if (a.entropy) launch_log_probs(k_token_log_probs<T, V, true, false>, a, grid, st);
        else launch_log_probs(k_token_log_probs<T, V, false, false>, a, grid, st);
    }
}

template <class T> Status lp_forward(LpArgs &a, cudaStream_t st) {
    constexpr int V = Elem<T>::kVec;
    // Rows that would leave SMs idle are shared by a cluster, as long as every CTA keeps at least two batches.
    a.cluster = 1;
    const LL perCta = (LL) kLpThreads * kLpBatch * (a.col == 1 ? V : 1) * 2;
    while (a.cluster < 8 && a.rows * a.cluster * 2 <= kNumSMs * 2 && a.vocab >= a.cluster * 2 * perCta) a.cluster *= 2;
    LL grid = a.rows * a.cluster;
    if (grid > 0x7fffffff / 8 * 8) grid = 0x7fffffff / 8 * 8;
    if (a.col == 1) lp_forward_kernels<T, V>(a, (unsigned) grid, st);
    else lp_forward_kernels<T, 1>(a, (unsigned) grid, st);
    ND_CUDA(cudaGetLastError());
    return kOk;
}

template <class T> Status lp_gradient(LpArgs &a, cudaStream_t st) {
    constexpr int V = Elem<T>::kVec;
    const bool unit = a.col == 1 && a.dCol == 1;
    a.chunks = (int) ceil_div(ceil_div(a.vocab, unit ? V : 1), (LL) kLpGradThreads * kLpGradWords);
    const LL units = a.rows * a.chunks;
    const dim3 grid((unsigned) (units < 0x7fffffffLL ? units : 0x7fffffffLL));
    const dim3 block(kLpGradThreads);
    if (unit) {
        if (a.gEntropy) launch_kernel(k_token_log_probs_grad<T, V, true>, grid, block, st, a);
        else launch_kernel(k_token_log_probs_grad<T, V, false>, grid, block, st, a);
    } else {
        if (a.gEntropy) launch_kernel(k_token_log_probs_grad<T, 1, true>, grid, block, st, a);
        else launch_kernel(k_token_log_probs_grad<T, 1, false>, grid, block, st, a);
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
    // the exponent of the largest half, and of any difference that matters, has to stay a finite float
    const double s = dtype == kF64 ? scale : (double) (float) scale;
    if (!(s > 0 && std::isfinite(s) && s <= 1e30)) return bad_arg("log probabilities: scale must be positive and at most 1e30");
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
        case kF32: return lp_forward<float>(a, cs);
        case kF64: return lp_forward<double>(a, cs);
        default: return lp_forward<__half>(a, cs);
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
        case kF32: return lp_gradient<float>(a, cs);
        case kF64: return lp_gradient<double>(a, cs);
        default: return lp_gradient<__half>(a, cs);
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
