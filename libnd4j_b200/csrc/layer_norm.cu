// Layer norm along a dimension list and its gradients. For every TAD x of length n, with gain g and bias b of length n:
//
//   mean = sum(x) / n,  invStd = 1 / sqrt(sum((x - mean)^2) / n + epsilon),  h = (x - mean) * invStd,  z = h * g + b
//
//   d = dz * g,  dx = invStd * (d - sum(d) / n - h * sum(d * h) / n),  dg = sum over TADs of dz * h,  db = sum of dz
//
// What bounds both: HBM. Forward reads x and writes z, backward reads x and dz and writes dx; the statistics, the sums
// inside a row and the weights' gradients must not cost another sweep. So a row lives in the registers of the threads
// that read it: the variance is taken around the mean from registers (no cancellation, unlike sum(x^2) - n mean^2), and
// the backward kernel is persistent, every thread keeping the running sums of dg and db for the columns it holds,
// which become one partial row per CTA at the end and are folded by a second, small launch in a fixed order.
// All sums are held in float for float and half data and in double for double; every result is rounded once.
//
// Rows that one CTA cannot hold are split over a cluster of up to eight; longer ones still, and rows that are not of unit
// stride, take the sweeping kernels at the end of the file.
//
// Measured (device time of the main launch): forward, 16384 rows of 4096 floats, 85 us = 6.3 TB/s; backward, 65536 rows of
// 1024 floats, 127 us = 6.3 TB/s, and 7 us for the fold; 32768 rows of 4096 halves, 151 us = 5.3 TB/s.
#include "../../include/nd4j_b200.h"
#include <cooperative_groups.h>
#include "device_utils.cuh"
#include "entry_checks.h"

namespace cg = cooperative_groups;

namespace nd4jb200 {
namespace {

struct LnArgs {
    const void *x, *dz, *gain, *bias;
    void *z;                         // forward: z; backward: dx (may be null)
    void *mean, *invStd;             // written (or null) by forward, read by backward; one wide value per TAD, dense
    LL rows, cols;
    LL xRow, zRow, dzRow;            // distance of two rows (unit column stride)
    double epsilon;
    void *partials;                  // backward: [CTA][2][cols] wide values
    void *dGain, *dBias;             // may be null
    int numPartials;
    int cluster;                     // rows split over the CTAs of a cluster: their number, and the columns of each
    int splitCols;
    int statBytes;                   // backward: where the statistics of the staged rows begin in shared memory
    View xOuter, xInner, zOuter, zInner, dzOuter, dzInner;      // for the sweeping kernels
};

template <class C> ND_D C ln_warp_sum(C v) {
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// V consecutive values: a 16-byte word, a 4-byte one (two halves), or a single value.
template <class T, int V> struct LnRun {
    T v[V];
    ND_D void load(const T *p) {
        if constexpr (V == 1) v[0] = *p;
        else if constexpr (V * sizeof(T) == 4) *reinterpret_cast<unsigned *>(v) = *reinterpret_cast<const unsigned *>(p);
        else *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
    }
    ND_D void store(T *p) const {
        if constexpr (V == 1) *p = v[0];
        else if constexpr (V * sizeof(T) == 4) *reinterpret_cast<unsigned *>(p) = *reinterpret_cast<const unsigned *>(v);
        else *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(v);
    }
};
template <class T, int V> struct alignas(V * sizeof(T)) LnWord : LnRun<T, V> {};

// Sum over the CTA, the same bits in every thread.
template <class C> ND_D C ln_row_sum(C v, C *slots) {
    v = ln_warp_sum(v);
    const int warps = blockDim.x >> 5;
    __syncthreads();                                  // slots may still be read from the sum before
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    C r = slots[0];
    for (int k = 1; k < warps; k++) r += slots[k];
    return r;
}

// Two floats that one instruction adds or multiplies (add / mul / fma.rn.f32x2: each half rounds like the scalar
// instruction); a single double. Half rows are bound by the issue of instructions, which this halves.
template <class C> struct LnPack;
template <> struct LnPack<float> {
    static constexpr int W = 2;
    unsigned long long v;
    static ND_D LnPack of(float a, float b) { LnPack r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
    static ND_D LnPack all(float a) { return of(a, a); }
    ND_D float get(int k) const {
        float a, b;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
        return k ? b : a;
    }
    ND_D float sum() const { return get(0) + get(1); }
    static ND_D LnPack add(LnPack a, LnPack b) { LnPack r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
    static ND_D LnPack mul(LnPack a, LnPack b) { LnPack r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
    static ND_D LnPack fma(LnPack a, LnPack b, LnPack c) { LnPack r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
};
template <> struct LnPack<double> {
    static constexpr int W = 1;
    double v;
    static ND_D LnPack all(double a) { return LnPack{a}; }
    ND_D double get(int) const { return v; }
    ND_D double sum() const { return v; }
    static ND_D LnPack add(LnPack a, LnPack b) { return LnPack{a.v + b.v}; }
    static ND_D LnPack mul(LnPack a, LnPack b) { return LnPack{a.v * b.v}; }
    static ND_D LnPack fma(LnPack a, LnPack b, LnPack c) { return LnPack{::fma(a.v, b.v, c.v)}; }
};
// The values of a thread's NP words as packs, `beyond` where there is no word, and back.
template <class T, int V, int NP> struct LnVals {
    typedef typename Elem<T>::C C;
    typedef LnPack<C> P;
    static constexpr int N = NP * V / P::W;
    static_assert(NP * V % P::W == 0, "a thread holds whole packs");
    P p[N];
    ND_D void zero() {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = P::all(C(0));
    }
    template <class W, class G> ND_D void from(const W (&w)[NP], const G &g, C beyond = C(0)) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            C e[P::W];
#pragma unroll
            for (int k = 0; k < P::W; k++) {
                const int at = i * P::W + k;
                e[k] = g.exists(at) ? Elem<T>::to_c(w[at / V].v[at % V]) : beyond;
            }
            if constexpr (P::W == 2) p[i] = P::of(e[0], e[1]);
            else p[i] = P::all(e[0]);
        }
    }
    template <class W> ND_D void to(W (&w)[NP]) const {
#pragma unroll
        for (int at = 0; at < NP * V; at++) w[at / V].v[at % V] = Elem<T>::from_c(p[at / P::W].get(at % P::W));
    }
};

// Rows on their way into shared memory: D iterations ahead by asynchronous copies, which hold far more of them in flight
// than registers could (backward, 65536 rows of 1024 floats: 163 us with one row ahead in registers, 142 so).
//
// kLnOwn: rows of whole, aligned 16-byte words. Every thread copies the very words that it will read, so that nothing but
// its own copies has to be waited for. Otherwise the group copies the aligned words that a row lies in (and, element by
// element, what it shares with its neighbours' words), and every thread picks its columns from them behind a barrier;
// half rows in pairs of columns, which are a 4-byte word in every second row of odd length. kLnFull: as kLnOwn, with every
// word of every thread inside the row, so that no bounds are kept (forward, 16384 rows of 4096 floats: 28 instructions
// per value with them). kLn...Most: every word of a thread but its last one is, so that bounds are kept for that one.
enum LnMode { kLnPicked = 0, kLnOwn = 1, kLnFull = 2, kLnPickedMost = 3, kLnOwnMost = 4 };
ND_HD constexpr bool ln_own(int mode) { return mode == kLnOwn || mode == kLnFull || mode == kLnOwnMost; }
ND_HD constexpr bool ln_most(int mode) { return mode == kLnPickedMost || mode == kLnOwnMost; }
ND_D void ln_copy(void *to, const void *from) {
    const unsigned s = (unsigned) __cvta_generic_to_shared(to);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(from) : "memory");
}
template <class C> ND_D void ln_copy_value(C *to, const C *from) {
    const unsigned s = (unsigned) __cvta_generic_to_shared(to);
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(s), "l"(from), "n"(sizeof(C)) : "memory");
}
ND_D void ln_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> ND_D void ln_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
ND_D void ln_group_barrier(int group, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory"); }

// Bytes that one staged row may take: its words, one more for the shift, kept to whole words.
inline ND_HD int ln_staged(LL cols, int elem) { return (int) ((cols * elem + 15) / 16 * 16 + 16); }

// A CTA's groups of G threads, each holding one row at a time: thread t the words t, t + G, ... (NP at most) of V values.
// The row's last word may be cut short: `live` counts the thread's values that exist, the first ones of its words.
template <class T, int V, int NP, int NA, int MODE> struct LnGroup {
    static constexpr bool OWN = ln_own(MODE), FULL = MODE == kLnFull;
    static constexpr int SURE = FULL ? NP : (ln_most(MODE) ? NP - 1 : 0);      // words that every thread has whole
    unsigned char *smem;
    int G, groups, group, t, have, live, staged;
    LL cols;
    ND_D LnGroup(unsigned char *m, int g, LL c) : smem(m), G(g), cols(c) {
        groups = blockDim.x / G;
        group = threadIdx.x / G;
        t = threadIdx.x - group * G;
        const int words = (int) ((cols + V - 1) / V);
        have = t < words ? (words - 1 - t) / G + 1 : 0;
        live = have * V;
        if (have > 0 && word(have - 1) == words - 1) live -= words * V - (int) cols;
        staged = OWN ? 0 : ln_staged(cols, sizeof(T));
    }
    ND_D bool holds(int j) const { return j < SURE || j < have; }
    ND_D bool exists(int at) const { return at < SURE * V || at < live; }
    ND_D int word(int j) const { return t + G * j; }
    ND_D int column(int at) const { return word(at / V) * V + at % V; }
    // where stage d keeps word j of array q for this thread, or (not OWN) array q of this group
    ND_D LnWord<T, V> *own(int d, int q, int j) const {
        return reinterpret_cast<LnWord<T, V> *>(smem) + ((d * NA + q) * NP + j) * blockDim.x + threadIdx.x;
    }
    ND_D unsigned char *shared(int d, int q) const { return smem + ((d * NA + q) * groups + group) * staged; }
    static ND_D int shift(const T *row) { return (int) (reinterpret_cast<unsigned long long>(row) & 15); }
    ND_D void fetch(int d, int q, const T *row) const {
        if constexpr (OWN) {
#pragma unroll
            for (int j = 0; j < NP; j++) if (holds(j)) ln_copy(own(d, q, j), row + word(j) * V);
        } else {
            const int off = shift(row), end = off + (int) cols * (int) sizeof(T), last = end / 16 * 16;
            const char *from = reinterpret_cast<const char *>(row) - off;
            unsigned char *to = shared(d, q);
            for (int w = (off + 15) / 16 * 16 + t * 16; w < last; w += G * 16) ln_copy(to + w, from + w);
            const int e = t * (int) sizeof(T);                // element of the first and of the last word
            if (e < 16) {
                if (e >= off && off > 0 && e < end) *reinterpret_cast<T *>(to + e) = *reinterpret_cast<const T *>(from + e);
                if (last + e < end && last + e >= off) *reinterpret_cast<T *>(to + last + e) = *reinterpret_cast<const T *>(from + last + e);
            }
        }
    }
    ND_D void read(int d, int q, const T *row, LnWord<T, V> (&w)[NP]) const {
        if constexpr (OWN) {
#pragma unroll
            for (int j = 0; j < NP; j++) if (holds(j)) w[j] = *own(d, q, j);
        } else {
            const T *s = reinterpret_cast<const T *>(shared(d, q) + shift(row));
            pick(s, w);
        }
    }
    // The thread's values of a row at p, which need not be aligned to words (values behind the last are read as well when
    // `p` is a staged row: its buffer reaches a word further).
    ND_D void pick(const T *p, LnWord<T, V> (&w)[NP]) const {
        if (V == 1 || (reinterpret_cast<unsigned long long>(p) & (sizeof(T) * V - 1)) == 0) {
#pragma unroll
            for (int j = 0; j < NP; j++) if (holds(j)) w[j].load(p + word(j) * V);
        } else {
#pragma unroll
            for (int j = 0; j < NP; j++)
#pragma unroll
                for (int k = 0; k < V; k++) if (holds(j)) w[j].v[k] = p[word(j) * V + k];
        }
    }
    // The thread's values of a vector in global memory.
    ND_D void load(const T *p, LnWord<T, V> (&w)[NP]) const {
#pragma unroll
        for (int at = 0; at < NP * V; at++) if (exists(at)) w[at / V].v[at % V] = p[column(at)];
    }
    ND_D void store(T *p, const LnWord<T, V> (&w)[NP]) const {
        if (OWN || V == 1) {
#pragma unroll
            for (int j = 0; j < NP; j++) if (holds(j)) w[j].store(p + word(j) * V);
        } else if ((reinterpret_cast<unsigned long long>(p) & (sizeof(T) * V - 1)) == 0) {
#pragma unroll
            for (int j = 0; j < NP; j++) {
                if (exists(j * V + V - 1)) w[j].store(p + word(j) * V);
                else if (exists(j * V)) p[word(j) * V] = w[j].v[0];
            }
        } else {
#pragma unroll
            for (int at = 0; at < NP * V; at++) if (exists(at)) p[column(at)] = w[at / V].v[at % V];
        }
    }
};

// Sum over the group's warps; `slots` holds one value per warp of the CTA and must not be in use.
template <int MAXW, class S, class ADD> ND_D S ln_group_sum(S v, S *slots, int group, int G, ADD add) {
    const int warps = G >> 5, warp = threadIdx.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) slots[warp] = v;
    ln_group_barrier(group, G);
    const S *mine = slots + group * warps;
    S r = mine[0];
#pragma unroll
    for (int k = 1; k < MAXW; k++) if (k < warps) r = add(r, mine[k]);
    return r;
}

// Rows that one CTA cannot hold are split over the CTAs of a cluster, which join their sums through distributed shared
// memory; without a split this CTA has the row to itself. `unit` counts clusters (or CTAs).
template <bool SPLIT> struct LnPart {
    int rank, unit, units, cols;
    LL first;                        // column
    ND_D LnPart(const LnArgs &a) : rank(0), unit(blockIdx.x), units(gridDim.x), cols((int) a.cols), first(0) {
        if constexpr (SPLIT) {
            rank = (int) cg::this_cluster().block_rank();
            unit = blockIdx.x / a.cluster;
            units = gridDim.x / a.cluster;
            first = (LL) rank * a.splitCols;
            cols = a.cols - first < a.splitCols ? (int) (a.cols - first) : a.splitCols;
        }
    }
    // Sum over the cluster, in the order of the CTAs. `joint` is written again only after another join in between.
    template <class S, class ADD> ND_D S join(const LnArgs &a, S v, S *joint, ADD add) const {
        if constexpr (SPLIT) {
            cg::cluster_group cl = cg::this_cluster();
            if (threadIdx.x == 0) *joint = v;
            cl.sync();
            v = *cl.map_shared_rank(joint, 0);
            for (int q = 1; q < a.cluster; q++) v = add(v, *cl.map_shared_rank(joint, q));
        }
        return v;
    }
    ND_D void leave() const { if constexpr (SPLIT) cg::this_cluster().sync(); }      // nobody reads this CTA's memory any more
};

// Forward: two sums per row, the second around the mean. The slots alternate over four sets, so that a set is written
// again only two barriers after it was read.
template <class T, int V, int NP, int D, int MAXT, int CTAS, int MODE, bool SPLIT>
__global__ void __launch_bounds__(MAXT, CTAS) k_ln_forward(const LnArgs a, const int G) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    typedef LnPack<C> P;
    typedef LnVals<T, V, NP> Vals;
    extern __shared__ __align__(16) unsigned char ln_smem[];
    __shared__ C slots[4][MAXT / 32];
    constexpr bool OWN = ln_own(MODE);
    __shared__ C joint[4];
    const LnPart<SPLIT> part(a);
    const LnGroup<T, V, NP, 1, MODE> g(ln_smem, G, part.cols);
    const T *px = static_cast<const T *>(a.x) + part.first;
    T *pz = static_cast<T *>(a.z) + part.first;
    const C invN = C(1) / (C) a.cols;
    Vals gain, bias;
    LnWord<T, V> w[NP];
    if (a.gain) { g.load(static_cast<const T *>(a.gain) + part.first, w); gain.from(w, g); }
    if (a.bias) { g.load(static_cast<const T *>(a.bias) + part.first, w); bias.from(w, g); }
#pragma unroll
    for (int i = 0; i < Vals::N; i++) {
        if (!a.gain) gain.p[i] = P::all(C(1));
        if (!a.bias) bias.p[i] = P::all(C(0));
    }
    const LL step = (LL) part.units * g.groups;
    LL r = (LL) part.unit * g.groups + g.group;
#pragma unroll
    for (int d = 0; d < D; d++) { if (r + d * step < a.rows) g.fetch(d, 0, px + (r + d * step) * a.xRow); ln_commit(); }
    int stage = 0;
    auto plus = [](C x, C y) { return x + y; };
    for (int parity = 0; r < a.rows; r += step, parity ^= 2) {
        ln_wait<D - 1>();
        if (!OWN) ln_group_barrier(g.group, G);                // everyone's copies of this row stand
        g.read(stage, 0, px + r * a.xRow, w);
        Vals v;
        v.from(w, g);
        P s = v.p[0];
#pragma unroll
        for (int i = 1; i < Vals::N; i++) s = P::add(s, v.p[i]);
        C sum = ln_group_sum<MAXT / 32>(ln_warp_sum(s.sum()), slots[parity], g.group, G, plus);
        sum = part.join(a, sum, joint + parity, plus);
        if (!OWN && (G >> 5) == 1) __syncwarp();
        // the stage has been read (OWN: by this thread, which alone uses these words; otherwise by all: the barrier)
        if (r + D * step < a.rows) g.fetch(stage, 0, px + (r + D * step) * a.xRow);
        ln_commit();
        const C mean = sum * invN;
        const P away = P::all(-mean);
        s = P::all(C(0));
#pragma unroll
        for (int i = 0; i < Vals::N; i++) {
            v.p[i] = P::add(v.p[i], away);
            const bool whole = g.exists(i * P::W + P::W - 1), some = g.exists(i * P::W);
            if (whole) s = P::fma(v.p[i], v.p[i], s);
            else if (some) { if constexpr (P::W == 2) { const P one = P::of(v.p[i].get(0), C(0)); s = P::fma(one, one, s); } }
        }
        sum = ln_group_sum<MAXT / 32>(ln_warp_sum(s.sum()), slots[parity + 1], g.group, G, plus);
        sum = part.join(a, sum, joint + parity + 1, plus);
        const C inv = C(1) / sqrt(sum * invN + (C) a.epsilon);
        if (g.t == 0 && part.rank == 0) {
            if (a.mean) static_cast<C *>(a.mean)[r] = mean;
            if (a.invStd) static_cast<C *>(a.invStd)[r] = inv;
        }
        const P scale = P::all(inv);
#pragma unroll
        for (int i = 0; i < Vals::N; i++) v.p[i] = P::fma(P::mul(v.p[i], scale), gain.p[i], bias.p[i]);
        v.to(w);
        g.store(pz + r * a.zRow, w);
        stage = stage + 1 == D ? 0 : stage + 1;
    }
    ln_wait<0>();
    part.leave();
}

template <class C> struct LnPair { C a, b; };

// Backward: each thread holds the same columns of every row it meets, and therefore their sums of dg and db; a group
// waits once per row, on a barrier of its own.
template <class T, int V, int NP, int D, int MAXT, int CTAS, int MODE, bool SPLIT>
__global__ void __launch_bounds__(MAXT, CTAS) k_ln_backward(const LnArgs a, const int G) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    typedef LnPack<C> P;
    typedef LnVals<T, V, NP> Vals;
    extern __shared__ __align__(16) unsigned char ln_smem[];
    __shared__ LnPair<C> slots[2][MAXT / 32];
    constexpr bool OWN = ln_own(MODE);
    __shared__ LnPair<C> joint[2];
    const LnPart<SPLIT> part(a);
    const LnGroup<T, V, NP, 2, MODE> g(ln_smem, G, part.cols);
    const T *px = static_cast<const T *>(a.x) + part.first, *pdz = static_cast<const T *>(a.dz) + part.first;
    T *pdx = a.z ? static_cast<T *>(a.z) + part.first : nullptr;
    const C *pMean = static_cast<const C *>(a.mean), *pInv = static_cast<const C *>(a.invStd);
    const C invN = C(1) / (C) a.cols;
    Vals gain, sg, sb;
    LnWord<T, V> w[NP];
    if (a.gain) { g.load(static_cast<const T *>(a.gain) + part.first, w); gain.from(w, g); }
    else {
#pragma unroll
        for (int i = 0; i < Vals::N; i++) gain.p[i] = P::all(C(1));
    }
    sg.zero();
    sb.zero();
    const LL step = (LL) part.units * g.groups;
    LL r = (LL) part.unit * g.groups + g.group;
    // Half: mean and invStd travel with their row, a copy for every warp, made by its first two lanes; loaded one row ahead
    // into registers, they were what these shorter rows waited for (32768 rows of 4096 halves: 212 us, 153 so). Float and
    // double rows last long enough for the load, and are better off without the two warp barriers (65536 rows of 1024
    // floats: 141 us, 149 with them).
    constexpr bool STAGED = sizeof(T) == 2;
    const int lane = threadIdx.x & 31;
    C *stats = reinterpret_cast<C *>(ln_smem + a.statBytes) + (threadIdx.x >> 5) * 2;
    auto stat = [&](int d) { return stats + d * (blockDim.x >> 5) * 2; };
    auto fetch = [&](int d, LL row) {
        if (row < a.rows) {
            g.fetch(d, 0, px + row * a.xRow);
            g.fetch(d, 1, pdz + row * a.dzRow);
            if (STAGED && lane < 2) ln_copy_value(stat(d) + lane, (lane == 0 ? pMean : pInv) + row);
        }
        ln_commit();
    };
#pragma unroll
    for (int d = 0; d < D; d++) fetch(d, r + d * step);
    C mean = C(0), inv = C(0), nextMean = C(0), nextInv = C(0);
    if (!STAGED && r < a.rows) { nextMean = pMean[r]; nextInv = pInv[r]; }
    int stage = 0;
    auto plus = [](const LnPair<C> &x, const LnPair<C> &y) { return LnPair<C>{x.a + y.a, x.b + y.b}; };
    for (int parity = 0; r < a.rows; r += step, parity ^= 1) {
        if (!STAGED) {
            mean = nextMean; inv = nextInv;
            if (r + step < a.rows) { nextMean = pMean[r + step]; nextInv = pInv[r + step]; }
        }
        ln_wait<D - 1>();
        if (STAGED) { __syncwarp(); mean = stat(stage)[0]; inv = stat(stage)[1]; }
        if (!OWN) ln_group_barrier(g.group, G);                // everyone's copies of this row stand
        Vals h, d;
        g.read(stage, 0, px + r * a.xRow, w);
        h.from(w, g, mean);                               // beyond the row: h = 0, dz = 0
        g.read(stage, 1, pdz + r * a.dzRow, w);
        d.from(w, g);
        const P away = P::all(-mean), scale = P::all(inv);
        P pa = P::all(C(0)), pb = pa;
#pragma unroll
        for (int i = 0; i < Vals::N; i++) {
            h.p[i] = P::mul(P::add(h.p[i], away), scale);
            sg.p[i] = P::fma(d.p[i], h.p[i], sg.p[i]);
            sb.p[i] = P::add(sb.p[i], d.p[i]);
            d.p[i] = P::mul(d.p[i], gain.p[i]);
            pa = P::add(pa, d.p[i]);
            pb = P::fma(d.p[i], h.p[i], pb);
        }
        if (STAGED) __syncwarp();                              // the warp has read its statistics
        if (OWN) fetch(stage, r + D * step);                   // and this thread these words
        LnPair<C> s = {ln_warp_sum(pa.sum()), ln_warp_sum(pb.sum())};
        s = ln_group_sum<MAXT / 32>(s, slots[parity], g.group, G, plus);
        s = part.join(a, s, joint + parity, plus);
        if (!OWN) { if ((G >> 5) == 1) __syncwarp(); fetch(stage, r + D * step); }         // nobody reads this stage any more
        if (pdx) {
            const P ma = P::all(-s.a * invN), mb = P::all(-s.b * invN);
#pragma unroll
            for (int i = 0; i < Vals::N; i++) d.p[i] = P::mul(P::fma(h.p[i], mb, P::add(d.p[i], ma)), scale);
            d.to(w);
            g.store(pdx + r * a.zRow, w);
        }
        stage = stage + 1 == D ? 0 : stage + 1;
    }
    ln_wait<0>();
    part.leave();
    if (!a.dGain && !a.dBias) return;
    // the CTA's groups add up in shared memory, one after the other, then the CTA's sums become a partial row
    C *pg = static_cast<C *>(a.partials) + (LL) part.unit * 2 * a.cols + part.first, *pb = pg + a.cols;
    C *tg = reinterpret_cast<C *>(ln_smem), *tb = tg + part.cols;
    __syncthreads();                                           // the stages have been read by all groups
    for (int q = 0; q < g.groups; q++) {
        if (q == g.group) {
#pragma unroll
            for (int at = 0; at < NP * V; at++) {
                if (g.exists(at)) {
                    const int c = g.column(at);
                    C vg = sg.p[at / P::W].get(at % P::W), vb = sb.p[at / P::W].get(at % P::W);
                    if (q > 0) { vg += tg[c]; vb += tb[c]; }
                    if (q + 1 < g.groups) { tg[c] = vg; tb[c] = vb; }
                    else if (part.units > 1) { pg[c] = vg; pb[c] = vb; }
                    else {                                     // the only partial row is the result
                        if (a.dGain) static_cast<T *>(a.dGain)[part.first + c] = Elem<T>::from_c(vg);
                        if (a.dBias) static_cast<T *>(a.dBias)[part.first + c] = Elem<T>::from_c(vb);
                    }
                }
            }
        }
        if (g.groups > 1) __syncthreads();
    }
}

// Folds the partial rows: a CTA takes 32 columns, its 32 warps share out the partials.
template <class T>
__global__ void __launch_bounds__(1024) k_ln_fold(const LnArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    __shared__ C tg[32][33], tb[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const LL c = (LL) blockIdx.x * 32 + lane;
    const C *p = static_cast<const C *>(a.partials);
    C g = C(0), b = C(0);
    if (c < a.cols) {
        int q = warp;
        for (; q + 96 < a.numPartials; q += 128) {              // eight loads in flight
            C vg[4], vb[4];
#pragma unroll
            for (int u = 0; u < 4; u++) { vg[u] = p[(LL) (q + 32 * u) * 2 * a.cols + c]; vb[u] = p[((LL) (q + 32 * u) * 2 + 1) * a.cols + c]; }
#pragma unroll
            for (int u = 0; u < 4; u++) { g += vg[u]; b += vb[u]; }
        }
        for (; q < a.numPartials; q += 32) { g += p[(LL) q * 2 * a.cols + c]; b += p[((LL) q * 2 + 1) * a.cols + c]; }
    }
    tg[warp][lane] = g; tb[warp][lane] = b;
    __syncthreads();
    // thread (warp, lane) now sums column `warp`'s 32 values across lanes
    g = ln_warp_sum(tg[lane][warp]);
    b = ln_warp_sum(tb[lane][warp]);
    const LL out = (LL) blockIdx.x * 32 + warp;
    if (lane == 0 && out < a.cols) {
        if (a.dGain) static_cast<T *>(a.dGain)[out] = Elem<T>::from_c(g);
        if (a.dBias) static_cast<T *>(a.dBias)[out] = Elem<T>::from_c(b);
    }
}

// ---- any strides, any length: a CTA per row that sweeps it -------------------------------------------------------
constexpr int kLnSweepThreads = 512;

template <class T>
__global__ void __launch_bounds__(kLnSweepThreads) k_ln_forward_sweep(const LnArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    __shared__ C slots[32];
    const C n = (C) a.cols;
    const T *gain = static_cast<const T *>(a.gain), *bias = static_cast<const T *>(a.bias);
    for (LL r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + view_offset(a.xOuter, r);
        T *z = static_cast<T *>(a.z) + view_offset(a.zOuter, r);
        C s = C(0);
        for (LL c = threadIdx.x; c < a.cols; c += kLnSweepThreads) s += Elem<T>::load(x + view_offset(a.xInner, c));
        const C mean = ln_row_sum(s, slots) / n;
        s = C(0);
        for (LL c = threadIdx.x; c < a.cols; c += kLnSweepThreads) {
            const C v = Elem<T>::load(x + view_offset(a.xInner, c)) - mean;
            s = fma(v, v, s);
        }
        const C inv = C(1) / sqrt(ln_row_sum(s, slots) / n + (C) a.epsilon);
        if (threadIdx.x == 0) {
            if (a.mean) static_cast<C *>(a.mean)[r] = mean;
            if (a.invStd) static_cast<C *>(a.invStd)[r] = inv;
        }
        for (LL c = threadIdx.x; c < a.cols; c += kLnSweepThreads) {
            const C h = (Elem<T>::load(x + view_offset(a.xInner, c)) - mean) * inv;
            const C g = gain ? Elem<T>::load(gain + c) : C(1), b = bias ? Elem<T>::load(bias + c) : C(0);
            Elem<T>::store(z + view_offset(a.zInner, c), fma(h, g, b));
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kLnSweepThreads) k_ln_backward_sweep(const LnArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    __shared__ C slots[32];
    const C n = (C) a.cols;
    const T *gain = static_cast<const T *>(a.gain);
    for (LL r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + view_offset(a.xOuter, r);
        const T *dz = static_cast<const T *>(a.dz) + view_offset(a.dzOuter, r);
        T *dx = static_cast<T *>(a.z) + view_offset(a.zOuter, r);
        const C mean = static_cast<const C *>(a.mean)[r], inv = static_cast<const C *>(a.invStd)[r];
        C sa = C(0), sb = C(0);
        for (LL c = threadIdx.x; c < a.cols; c += kLnSweepThreads) {
            const C h = (Elem<T>::load(x + view_offset(a.xInner, c)) - mean) * inv;
            const C d = Elem<T>::load(dz + view_offset(a.dzInner, c)) * (gain ? Elem<T>::load(gain + c) : C(1));
            sa += d;
            sb = fma(d, h, sb);
        }
        sa = ln_row_sum(sa, slots) / n;
        sb = ln_row_sum(sb, slots) / n;
        for (LL c = threadIdx.x; c < a.cols; c += kLnSweepThreads) {
            const C h = (Elem<T>::load(x + view_offset(a.xInner, c)) - mean) * inv;
            const C d = Elem<T>::load(dz + view_offset(a.dzInner, c)) * (gain ? Elem<T>::load(gain + c) : C(1));
            Elem<T>::store(dx + view_offset(a.zInner, c), inv * (d - sa - h * sb));
        }
    }
}

// Partial sums of dg and db: a CTA takes 32 columns and every gridDim.y-th block of 16 rows.
template <class T>
__global__ void __launch_bounds__(512) k_ln_weights_sweep(const LnArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    __shared__ C tg[16][33], tb[16][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (LL block = blockIdx.x; block * 32 < a.cols; block += gridDim.x) {
        const LL c = block * 32 + lane;
        C g = C(0), b = C(0);
        if (c < a.cols) {
            const LL xo = view_offset(a.xInner, c), dzo = view_offset(a.dzInner, c);
            for (LL r = (LL) blockIdx.y * 16 + warp; r < a.rows; r += (LL) gridDim.y * 16) {
                const C mean = static_cast<const C *>(a.mean)[r], inv = static_cast<const C *>(a.invStd)[r];
                const C h = (Elem<T>::load(static_cast<const T *>(a.x) + view_offset(a.xOuter, r) + xo) - mean) * inv;
                const C dz = Elem<T>::load(static_cast<const T *>(a.dz) + view_offset(a.dzOuter, r) + dzo);
                g = fma(dz, h, g);
                b += dz;
            }
        }
        __syncthreads();
        tg[warp][lane] = g; tb[warp][lane] = b;
        __syncthreads();
        if (warp == 0 && c < a.cols) {
            for (int q = 1; q < 16; q++) { g += tg[q][lane]; b += tb[q][lane]; }
            C *p = static_cast<C *>(a.partials) + (LL) blockIdx.y * 2 * a.cols;
            p[c] = g;
            p[a.cols + c] = b;
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------
// How rows are held: so many values per thread while up to 256 threads hold the row (a CTA then takes as many rows as fit
// and shares its SM with others), a CTA of up to 512 threads beyond, with twice the values once that is too few. More
// values per thread spread the work that every row costs a thread; the registers set the limit. Forward: 16 (double: 8).
// Backward: 8 floats, but 16 halves, whose bytes are fewer for the same instructions (65536 rows of 1024 halves: 124 us
// with 8 values, 87 with 16), 4 doubles.
template <class T> struct LnFit {
    static constexpr int kForward = sizeof(T) == 8 ? 8 : 16;
    static constexpr int kForwardStages = sizeof(T) == 2 ? 6 : 4;       // 144 .. 192 KB of rows per SM
    static constexpr int kBackward = sizeof(T) == 8 ? 4 : (sizeof(T) == 4 ? 8 : 16);
    static constexpr int kBackwardCtas = sizeof(T) == 2 ? 2 : 3;
    static constexpr int kBackwardStages = sizeof(T) == 2 ? 5 : (sizeof(T) == 4 ? 4 : 3);
    static constexpr bool kBackwardTwice = sizeof(T) > 2;               // 32 halves and their sums do not fit
    static constexpr int kBackwardMost = kBackwardTwice ? 2 * kBackward : kBackward;
    static constexpr int kPick = sizeof(T) == 2 ? 2 : 1;                // values per word of rows that are no whole words
};
inline int threads_for(LL cols, int perThread, int most) {
    LL t = ceil_div(ceil_div(cols, perThread), 32) * 32;
    return t > most ? 0 : (int) t;
}
inline unsigned grid_for(LL n) { return (unsigned) (n < 0x7fffffffLL ? (n > 0 ? n : 1) : 0x7fffffffLL); }

template <class K> inline void launch_with_smem(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t st, const LnArgs &a, int G) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned) a.cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = g_tuning[kTuneOverlapLaunch] ? attr : attr + 1;
    cfg.numAttrs = (g_tuning[kTuneOverlapLaunch] ? 1 : 0) + (a.cluster > 1 ? 1 : 0);
    cudaLaunchKernelEx(&cfg, kernel, a, G);
    count_launch();
}

// Cluster and columns per CTA of rows that are longer than `most`; 1 for the others, 0 for those that 8 CTAs cannot hold.
inline int ln_split(LnArgs &a, LL most) {
    a.cluster = 1;
    a.splitCols = 0;
    if (a.cols <= most) return 1;
    while (a.cluster < 8 && a.cluster * most < a.cols) a.cluster *= 2;
    a.splitCols = (int) (ceil_div(ceil_div(a.cols, a.cluster), 8) * 8);        // whole words of every type
    return a.cluster * most < a.cols ? 0 : a.cluster;
}

template <class T, int V, int NP, int D, int MAXT, int CTAS, int MODE, bool SPLIT = false>
Status ln_forward_rows(const LnArgs &a, int G, int block, cudaStream_t st) {
    const int groups = block / G;
    const LL cols = SPLIT ? a.splitCols : a.cols;
    const size_t smem = ln_own(MODE) ? (size_t) D * NP * V * sizeof(T) * block : (size_t) D * groups * ln_staged(cols, sizeof(T));
    auto kernel = k_ln_forward<T, V, NP, D, MAXT, CTAS, MODE, SPLIT>;
    static std::atomic<unsigned long long> asked{0};
    ND_TRY(allow_shared(reinterpret_cast<const void *>(kernel), smem, asked));
    LL units = (LL) kNumSMs * CTAS / a.cluster;
    if (units > ceil_div(a.rows, groups)) units = ceil_div(a.rows, groups);
    launch_with_smem(kernel, dim3((unsigned) (units * a.cluster)), dim3((unsigned) block), smem, st, a, G);
    ND_CUDA(cudaGetLastError());
    return kOk;
}

template <class T, int V, int NP, int D, int MAXT, int CTAS, int MODE>
Status ln_forward_held(const LnArgs &a, int G, int block, cudaStream_t st) {
    if (MODE == kLnOwn && a.cols == (LL) G * NP * V) return ln_forward_rows<T, V, NP, D, MAXT, CTAS, MODE == kLnOwn ? kLnFull : MODE>(a, G, block, st);
    if (NP > 1 && a.cols / V >= (LL) G * (NP - 1))
        return ln_forward_rows<T, V, NP, D, MAXT, CTAS, NP == 1 ? MODE : (MODE == kLnOwn ? kLnOwnMost : kLnPickedMost)>(a, G, block, st);
    return ln_forward_rows<T, V, NP, D, MAXT, CTAS, MODE>(a, G, block, st);
}

template <class T, int V, int MODE> Status ln_forward_fit(const LnArgs &a, cudaStream_t st) {
    constexpr int S = LnFit<T>::kForward, D = LnFit<T>::kForwardStages;
    // rows that a warp holds with a quarter of the values (half: with one word): most of its instructions would be idle
    constexpr int Q = S / 4 > Elem<T>::kVec ? S / 4 : Elem<T>::kVec;
    if (a.cols <= 32 * Q) return ln_forward_held<T, V, Q / V, D, 256, 4, MODE>(a, 32, 256, st);
    if (int G = threads_for(a.cols, S, 256)) return ln_forward_held<T, V, S / V, D, 256, 3, MODE>(a, G, 256 / G * G, st);
    if (int G = threads_for(a.cols, S, 512)) return ln_forward_held<T, V, S / V, D, 512, 1, MODE>(a, G, G, st);
    if (int G = threads_for(a.cols, 2 * S, 512)) return ln_forward_held<T, V, 2 * S / V, 3, 512, 1, MODE>(a, G, G, st);
    const int G = threads_for(a.splitCols, 2 * S, 512);
    return ln_forward_rows<T, V, 2 * S / V, 3, 512, 1, MODE, true>(a, G, G, st);
}

template <class T> Status ln_forward(LnArgs &a, bool rows, bool words, cudaStream_t st) {
    if (rows && ln_split(a, 2 * LnFit<T>::kForward * 512))
        return words ? ln_forward_fit<T, Elem<T>::kVec, kLnOwn>(a, st) : ln_forward_fit<T, LnFit<T>::kPick, kLnPicked>(a, st);
    launch_kernel(k_ln_forward_sweep<T>, dim3(grid_for(a.rows)), dim3(kLnSweepThreads), st, a);
    ND_CUDA(cudaGetLastError());
    return kOk;
}

// Launches the kernel for rows of unit stride: `block` threads in groups of G, D stages of rows in shared memory.
template <class T, int V, int NP, int D, int MAXT, int CTAS, int MODE, bool SPLIT = false>
Status ln_backward_rows(LnArgs &a, int G, int block, cudaStream_t st) {
    typedef typename Elem<T>::C C;
    const int groups = block / G;
    const LL cols = SPLIT ? a.splitCols : a.cols;
    const size_t stages = ln_own(MODE) ? (size_t) D * 2 * NP * V * sizeof(T) * block : (size_t) D * 2 * groups * ln_staged(cols, sizeof(T));
    const size_t fold = groups > 1 ? 2 * (size_t) cols * sizeof(C) : 0;
    const size_t rowsAndStats = stages + (size_t) D * 2 * (block / 32) * sizeof(C);
    const size_t smem = rowsAndStats > fold ? rowsAndStats : fold;
    a.statBytes = (int) stages;
    auto kernel = k_ln_backward<T, V, NP, D, MAXT, CTAS, MODE, SPLIT>;
    static std::atomic<unsigned long long> asked{0};
    ND_TRY(allow_shared(reinterpret_cast<const void *>(kernel), smem, asked));
    LL units = (LL) kNumSMs * CTAS / a.cluster;
    if (units > ceil_div(a.rows, groups)) units = ceil_div(a.rows, groups);
    a.numPartials = (int) units;
    Scratch scratch(st);
    const bool weights = (a.dGain || a.dBias) && units > 1;
    if (weights) {
        ND_TRY(scratch.alloc((size_t) units * 2 * (size_t) a.cols * sizeof(C)));
        a.partials = scratch.at<void>(0);
    }
    launch_with_smem(kernel, dim3((unsigned) (units * a.cluster)), dim3((unsigned) block), smem, st, a, G);
    if (weights) launch_kernel(k_ln_fold<T>, dim3((unsigned) ceil_div(a.cols, 32)), dim3(1024), st, a);
    ND_CUDA(cudaGetLastError());
    return kOk;
}

template <class T, int V, int NP, int D, int MAXT, int CTAS, int MODE>
Status ln_backward_held(LnArgs &a, int G, int block, cudaStream_t st) {
    if (MODE == kLnOwn && a.cols == (LL) G * NP * V) return ln_backward_rows<T, V, NP, D, MAXT, CTAS, MODE == kLnOwn ? kLnFull : MODE>(a, G, block, st);
    if (NP > 1 && a.cols / V >= (LL) G * (NP - 1))
        return ln_backward_rows<T, V, NP, D, MAXT, CTAS, NP == 1 ? MODE : (MODE == kLnOwn ? kLnOwnMost : kLnPickedMost)>(a, G, block, st);
    return ln_backward_rows<T, V, NP, D, MAXT, CTAS, MODE>(a, G, block, st);
}

template <class T, int V, int MODE> Status ln_backward_fit(LnArgs &a, cudaStream_t st) {
    typedef LnFit<T> F;
    constexpr int S = F::kBackward;
    if (int G = threads_for(a.cols, S, 256)) return ln_backward_held<T, V, S / V, F::kBackwardStages, 256, F::kBackwardCtas, MODE>(a, G, 256 / G * G, st);
    if (int G = threads_for(a.cols, S, 512)) return ln_backward_held<T, V, S / V, F::kBackwardStages, 512, 1, MODE>(a, G, G, st);
    constexpr int M = F::kBackwardMost, D = M > S ? 3 : F::kBackwardStages;
    if constexpr (M > S) {
        if (int G = threads_for(a.cols, M, 512)) return ln_backward_held<T, V, M / V, D, 512, 1, MODE>(a, G, G, st);
    }
    const int G = threads_for(a.splitCols, M, 512);
    return ln_backward_rows<T, V, M / V, D, 512, 1, MODE, true>(a, G, G, st);
}

template <class T> Status ln_backward(LnArgs &a, bool rows, bool words, cudaStream_t st) {
    typedef typename Elem<T>::C C;
    if (rows && a.rows > 0 && ln_split(a, LnFit<T>::kBackwardMost * 512))
        return words ? ln_backward_fit<T, Elem<T>::kVec, kLnOwn>(a, st) : ln_backward_fit<T, LnFit<T>::kPick, kLnPicked>(a, st);
    Scratch scratch(st);
    if (a.dGain || a.dBias) {
        // before dx is written, which may take the place of x or dz
        const LL blocks = ceil_div(a.cols, 32);
        LL split = ceil_div((LL) kNumSMs * 4, blocks);
        if (split > ceil_div(a.rows, 16)) split = ceil_div(a.rows, 16);
        a.numPartials = (int) split;
        if (split > 0) {
            ND_TRY(scratch.alloc((size_t) split * 2 * (size_t) a.cols * sizeof(C)));
            a.partials = scratch.at<void>(0);
            launch_kernel(k_ln_weights_sweep<T>, dim3(grid_for(blocks), (unsigned) split), dim3(512), st, a);
        }
        launch_kernel(k_ln_fold<T>, dim3(grid_for(blocks)), dim3(1024), st, a);
    }
    if (a.z && a.rows > 0) launch_kernel(k_ln_backward_sweep<T>, dim3(grid_for(a.rows)), dim3(kLnSweepThreads), st, a);
    ND_CUDA(cudaGetLastError());
    return kOk;
}

struct LnShape { ShapeDesc d; TadPlan plan; };

Status ln_plan(const Nd4jLong *info, const char *name, const int *dimension, int dimensionLength, LnShape *s) {
    ND_TRY(parse_shape(info, name, &s->d));
    if (s->d.length == 0) return kOk;
    ND_TRY(make_tad_plan(s->d, dimension, dimensionLength, &s->plan));
    if (s->plan.whole) ND_TRY(coord_view(s->d, &s->plan.inner));      // columns are counted in c-order of the axes
    return kOk;
}

// Length of a TAD of an array without elements.
Status ln_empty_tad(const ShapeDesc &d, const int *dimension, int dimensionLength, LL *tadLen) {
    *tadLen = 1;
    bool seen[kMaxRank] = {false};
    for (int i = 0; i < dimensionLength; i++) {
        const int ax = dimension[i] < 0 ? dimension[i] + d.rank : dimension[i];
        if (ax < 0 || ax >= d.rank) return bad_arg("a dimension is not an axis of x");
        if (!seen[ax]) *tadLen *= d.shape[ax];
        seen[ax] = true;
    }
    return kOk;
}

bool ln_unit_rows(const TadPlan &p) { return (p.inner.rank == 0 || (p.inner.rank == 1 && p.inner.stride[0] == 1)) && p.outer.rank <= 1; }
LL ln_row_step(const TadPlan &p) { return p.outer.rank == 1 ? p.outer.stride[0] : 0; }
bool ln_words(const void *p, const TadPlan &plan, LL V) { return aligned16(p) && ln_row_step(plan) % V == 0; }

Status ln_vector(const void *p, const char *name, LL cols, size_t elem, Span *s) {
    *s = span_of(p, p ? cols : 0, elem);
    if (p) ND_TRY(require_aligned(p, elem, name));
    return kOk;
}

Status ln_forward_entry(void *stream, int dtype, const void *x, const Nd4jLong *xShapeInfo, const void *gain, const void *bias,
                        double epsilon, void *z, const Nd4jLong *zShapeInfo, void *mean, void *invStd, const int *dimension,
                        int dimensionLength) {
    ND_TRY(require_dtype(dtype));
    ND_TRY(require(dimension, "dimension"));
    if (dimensionLength < 1) return bad_arg("layer norm: the dimension list is empty");
    const size_t elem = size_of_dtype(dtype), wide = size_of_wide(dtype);
    const double eps = dtype == kF64 ? epsilon : (double) (float) epsilon;
    if (!(eps > 0 && std::isfinite(eps))) return bad_arg("layer norm: epsilon must be positive and finite");
    LnShape xs, zs;
    ND_TRY(ln_plan(xShapeInfo, "xShapeInfo", dimension, dimensionLength, &xs));
    ND_TRY(ln_plan(zShapeInfo, "zShapeInfo", dimension, dimensionLength, &zs));
    if (!equal_shape(xs.d, zs.d)) return bad_arg("layer norm: x and z differ in shape");
    if (xs.d.length == 0) return kOk;
    ND_TRY(require(x, "x")); ND_TRY(require(z, "z"));
    ND_TRY(require_aligned(x, elem, "x")); ND_TRY(require_aligned(z, elem, "z"));
    ND_TRY(check_written(zs.d, "z"));
    ND_TRY(check_alias(z, zs.d, "z", x, xs.d, "x", elem));
    const LL rows = xs.plan.numTads, cols = xs.plan.tadLen;
    Span sg, sb, sm, si;
    ND_TRY(ln_vector(gain, "gain", cols, elem, &sg));
    ND_TRY(ln_vector(bias, "bias", cols, elem, &sb));
    ND_TRY(ln_vector(mean, "mean", rows, wide, &sm));
    ND_TRY(ln_vector(invStd, "invStd", rows, wide, &si));
    const Span sx = span_of(x, xs.d, elem), sz = span_of(z, zs.d, elem);
    ND_TRY(check_apart(sz, "z", sg, "gain")); ND_TRY(check_apart(sz, "z", sb, "bias"));
    for (const Span &s : {sx, sz, sg, sb}) { ND_TRY(check_apart(sm, "mean", s, "another array")); ND_TRY(check_apart(si, "invStd", s, "another array")); }
    ND_TRY(check_apart(sm, "mean", si, "invStd"));
    LnArgs a = {};
    a.x = x; a.gain = gain; a.bias = bias; a.z = z; a.mean = mean; a.invStd = invStd;
    a.rows = rows; a.cols = cols; a.epsilon = eps;
    a.xRow = ln_row_step(xs.plan); a.zRow = ln_row_step(zs.plan);
    a.xOuter = xs.plan.outer; a.xInner = xs.plan.inner; a.zOuter = zs.plan.outer; a.zInner = zs.plan.inner;
    const bool unit = ln_unit_rows(xs.plan) && ln_unit_rows(zs.plan);
    const LL V = 16 / (LL) elem;
    const bool words = unit && cols % V == 0 && ln_words(x, xs.plan, V) && ln_words(z, zs.plan, V) &&
                       aligned16(gain) && aligned16(bias);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kF32: return ln_forward<float>(a, unit, words, st);
        case kF64: return ln_forward<double>(a, unit, words, st);
        default: return ln_forward<__half>(a, unit, words, st);
    }
}

Status ln_backward_entry(void *stream, int dtype, const void *x, const Nd4jLong *xShapeInfo, const void *gain, const void *mean,
                         const void *invStd, const void *dz, const Nd4jLong *dzShapeInfo, void *dx, const Nd4jLong *dxShapeInfo,
                         void *dGain, void *dBias, const int *dimension, int dimensionLength) {
    ND_TRY(require_dtype(dtype));
    ND_TRY(require(dimension, "dimension"));
    if (dimensionLength < 1) return bad_arg("layer norm gradient: the dimension list is empty");
    const size_t elem = size_of_dtype(dtype), wide = size_of_wide(dtype);
    LnShape xs, ds, os;
    ND_TRY(ln_plan(xShapeInfo, "xShapeInfo", dimension, dimensionLength, &xs));
    ND_TRY(ln_plan(dzShapeInfo, "dzShapeInfo", dimension, dimensionLength, &ds));
    if (!equal_shape(xs.d, ds.d)) return bad_arg("layer norm gradient: x and dz differ in shape");
    if (dx) {
        ND_TRY(ln_plan(dxShapeInfo, "dxShapeInfo", dimension, dimensionLength, &os));
        if (!equal_shape(xs.d, os.d)) return bad_arg("layer norm gradient: x and dx differ in shape");
        ND_TRY(check_written(os.d, "dx"));
    }
    LL rows = 0, cols = 0;
    if (xs.d.length > 0) {
        rows = xs.plan.numTads; cols = xs.plan.tadLen;
        ND_TRY(require(x, "x")); ND_TRY(require(dz, "dz")); ND_TRY(require(mean, "mean")); ND_TRY(require(invStd, "invStd"));
    } else ND_TRY(ln_empty_tad(xs.d, dimension, dimensionLength, &cols));
    if (cols == 0 || (!dx && !dGain && !dBias)) return kOk;
    LnArgs a = {};
    a.x = x; a.dz = dz; a.gain = gain; a.mean = const_cast<void *>(mean); a.invStd = const_cast<void *>(invStd);
    a.z = rows > 0 ? dx : nullptr; a.dGain = dGain; a.dBias = dBias; a.rows = rows; a.cols = cols;
    bool unit = false, words = false;
    Span sg, sm, si, sdg, sdb;
    ND_TRY(ln_vector(gain, "gain", cols, elem, &sg));
    ND_TRY(ln_vector(mean, "mean", rows, wide, &sm));
    ND_TRY(ln_vector(invStd, "invStd", rows, wide, &si));
    ND_TRY(ln_vector(dGain, "dGain", cols, elem, &sdg));
    ND_TRY(ln_vector(dBias, "dBias", cols, elem, &sdb));
    ND_TRY(check_apart(sdg, "dGain", sdb, "dBias"));
    for (const Span &s : {sg, sm, si}) { ND_TRY(check_apart(sdg, "dGain", s, "an operand")); ND_TRY(check_apart(sdb, "dBias", s, "an operand")); }
    if (rows > 0) {
        ND_TRY(require_aligned(x, elem, "x")); ND_TRY(require_aligned(dz, elem, "dz"));
        const Span sx = span_of(x, xs.d, elem), sdz = span_of(dz, ds.d, elem);
        for (const Span &s : {sx, sdz}) { ND_TRY(check_apart(sdg, "dGain", s, "an operand")); ND_TRY(check_apart(sdb, "dBias", s, "an operand")); }
        const LL V = 16 / (LL) elem;
        a.xOuter = xs.plan.outer; a.xInner = xs.plan.inner; a.dzOuter = ds.plan.outer; a.dzInner = ds.plan.inner;
        a.xRow = ln_row_step(xs.plan); a.dzRow = ln_row_step(ds.plan);
        unit = ln_unit_rows(xs.plan) && ln_unit_rows(ds.plan);
        words = cols % V == 0 && ln_words(x, xs.plan, V) && ln_words(dz, ds.plan, V) && aligned16(gain);
        if (dx) {
            ND_TRY(require_aligned(dx, elem, "dx"));
            ND_TRY(check_alias(dx, os.d, "dx", x, xs.d, "x", elem));
            ND_TRY(check_alias(dx, os.d, "dx", dz, ds.d, "dz", elem));
            const Span sdx = span_of(dx, os.d, elem);
            for (const Span &s : {sg, sm, si, sdg, sdb}) ND_TRY(check_apart(sdx, "dx", s, "another array"));
            a.zOuter = os.plan.outer; a.zInner = os.plan.inner; a.zRow = ln_row_step(os.plan);
            unit = unit && ln_unit_rows(os.plan);
            words = words && ln_words(dx, os.plan, V);
        }
        words = words && unit;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kF32: return ln_backward<float>(a, unit, words, st);
        case kF64: return ln_backward<double>(a, unit, words, st);
        default: return ln_backward<__half>(a, unit, words, st);
    }
}

}  // namespace
}  // namespace nd4jb200

using namespace nd4jb200;

#pragma GCC visibility push(default)
extern "C" {

int nd4jb200_exec_layer_norm(void *stream, int dtype, const void *x, const Nd4jLong *xShapeInfo, const void *gain,
                             const void *bias, double epsilon, void *z, const Nd4jLong *zShapeInfo, void *mean, void *invStd,
                             const int *dimension, int dimensionLength) {
    return c_entry([&] { return ln_forward_entry(stream, dtype, x, xShapeInfo, gain, bias, epsilon, z, zShapeInfo, mean, invStd,
                                                 dimension, dimensionLength); });
}

int nd4jb200_exec_layer_norm_grad(void *stream, int dtype, const void *x, const Nd4jLong *xShapeInfo, const void *gain,
                                  const void *mean, const void *invStd, const void *dz, const Nd4jLong *dzShapeInfo, void *dx,
                                  const Nd4jLong *dxShapeInfo, void *dGain, void *dBias, const int *dimension,
                                  int dimensionLength) {
    return c_entry([&] { return ln_backward_entry(stream, dtype, x, xShapeInfo, gain, mean, invStd, dz, dzShapeInfo, dx,
                                                  dxShapeInfo, dGain, dBias, dimension, dimensionLength); });
}

}  // extern "C"
#pragma GCC visibility pop
