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
// Rows that do not fit (long, or not of unit stride) take the sweeping kernels at the end of the file.
#include "../../include/nd4j_b200.h"
#include "device_utils.cuh"
#include "entry_checks.h"

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
    View xOuter, xInner, zOuter, zInner, dzOuter, dzInner;      // for the sweeping kernels
};

template <class C> ND_D C ln_warp_sum(C v) {
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// V consecutive values, as one 128-bit word or one by one.
template <class T, int V> struct LnRun {
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
template <class T, int V> struct alignas(V == 1 ? sizeof(T) : 16) LnWord : LnRun<T, V> {};

// Sum over the CTA (or the warp, when a row belongs to one warp), the same bits in every thread.
template <bool WARP, class C> ND_D C ln_row_sum(C v, C *slots) {
    v = ln_warp_sum(v);
    if (WARP) return v;
    const int warps = blockDim.x >> 5;
    __syncthreads();                                  // slots may still be read from the sum before
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    C r = slots[0];
    for (int k = 1; k < warps; k++) r += slots[k];
    return r;
}

// A row in the registers of a warp (WARP) or of the whole CTA: NP words of V values per thread, thread t holding words
// t, t + G, ...
template <class T, int V, int NP, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) k_ln_forward(const LnArgs a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    __shared__ C slots[32];
    const int G = WARP ? 32 : blockDim.x;
    const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const LL first = WARP ? (LL) blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const LL step = WARP ? (LL) gridDim.x * (blockDim.x >> 5) : gridDim.x;
    const int words = (int) (a.cols / V);
    const C n = (C) a.cols;
    const T *gain = static_cast<const T *>(a.gain), *bias = static_cast<const T *>(a.bias);
    for (LL r = first; r < a.rows; r += step) {
        const T *x = static_cast<const T *>(a.x) + r * a.xRow;
        T *z = static_cast<T *>(a.z) + r * a.zRow;
        LnWord<T, V> w[NP];
        C sum = C(0);
#pragma unroll
        for (int j = 0; j < NP; j++) if (t + G * j < words) w[j].load(x + (LL) (t + G * j) * V);
        C v[NP][V];
#pragma unroll
        for (int j = 0; j < NP; j++) {
            const bool in = t + G * j < words;
#pragma unroll
            for (int k = 0; k < V; k++) { v[j][k] = in ? Elem<T>::to_c(w[j].v[k]) : C(0); sum += v[j][k]; }
        }
        const C mean = ln_row_sum<WARP>(sum, slots) / n;
        C sq = C(0);
#pragma unroll
        for (int j = 0; j < NP; j++) {
            if (t + G * j < words) {
#pragma unroll
                for (int k = 0; k < V; k++) { v[j][k] -= mean; sq = fma(v[j][k], v[j][k], sq); }
            }
        }
        const C inv = C(1) / sqrt(ln_row_sum<WARP>(sq, slots) / n + (C) a.epsilon);
        if (t == 0) {
            if (a.mean) static_cast<C *>(a.mean)[r] = mean;
            if (a.invStd) static_cast<C *>(a.invStd)[r] = inv;
        }
#pragma unroll
        for (int j = 0; j < NP; j++) {
            const int c = (t + G * j) * V;
            if (t + G * j < words) {
                LnWord<T, V> g, b, o;
                if (gain) g.load(gain + c);
                if (bias) b.load(bias + c);
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const C h = v[j][k] * inv;
                    o.v[k] = Elem<T>::from_c(fma(h, gain ? Elem<T>::to_c(g.v[k]) : C(1), bias ? Elem<T>::to_c(b.v[k]) : C(0)));
                }
                o.store(z + c);
            }
        }
    }
}

template <class C> struct LnPair { C a, b; };

// Backward over rows held by groups of G threads (several groups per CTA when rows are short). Each thread holds the
// same columns of every row it meets, and therefore their sums of dg and db; a group waits once per row, on a barrier of
// its own. Rows are fetched D iterations ahead by asynchronous copies into shared memory, which holds far more of them
// in flight than registers could (65536 rows of 1024 floats: 163 us with one row ahead in registers).
//
// OWN: every thread copies the very words that it will read, so that nothing but its own copies has to be waited for;
// needs words of 4, 8 or 16 bytes. Otherwise (half rows of odd length or offset) the group copies the aligned 16-byte
// words that a row lies in and every thread picks its columns from them behind a barrier.
template <int BYTES> ND_D void ln_copy(void *to, const void *from) {
    const unsigned s = (unsigned) __cvta_generic_to_shared(to);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(s), "l"(from), "n"(BYTES) : "memory");
}
ND_D void ln_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> ND_D void ln_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
ND_D void ln_group_barrier(int group, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory"); }

// Bytes that one staged row may take: its words, one more for the shift, kept to whole words.
inline ND_HD int ln_staged(LL cols, int elem) { return (int) ((cols * elem + 15) / 16 * 16 + 16); }

template <class T, int V, int NP, int D, int MAXT, int CTAS, bool OWN>
__global__ void __launch_bounds__(MAXT, CTAS) k_ln_backward(const LnArgs a, const int G) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    extern __shared__ __align__(16) unsigned char ln_smem[];
    __shared__ LnPair<C> slots[2][MAXT / 32];
    const int groups = blockDim.x / G, group = threadIdx.x / G, t = threadIdx.x - group * G;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, firstWarp = group * (G >> 5), warps = G >> 5;
    const int words = (int) (a.cols / V);
    const C invN = C(1) / (C) a.cols;
    const T *px = static_cast<const T *>(a.x), *pdz = static_cast<const T *>(a.dz);
    T *pdx = static_cast<T *>(a.z);
    const C *pMean = static_cast<const C *>(a.mean), *pInv = static_cast<const C *>(a.invStd);
    C gain[NP][V], sg[NP][V], sb[NP][V];
#pragma unroll
    for (int j = 0; j < NP; j++) {
        LnWord<T, V> g;
        const bool in = t + G * j < words;
        if (in && a.gain) g.load(static_cast<const T *>(a.gain) + (t + G * j) * V);
#pragma unroll
        for (int k = 0; k < V; k++) {
            gain[j][k] = in ? (a.gain ? Elem<T>::to_c(g.v[k]) : C(1)) : C(0);
            sg[j][k] = sb[j][k] = C(0);
        }
    }
    const LL step = (LL) gridDim.x * groups;
    const int staged = OWN ? 0 : ln_staged(a.cols, sizeof(T));

    // where stage d keeps word j of array q for this thread, or (not OWN) array q of this group
    auto own = [&](int d, int q, int j) { return reinterpret_cast<LnWord<T, V> *>(ln_smem) + ((d * 2 + q) * NP + j) * blockDim.x + threadIdx.x; };
    auto shared = [&](int d, int q) { return ln_smem + ((d * 2 + q) * groups + group) * staged; };
    auto shift = [](const T *row) { return (int) (reinterpret_cast<unsigned long long>(row) & 15); };
    auto fetch = [&](int d, LL row) {
        if (row < a.rows) {
            const T *src[2] = {px + row * a.xRow, pdz + row * a.dzRow};
#pragma unroll
            for (int q = 0; q < 2; q++) {
                if constexpr (OWN) {
#pragma unroll
                    for (int j = 0; j < NP; j++)
                        if (t + G * j < words) ln_copy<sizeof(T) * V>(own(d, q, j), src[q] + (t + G * j) * V);
                } else {
                    const int off = shift(src[q]), bytes = (int) a.cols * (int) sizeof(T);
                    const char *from = reinterpret_cast<const char *>(src[q]) - off;
                    unsigned char *to = shared(d, q);
                    // the words wholly inside the row are copied as such, the at most two others element by element
                    for (int w = t; w * 16 < off + bytes; w += G) {
                        if (w * 16 >= off && w * 16 + 16 <= off + bytes) ln_copy<16>(to + w * 16, from + w * 16);
                        else {
#pragma unroll
                            for (int e = 0; e < 16; e += (int) sizeof(T)) {
                                const int at = w * 16 + e;
                                if (at >= off && at < off + bytes) *reinterpret_cast<T *>(to + at) = *reinterpret_cast<const T *>(from + at);
                            }
                        }
                    }
                }
            }
        }
        ln_commit();
    };
    LL r = (LL) blockIdx.x * groups + group;
    C mean = C(0), inv = C(0);
    if (r < a.rows) { mean = pMean[r]; inv = pInv[r]; }
#pragma unroll
    for (int d = 0; d < D; d++) fetch(d, r + d * step);
    int stage = 0;
    for (int parity = 0; r < a.rows; r += step, parity ^= 1) {
        C nextMean = C(0), nextInv = C(0);
        if (r + step < a.rows) { nextMean = pMean[r + step]; nextInv = pInv[r + step]; }
        ln_wait<D - 1>();
        const T *sx = nullptr, *sd = nullptr;
        if constexpr (!OWN) {
            ln_group_barrier(group, G);                        // everyone's copies of this row stand
            sx = reinterpret_cast<const T *>(shared(stage, 0) + shift(px + r * a.xRow));
            sd = reinterpret_cast<const T *>(shared(stage, 1) + shift(pdz + r * a.dzRow));
        }
        C h[NP][V], d[NP][V];
        LnPair<C> s = {C(0), C(0)};
#pragma unroll
        for (int j = 0; j < NP; j++) {
            const bool in = t + G * j < words;
            LnWord<T, V> wx, wd;
            if (in) {
                if constexpr (OWN) { wx = *own(stage, 0, j); wd = *own(stage, 1, j); }
                else { wx.v[0] = sx[t + G * j]; wd.v[0] = sd[t + G * j]; }
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                h[j][k] = in ? (Elem<T>::to_c(wx.v[k]) - mean) * inv : C(0);
                const C dz = in ? Elem<T>::to_c(wd.v[k]) : C(0);
                sg[j][k] = fma(dz, h[j][k], sg[j][k]);
                sb[j][k] += dz;
                d[j][k] = dz * gain[j][k];
                s.a += d[j][k];
                s.b = fma(d[j][k], h[j][k], s.b);
            }
        }
        if (OWN) fetch(stage, r + D * step);                   // these words have been read
        s.a = ln_warp_sum(s.a);
        s.b = ln_warp_sum(s.b);
        if (warps > 1 || !OWN) {
            if (lane == 0) slots[parity][warp] = s;
            ln_group_barrier(group, G);
            s = slots[parity][firstWarp];
            for (int k = 1; k < warps; k++) { s.a += slots[parity][firstWarp + k].a; s.b += slots[parity][firstWarp + k].b; }
        }
        if (!OWN) fetch(stage, r + D * step);                  // nobody reads this stage any more
        if (pdx) {
            s.a *= invN; s.b *= invN;
            T *dx = pdx + r * a.zRow;
#pragma unroll
            for (int j = 0; j < NP; j++) {
                if (t + G * j < words) {
                    LnWord<T, V> o;
#pragma unroll
                    for (int k = 0; k < V; k++) o.v[k] = Elem<T>::from_c(inv * (d[j][k] - s.a - h[j][k] * s.b));
                    o.store(dx + (t + G * j) * V);
                }
            }
        }
        mean = nextMean; inv = nextInv;
        stage = stage + 1 == D ? 0 : stage + 1;
    }
    ln_wait<0>();
    if (!a.dGain && !a.dBias) return;
    // the CTA's groups add up in shared memory, one after the other, then the CTA's sums become a partial row
    C *pg = static_cast<C *>(a.partials) + (LL) blockIdx.x * 2 * a.cols, *pb = pg + a.cols;
    C *tg = reinterpret_cast<C *>(ln_smem), *tb = tg + a.cols;
    __syncthreads();                                           // the stages have been read by all groups
    for (int q = 0; q < groups; q++) {
        if (q == group) {
#pragma unroll
            for (int j = 0; j < NP; j++) {
                if (t + G * j < words) {
#pragma unroll
                    for (int k = 0; k < V; k++) {
                        const int c = (t + G * j) * V + k;
                        C vg = sg[j][k], vb = sb[j][k];
                        if (q > 0) { vg += tg[c]; vb += tb[c]; }
                        if (q + 1 < groups) { tg[c] = vg; tb[c] = vb; }
                        else { pg[c] = vg; pb[c] = vb; }
                    }
                }
            }
        }
        if (groups > 1) __syncthreads();
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
        const C mean = ln_row_sum<false>(s, slots) / n;
        s = C(0);
        for (LL c = threadIdx.x; c < a.cols; c += kLnSweepThreads) {
            const C v = Elem<T>::load(x + view_offset(a.xInner, c)) - mean;
            s = fma(v, v, s);
        }
        const C inv = C(1) / sqrt(ln_row_sum<false>(s, slots) / n + (C) a.epsilon);
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
        sa = ln_row_sum<false>(sa, slots) / n;
        sb = ln_row_sum<false>(sb, slots) / n;
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
template <class T> struct LnFit {
    // values per thread the register budget is set for: 32 / 16 of float, half of that of double
    static constexpr int kBig = sizeof(typename Elem<T>::C) == 8 ? 16 : 32;
    static constexpr int kMid = kBig / 2;
    static constexpr int kSmall = kBig / 4;
};
inline int threads_for(LL cols, int perThread, int most) {
    LL t = ceil_div(ceil_div(cols, perThread), 32) * 32;
    return t > most ? 0 : (int) t;
}
inline unsigned grid_for(LL n) { return (unsigned) (n < 0x7fffffffLL ? (n > 0 ? n : 1) : 0x7fffffffLL); }

template <class T, int V> void ln_forward_rows(const LnArgs &a, cudaStream_t st) {
    typedef LnFit<T> F;
    // A warp per row needs no barrier; from the length on that 32 threads cannot hold, the CTA shares the row.
    if (a.cols <= 32 * F::kBig)
        launch_kernel(k_ln_forward<T, V, F::kBig / V, true>, dim3(grid_for(ceil_div(a.rows, 8))), dim3(256), st, a);
    else if (int t = threads_for(a.cols, F::kMid, 1024))
        launch_kernel(k_ln_forward<T, V, F::kMid / V, false>, dim3(grid_for(a.rows)), dim3((unsigned) t), st, a);
    else
        launch_kernel(k_ln_forward<T, V, F::kBig / V, false>, dim3(grid_for(a.rows)), dim3(1024), st, a);
}

template <class T> Status ln_forward(LnArgs &a, bool rows, bool words, cudaStream_t st) {
    if (rows && a.cols <= 1024 * LnFit<T>::kBig) {
        if (words) ln_forward_rows<T, Elem<T>::kVec>(a, st);
        else ln_forward_rows<T, 1>(a, st);
    } else {
        launch_kernel(k_ln_forward_sweep<T>, dim3(grid_for(a.rows)), dim3(kLnSweepThreads), st, a);
    }
    ND_CUDA(cudaGetLastError());
    return kOk;
}

template <class K> inline void launch_with_smem(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t st, const LnArgs &a, int G) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_tuning[kTuneOverlapLaunch] ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, a, G);
    count_launch();
}

// Launches the kernel for rows of unit stride: `block` threads in groups of G, D stages of rows in shared memory.
template <class T, int V, int NP, int D, int MAXT, int CTAS, bool OWN>
Status ln_backward_rows(LnArgs &a, int G, int block, cudaStream_t st) {
    typedef typename Elem<T>::C C;
    const int groups = block / G;
    const size_t stages = OWN ? (size_t) D * 2 * NP * V * sizeof(T) * block : (size_t) D * 2 * groups * ln_staged(a.cols, sizeof(T));
    const size_t fold = groups > 1 ? 2 * (size_t) a.cols * sizeof(C) : 0;
    const size_t smem = stages > fold ? stages : fold;
    auto kernel = k_ln_backward<T, V, NP, D, MAXT, CTAS, OWN>;
    if (smem > 48 * 1024 - 512) ND_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem));
    LL grid = (LL) kNumSMs * CTAS;
    if (grid > ceil_div(a.rows, groups)) grid = ceil_div(a.rows, groups);
    a.numPartials = (int) grid;
    Scratch scratch(st);
    const bool weights = a.dGain || a.dBias;
    if (weights) {
        ND_TRY(scratch.alloc((size_t) grid * 2 * (size_t) a.cols * sizeof(C)));
        a.partials = scratch.at<void>(0);
    }
    launch_with_smem(kernel, dim3((unsigned) grid), dim3((unsigned) block), smem, st, a, G);
    if (weights) launch_kernel(k_ln_fold<T>, dim3((unsigned) ceil_div(a.cols, 32)), dim3(1024), st, a);
    ND_CUDA(cudaGetLastError());
    return kOk;
}

// V values per word and per copy. Up to 256 threads of kSmall values a CTA takes several rows at a time and shares the
// SM with two others; longer rows take a CTA, and twice the values per thread once 512 threads do not hold them.
template <class T, int V, bool OWN> Status ln_backward_fit(LnArgs &a, cudaStream_t st) {
    typedef LnFit<T> F;
    constexpr int kStages = sizeof(T) == 2 ? 6 : 4;          // 192 KB per SM for float and double, 144 KB for half
    if (int G = threads_for(a.cols, F::kSmall, 256)) return ln_backward_rows<T, V, F::kSmall / V, kStages, 256, 3, OWN>(a, G, 256 / G * G, st);
    if (int G = threads_for(a.cols, F::kSmall, 512)) return ln_backward_rows<T, V, F::kSmall / V, kStages, 512, 1, OWN>(a, G, G, st);
    return ln_backward_rows<T, V, F::kMid / V, 3, 512, 1, OWN>(a, threads_for(a.cols, F::kMid, 512), threads_for(a.cols, F::kMid, 512), st);
}

template <class T> Status ln_backward(LnArgs &a, bool rows, bool words, cudaStream_t st) {
    typedef typename Elem<T>::C C;
    if (rows && a.rows > 0 && threads_for(a.cols, LnFit<T>::kMid, 512)) {
        if (words) return ln_backward_fit<T, Elem<T>::kVec, true>(a, st);
        return ln_backward_fit<T, 1, sizeof(T) >= 4>(a, st);
    }
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
