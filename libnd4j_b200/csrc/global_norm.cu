// The Euclidean norm over all values of many tensors, and clipping by it:
//
//   norm = sqrt( sum over tensors and elements of x^2 ),    z = norm > maxNorm ? x * (maxNorm / norm) : x
//
// A training step bounds its update with it. Composed from the reduce and scalar families it takes a launch and a
// host round trip per tensor; here the tensors are cut into chunks of equal size, whatever their lengths, that the
// CTAs of one launch share out, and the value never visits the host.
//
// What bounds it: HBM. The norm reads every value once, clipping reads it again and writes it; of the second read,
// what the first left in L2 (126 MB) is found there, because the second launch takes the chunks in reverse order.
// Squares are summed in double: the sum of 2^27 of them in float would lose 1e-4 to the order of the additions, and
// squares of floats beyond 1.8e19 or below 1e-19 would leave the range of a float. (Half: the square of a half is exact in
// float, and the eight of one 128-bit word are added there, seven roundings of 2^-24, before they join the double sum.)
// Partial sums are one per CTA, folded in the same order by every CTA of the second launch, so the result does not depend
// on scheduling.
//
// Measured: 2^27 floats in 60 tensors, 87 us for the norm (6.2 TB/s) and 172 us for the scaling (6.2 TB/s) with cold
// caches, 270 us together where the second launch finds the first one's last chunks in L2. Two CTAs of 512 threads per SM
// keep 64 KB of reads in flight there.
#include "../../include/nd4j_b200.h"
#include <algorithm>
#include <cooperative_groups.h>
#include <vector>
#include "device_utils.cuh"
#include "entry_checks.h"

namespace cg = cooperative_groups;

namespace nd4jb200 {
namespace {

constexpr int kGnThreads = 512;
constexpr int kGnPacks = 4;                                 // 128-bit words per thread and chunk, all in flight at once
constexpr LL kGnChunk = (LL) kGnThreads * kGnPacks;         // in words
constexpr int kGnCtasPerSm = 2;
constexpr int kGnTensors = 256;                             // tensors per launch: the table travels as a kernel parameter, so
                                                            // that a captured graph holds a copy of its own
constexpr int kGnFewTensors = 64;                           // ... and a small one where few tensors are given
// Bytes of the first sweep left in L2 for the second (clipping 2^27 floats: 276 us with none, 272 with 32 MB, 270 with 80).
constexpr LL kGnKeep = 80LL << 20;

struct GnTensor {
    const void *x;
    void *z;
    LL length;
    int firstChunk;      // number of this tensor's first chunk
    int head;            // elements between the 16-byte boundary below x and x
};

template <int N> struct GnArgs {
    double *partials;        // of this launch's CTAs (norm), of all launches' CTAs (clip)
    int numPartials;         // clip: how many there are in all
    int numTensors;
    int numChunks;
    int keepFrom;            // chunks from this one on stay in L2 between the sweeps
    double maxNorm;
    void *norm;
    GnTensor t[N];
};

template <class T> ND_D double gn_square_sum(const Pack<T> &p) {
    double s = 0;
#pragma unroll
    for (int k = 0; k < Elem<T>::kVec; k++) { const double v = (double) p.v[k]; s = fma(v, v, s); }
    return s;
}
template <> ND_D double gn_square_sum<__half>(const Pack<__half> &p) {
    float s = 0;
#pragma unroll
    for (int k = 0; k < Elem<__half>::kVec; k++) { const float v = __half2float(p.v[k]); s = fmaf(v, v, s); }
    return (double) s;
}

// Sum over the CTA; every thread gets it. Warps by shuffles, then all warps' sums in the same order.
ND_D double gn_block_sum(double v, double *slots) {
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    double r = 0;
#pragma unroll
    for (int k = 0; k < kGnThreads / 32; k++) r += slots[k];
    return r;
}

// The tensor that chunk c belongs to: the last one whose first chunk is not behind c.
template <int N> ND_D int gn_find(const GnArgs<N> &a, int c) {
    int lo = 0, hi = a.numTensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].firstChunk <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// The words of one chunk. Word p of a tensor holds elements [p * V - head, p * V - head + V), so that every word is
// aligned; the first and the last may stick out and are read element by element, with zeros outside.
template <class T> ND_D Pack<T> gn_word(const T *x, LL e, LL length, bool keep) {
    constexpr int V = Elem<T>::kVec;
    Pack<T> v;
    if (e >= 0 && e + V <= length) {
        if (keep) v = load_pack_rw(x + e);
        else *reinterpret_cast<uint4 *>(&v) = __ldcs(reinterpret_cast<const uint4 *>(x + e));
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) v.v[k] = e + k >= 0 && e + k < length ? x[e + k] : Elem<T>::from_c(0);
    }
    return v;
}
template <class T> ND_D void gn_store(T *z, LL e, LL length, bool words, const Pack<T> &v) {
    constexpr int V = Elem<T>::kVec;
    if (words && e >= 0 && e + V <= length) __stcs(reinterpret_cast<uint4 *>(z + e), *reinterpret_cast<const uint4 *>(&v));
    else {
#pragma unroll
        for (int k = 0; k < V; k++) if (e + k >= 0 && e + k < length) z[e + k] = v.v[k];
    }
}
// What the values are multiplied with. A factor near or below the type's smallest normal value would lose bits, or all of
// them, that the products with values as large as such a norm still have: those are taken relative to the norm first, in double.
template <class C> struct GnFactor {
    C f;
    bool clip, tiny;
    double inv, most;
    ND_D GnFactor(double n, double m) : inv(1.0 / n), most(m) {
        clip = n > m && isfinite((C) n);
        const double q = clip ? m / n : 1.0;
        f = (C) q;
        tiny = q < (sizeof(C) == 4 ? 0x1p-100 : 0x1p-1000) && m > 0;
    }
};
template <class T> ND_D void gn_scale(Pack<T> &v, const GnFactor<typename Elem<T>::C> &g) {
    typedef typename Elem<T>::C C;
    if (!g.tiny) {
#pragma unroll
        for (int k = 0; k < Elem<T>::kVec; k++) v.v[k] = Elem<T>::from_c(Elem<T>::to_c(v.v[k]) * g.f);
    } else {
#pragma unroll
        for (int k = 0; k < Elem<T>::kVec; k++) v.v[k] = Elem<T>::from_c((C) ((double) Elem<T>::to_c(v.v[k]) * g.inv * g.most));
    }
}
template <class T> ND_D bool gn_words(const GnTensor &t) {          // z has x's place in a 16-byte word
    return ((reinterpret_cast<unsigned long long>(t.z) - (unsigned long long) t.head * sizeof(T)) & 15) == 0;
}
template <class T> ND_D void gn_load(const GnTensor &t, LL firstWord, bool keep, Pack<T> (&v)[kGnPacks]) {
#pragma unroll
    for (int j = 0; j < kGnPacks; j++)
        v[j] = gn_word(static_cast<const T *>(t.x), (firstWord + (LL) j * kGnThreads + threadIdx.x) * Elem<T>::kVec - t.head, t.length, keep);
}

template <class T, int N>
__global__ void __launch_bounds__(kGnThreads, kGnCtasPerSm) k_global_norm(const __grid_constant__ GnArgs<N> a) {
    grid_dependency_sync();
    __shared__ double slots[kGnThreads / 32];
    double s = 0;
    for (int c = blockIdx.x; c < a.numChunks; c += gridDim.x) {
        const GnTensor &t = a.t[gn_find(a, c)];
        Pack<T> v[kGnPacks];
        gn_load<T>(t, (LL) (c - t.firstChunk) * kGnChunk, c >= a.keepFrom, v);
#pragma unroll
        for (int j = 0; j < kGnPacks; j++) s += gn_square_sum<T>(v[j]);
    }
    s = gn_block_sum(s, slots);
    if (threadIdx.x == 0) a.partials[blockIdx.x] = s;
}

// Folds the partial sums and, with z, scales. A norm that is not finite scales nothing: the caller sees it in `norm`.
template <class T, int N, bool SCALE>
__global__ void __launch_bounds__(kGnThreads, kGnCtasPerSm) k_clip_by_norm(const __grid_constant__ GnArgs<N> a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    constexpr int V = Elem<T>::kVec;
    __shared__ double slots[kGnThreads / 32];
    double s = 0;
    for (int i = threadIdx.x; i < a.numPartials; i += kGnThreads) s += a.partials[i];
    const double norm = sqrt(gn_block_sum(s, slots));
    if (blockIdx.x == 0 && threadIdx.x == 0) *static_cast<C *>(a.norm) = (C) norm;
    if (!SCALE) return;
    const GnFactor<C> factor(norm, a.maxNorm);
    for (int c = a.numChunks - 1 - (int) blockIdx.x; c >= 0; c -= gridDim.x) {
        const GnTensor &t = a.t[gn_find(a, c)];
        if (!factor.clip && t.x == t.z) continue;
        const LL firstWord = (LL) (c - t.firstChunk) * kGnChunk;
        Pack<T> v[kGnPacks];
        gn_load<T>(t, firstWord, false, v);
        const bool words = gn_words<T>(t);
#pragma unroll
        for (int j = 0; j < kGnPacks; j++) {
            if (factor.clip) gn_scale<T>(v[j], factor);
            gn_store<T>(static_cast<T *>(t.z), (firstWord + (LL) j * kGnThreads + threadIdx.x) * V - t.head, t.length, words, v[j]);
        }
    }
}

// Few values: one launch of one cluster, which keeps them in registers between the two sweeps and joins its sums through
// distributed shared memory. Two words per thread: 30000 floats take 8.2 us (10.9 in two launches, both from the start of
// a replayed graph), 60000 10.3; with eight words 200000 floats take 14.3, since eight SMs then read what 54 would.
constexpr int kGnOneThreads = 1024, kGnOneCtas = 8, kGnOneWords = 2;
constexpr LL kGnOneMost = (LL) kGnOneThreads * kGnOneCtas * kGnOneWords;        // words
template <class T, bool SCALE>
__global__ void __launch_bounds__(kGnOneThreads) k_clip_at_once(const __grid_constant__ GnArgs<kGnFewTensors> a) {
    grid_dependency_sync();
    typedef typename Elem<T>::C C;
    constexpr int V = Elem<T>::kVec;
    __shared__ double warpSums[kGnOneThreads / 32], ctaSum;
    __shared__ GnTensor table[kGnFewTensors];                   // threads of a warp look at different tensors
    cg::cluster_group cl = cg::this_cluster();
    for (int i = threadIdx.x; i < a.numTensors; i += kGnOneThreads) table[i] = a.t[i];
    __syncthreads();
    Pack<T> v[kGnOneWords];
    int tensor[kGnOneWords];
    double s = 0;
    auto word = [&](int j) { return (j * kGnOneCtas + (int) blockIdx.x) * kGnOneThreads + (int) threadIdx.x; };
    auto element = [&](int j, const GnTensor &t) { return (LL) (word(j) - t.firstChunk) * V - t.head; };
#pragma unroll
    for (int j = 0; j < kGnOneWords; j++) {
        const int w = word(j);
        int lo = 0, hi = a.numTensors - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (table[mid].firstChunk <= w) lo = mid; else hi = mid - 1;
        }
        tensor[j] = w < a.numChunks ? lo : -1;                  // here the "chunks" are single words
        if (tensor[j] >= 0) v[j] = gn_word(static_cast<const T *>(table[lo].x), element(j, table[lo]), table[lo].length, true);
    }
#pragma unroll
    for (int j = 0; j < kGnOneWords; j++) if (tensor[j] >= 0) s += gn_square_sum<T>(v[j]);
    for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if ((threadIdx.x & 31) == 0) warpSums[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = warpSums[threadIdx.x];
        for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (threadIdx.x == 0) ctaSum = s;
    }
    cl.sync();
    s = 0;
#pragma unroll
    for (int q = 0; q < kGnOneCtas; q++) s += *cl.map_shared_rank(&ctaSum, q);
    cl.sync();                                                  // nobody leaves while its sum is being read
    const double norm = sqrt(s);
    if (blockIdx.x == 0 && threadIdx.x == 0) *static_cast<C *>(a.norm) = (C) norm;
    if (!SCALE) return;
    const GnFactor<C> factor(norm, a.maxNorm);
#pragma unroll
    for (int j = 0; j < kGnOneWords; j++) {
        if (tensor[j] < 0) continue;
        const GnTensor &t = table[tensor[j]];
        if (!factor.clip && t.x == t.z) continue;
        if (factor.clip) gn_scale<T>(v[j], factor);
        gn_store<T>(static_cast<T *>(t.z), element(j, t), t.length, gn_words<T>(t), v[j]);
    }
}

template <class T> Status gn_run_at_once(const std::vector<GnTensor> &all, LL words, bool scale, double maxNorm, void *norm, cudaStream_t st) {
    GnArgs<kGnFewTensors> a = {};
    a.numTensors = (int) all.size();
    a.numChunks = (int) words;
    a.maxNorm = maxNorm;
    a.norm = norm;
    LL first = 0;
    for (size_t i = 0; i < all.size(); i++) {
        a.t[i] = all[i];
        a.t[i].head = (int) ((reinterpret_cast<uintptr_t>(all[i].x) & 15) / sizeof(T));
        a.t[i].firstChunk = (int) first;
        first += ceil_div(all[i].length + a.t[i].head, Elem<T>::kVec);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kGnOneCtas); cfg.blockDim = dim3(kGnOneThreads); cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kGnOneCtas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_tuning[kTuneOverlapLaunch] ? 2 : 1;
    if (scale) cudaLaunchKernelEx(&cfg, k_clip_at_once<T, true>, a);
    else cudaLaunchKernelEx(&cfg, k_clip_at_once<T, false>, a);
    count_launch();
    ND_CUDA(cudaGetLastError());
    return kOk;
}

template <class T, int N>
Status gn_run(const std::vector<GnTensor> &all, bool scale, double maxNorm, void *norm, cudaStream_t st) {
    constexpr LL V = Elem<T>::kVec;
    const size_t launches = all.empty() ? 1 : (all.size() + N - 1) / N;
    constexpr int kGrid = kNumSMs * kGnCtasPerSm;
    if (launches * kGrid > (size_t) 1 << 24) return bad_arg("global norm: too many tensors");
    Scratch scratch(st);
    ND_TRY(scratch.alloc(launches * kGrid * sizeof(double)));
    double *partials = scratch.at<double>(0);
    std::vector<GnArgs<N>> args(launches);
    int numPartials = 0;
    for (size_t l = 0; l < launches; l++) {
        GnArgs<N> &a = args[l];
        a.numTensors = 0;
        LL chunks = 0;
        for (size_t i = l * N; i < all.size() && i < (l + 1) * N; i++) {
            GnTensor t = all[i];
            t.head = (int) ((reinterpret_cast<uintptr_t>(t.x) & 15) / sizeof(T));
            t.firstChunk = (int) chunks;
            chunks += ceil_div(ceil_div(t.length + t.head, V), kGnChunk);
            if (chunks > 0x3fffffff) return bad_arg("global norm: too many values in one call");
            a.t[a.numTensors++] = t;
        }
        a.numChunks = (int) chunks;
        // the launch whose values the second sweep begins with keeps its last ones in L2
        a.keepFrom = scale && l == launches - 1 ? (int) (chunks - kGnKeep / (kGnChunk * 16)) : (int) chunks;
        a.maxNorm = maxNorm;
        a.norm = norm;
        a.numPartials = chunks < kGrid ? (int) chunks : kGrid;      // for now: this launch's
        a.partials = partials + numPartials;
        if (a.numPartials > 0)
            launch_kernel(k_global_norm<T, N>, dim3((unsigned) a.numPartials), dim3(kGnThreads), st, a);
        numPartials += a.numPartials;
    }
    for (size_t l = launches; l-- > 0;) {                           // the values read last are scaled first
        GnArgs<N> &a = args[l];
        const unsigned grid = scale && a.numPartials > 0 ? (unsigned) a.numPartials : 1;
        a.partials = partials;
        a.numPartials = numPartials;
        if (scale) launch_kernel(k_clip_by_norm<T, N, true>, dim3(grid), dim3(kGnThreads), st, a);
        else if (l == 0) launch_kernel(k_clip_by_norm<T, N, false>, dim3(1), dim3(kGnThreads), st, a);
    }
    ND_CUDA(cudaGetLastError());
    return kOk;
}

// Every written range has to be its own: two tensors that share bytes would be scaled twice, in an order that nothing
// fixes, and a result over another tensor's operand would be read back as an operand.
Status gn_check_ranges(const std::vector<GnTensor> &all, size_t elem) {
    struct Range { uintptr_t lo, hi; size_t i; };
    std::vector<Range> z;
    z.reserve(all.size());
    bool sorted = true, apart = false;
    for (size_t i = 0; i < all.size(); i++) {
        const uintptr_t lo = reinterpret_cast<uintptr_t>(all[i].z);
        z.push_back(Range{lo, lo + (uintptr_t) all[i].length * elem, i});
        if (i > 0 && lo < z[i - 1].lo) sorted = false;
        if (all[i].x != all[i].z) apart = true;
    }
    if (!sorted) std::sort(z.begin(), z.end(), [](const Range &a, const Range &b) { return a.lo < b.lo; });
    for (size_t k = 1; k < z.size(); k++)
        if (z[k].lo < z[k - 1].hi) {
            std::ostringstream os;
            os << "clip by global norm: the results of tensors " << z[k - 1].i << " and " << z[k].i << " overlap";
            return bad_arg(os.str());
        }
    if (!apart) return kOk;
    for (size_t i = 0; i < all.size(); i++) {
        const uintptr_t lo = reinterpret_cast<uintptr_t>(all[i].x), hi = lo + (uintptr_t) all[i].length * elem;
        auto it = std::lower_bound(z.begin(), z.end(), hi, [](const Range &a, uintptr_t v) { return a.lo < v; });
        // ranges are disjoint and ascending: only those that begin below hi can meet [lo, hi), the last ones first
        while (it != z.begin()) {
            --it;
            if (it->hi <= lo) break;
            if (it->i == i && it->lo == lo) continue;       // in place
            std::ostringstream os;
            os << "clip by global norm: the result of tensor " << it->i << " overlaps the operand of tensor " << i;
            return bad_arg(os.str());
        }
    }
    return kOk;
}

template <class T> Status gn_choose(const std::vector<GnTensor> &all, bool scale, double maxNorm, void *norm, cudaStream_t st) {
    if (all.size() > kGnFewTensors) return gn_run<T, kGnTensors>(all, scale, maxNorm, norm, st);
    LL words = 0;
    for (const GnTensor &t : all) words += ceil_div(t.length + (LL) ((reinterpret_cast<uintptr_t>(t.x) & 15) / sizeof(T)), Elem<T>::kVec);
    if (words <= kGnOneMost) return gn_run_at_once<T>(all, words, scale, maxNorm, norm, st);
    return gn_run<T, kGnFewTensors>(all, scale, maxNorm, norm, st);
}

Status gn_entry(void *stream, int dtype, const void *const *x, void *const *z, bool clip, const Nd4jLong *lengths, int n,
                double maxNorm, void *norm) {
    ND_TRY(require_dtype(dtype));
    if (n < 0) return bad_arg("the number of tensors is negative");
    if (n > 0) { ND_TRY(require(x, "x")); ND_TRY(require(lengths, "lengths")); }
    ND_TRY(require(norm, "norm"));
    const size_t elem = size_of_dtype(dtype), wide = size_of_wide(dtype);
    ND_TRY(require_aligned(norm, wide, "norm"));
    if (clip && !(maxNorm >= 0 && std::isfinite(maxNorm))) return bad_arg("maxNorm must be finite and not negative");
    std::vector<GnTensor> all;
    all.reserve((size_t) n);
    const Span normSpan = span_of(norm, 1, wide);
    for (int i = 0; i < n; i++) {
        if (lengths[i] < 0 || lengths[i] > (1LL << 42)) return bad_arg("the length of a tensor is negative or too large");
        if (lengths[i] == 0) continue;
        GnTensor t = {};
        t.x = x[i];
        t.z = clip ? (z ? z[i] : const_cast<void *>(x[i])) : nullptr;
        t.length = lengths[i];
        ND_TRY(require(t.x, "a tensor of x"));
        ND_TRY(require_aligned(t.x, elem, "a tensor of x"));
        if (clip) {
            ND_TRY(require(t.z, "a tensor of z"));
            ND_TRY(require_aligned(t.z, elem, "a tensor of z"));
            ND_TRY(check_apart(normSpan, "norm", span_of(t.z, t.length, elem), "a tensor of z"));
        }
        ND_TRY(check_apart(normSpan, "norm", span_of(t.x, t.length, elem), "a tensor of x"));
        all.push_back(t);
    }
    if (clip) ND_TRY(gn_check_ranges(all, elem));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kF32: return gn_choose<float>(all, clip, maxNorm, norm, st);
        case kF64: return gn_choose<double>(all, clip, maxNorm, norm, st);
        default: return gn_choose<__half>(all, clip, maxNorm, norm, st);
    }
}

}  // namespace
}  // namespace nd4jb200

using namespace nd4jb200;

#pragma GCC visibility push(default)
extern "C" {

int nd4jb200_exec_global_norm(void *stream, int dtype, const void *const *x, const Nd4jLong *lengths, int n, void *norm) {
    return c_entry([&] { return gn_entry(stream, dtype, x, nullptr, false, lengths, n, 0, norm); });
}

int nd4jb200_exec_clip_by_global_norm(void *stream, int dtype, const void *const *x, void *const *z, const Nd4jLong *lengths,
                                      int n, double maxNorm, void *norm) {
    return c_entry([&] { return gn_entry(stream, dtype, x, z, true, lengths, n, maxNorm, norm); });
}

}  // extern "C"
#pragma GCC visibility pop
