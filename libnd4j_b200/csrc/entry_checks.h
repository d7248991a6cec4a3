// Host-side helpers of the operators between a language model's matrix products (layer_norm.cu, token_log_probs.cu,
// embedding.cu, global_norm.cu): the guard around a C entry point, argument checks that need no device access, and
// scratch memory that belongs to one call.
#pragma once
#include <cmath>
#include <exception>
#include <numeric>
#include <sstream>
#include "runtime.h"

namespace nd4jb200 {

// No C++ exception may leave a C entry point: what can be thrown here is a failed host allocation.
template <class F> inline int c_entry(F body) noexcept {
    try {
        return (int) body();
    } catch (...) {
        try { set_error("out of host memory"); } catch (...) {}
        return (int) kTooLarge;
    }
}

// Scratch of one call: taken from a stream-ordered pool and given back to it at the end of the scope, in stream
// order. Unlike the per-stream workspace it is never shared: calls from several host threads on one stream, and
// graphs captured on one stream and replayed on several, each work in memory of their own. (Inside a capture the
// allocation becomes a node of the graph.) The pool keeps what it was given, so that an eager call costs about a
// microsecond of host time, up to kScratchKept bytes per device: what it holds beyond that goes back to the device at the
// next synchronisation, and all that is not in use with nd4jb200_release_scratch. A table gradient over 32768 tokens of 2048
// halves takes 9 MB, layer norm's weights over rows of 4096 floats 10; a call that has to map its memory anew pays for it
// (512 MB: 1.6 ms with what it needs in the pool, 6.9 without).
constexpr unsigned long long kScratchKept = 1ull << 30;
class Scratch {
public:
    explicit Scratch(cudaStream_t s) : stream(s) {}
    Scratch(const Scratch &) = delete;
    Scratch &operator=(const Scratch &) = delete;
    ~Scratch() { if (ptr) cudaFreeAsync(ptr, stream); }
    Status alloc(size_t bytes);
    template <class P> P *at(size_t byteOffset) const { return reinterpret_cast<P *>(static_cast<char *>(ptr) + byteOffset); }
private:
    cudaStream_t stream;
    void *ptr = nullptr;
};
// Gives back to the current device what its pool holds and no call uses.
Status release_scratch();

// Lets a kernel use `bytes` of dynamic shared memory, asked for once per kernel and device (about a microsecond each time
// otherwise). `asked` is the kernel's own word, one bit per device.
inline Status allow_shared(const void *kernel, size_t bytes, std::atomic<unsigned long long> &asked) {
    if (bytes <= 46 * 1024) return kOk;             // 48 KB with what the kernels declare statically
    int device = 0;
    ND_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = 1ull << (device & 63);
    if (device < 64 && (asked.load(std::memory_order_relaxed) & bit)) return kOk;
    int most = 0;
    ND_CUDA(cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device));
    cudaFuncAttributes attr;
    ND_CUDA(cudaFuncGetAttributes(&attr, kernel));
    ND_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int) attr.sharedSizeBytes));
    asked.fetch_or(bit, std::memory_order_relaxed);
    return kOk;
}
inline size_t round_up(size_t n, size_t to) { return (n + to - 1) / to * to; }

inline size_t size_of_dtype(int dtype) { return dtype == kF64 ? 8 : (dtype == kF16 ? 2 : 4); }
inline size_t size_of_wide(int dtype) { return dtype == kF64 ? 8 : 4; }    // what sums and statistics are held in

inline Status require(const void *p, const char *name) {
    if (p == nullptr) return bad_arg(std::string(name) + " is null");
    return kOk;
}
inline Status require_dtype(int dtype) {
    if (dtype != kF32 && dtype != kF64 && dtype != kF16) return bad_arg("dtype must be 0 (float), 1 (double) or 2 (half)");
    return kOk;
}
inline Status require_aligned(const void *p, size_t bytes, const char *name) {
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0) return bad_arg(std::string(name) + " is not aligned to its element type");
    return kOk;
}

// Bytes [lo, hi) that an array's elements lie in, and whether they fill that range.
struct Span { uintptr_t lo, hi; bool filled; };
inline Span span_of(const void *p, const ShapeDesc &d, size_t elem) {
    LL lo = 0, hi = 0;
    for (int i = 0; i < d.rank; i++) {
        const LL reach = d.shape[i] > 0 ? (d.shape[i] - 1) * d.stride[i] : 0;
        if (reach < 0) lo += reach; else hi += reach;
    }
    const uintptr_t base = reinterpret_cast<uintptr_t>(p);
    Span s;
    s.lo = base + (uintptr_t) (lo * (LL) elem);
    s.hi = base + (uintptr_t) ((hi + 1) * (LL) elem);
    if (d.length == 0) s.hi = s.lo;
    s.filled = hi - lo + 1 == d.length;
    return s;
}
inline Span span_of(const void *p, LL n, size_t elem) {
    const uintptr_t base = reinterpret_cast<uintptr_t>(p);
    return Span{base, base + (uintptr_t) n * elem, true};
}
// Whether two arrays certainly share bytes. The first and the last byte of a span belong to an element in any case, and
// those between to one where the span is filled.
inline bool meet(const Span &a, const Span &b) {
    if (!(a.lo < b.hi && b.lo < a.hi && a.lo < a.hi && b.lo < b.hi)) return false;
    if (a.filled && b.filled) return true;
    if (a.lo == b.lo || a.hi == b.hi) return true;
    const bool inA = a.lo <= b.lo || b.hi <= a.hi, inB = b.lo <= a.lo || a.hi <= b.hi;     // an end of one inside the other
    return (a.filled && inA) || (b.filled && inB);
}

inline bool same_layout(const ShapeDesc &a, const ShapeDesc &b) {
    if (a.rank != b.rank) return false;
    for (int i = 0; i < a.rank; i++)
        if (a.shape[i] != b.shape[i] || (a.shape[i] > 1 && a.stride[i] != b.stride[i])) return false;
    return true;
}

// A result may take the place of an operand (same address, same layout). Where the two certainly share bytes in any
// other way the call is refused; interleaved views of one parent cannot be told apart here and are the caller's care.
inline Status check_alias(const void *out, const ShapeDesc &od, const char *outName, const void *in, const ShapeDesc &id,
                          const char *inName, size_t elem) {
    if (out == in && same_layout(od, id)) return kOk;
    const Span a = span_of(out, od, elem), b = span_of(in, id, elem);
    if (meet(a, b) || (out == in && od.length > 0))
        return bad_arg(std::string(outName) + " overlaps " + inName + " without being the same array");
    return kOk;
}
inline Status check_apart(const Span &a, const char *aName, const Span &b, const char *bName) {
    if (meet(a, b)) return bad_arg(std::string(aName) + " overlaps " + bName);
    return kOk;
}
// A written array needs a place of its own for every element: two of them would be written by different CTAs, in an order
// that nothing fixes. Two axes of strides s and t meet where i s = j t, first at i = t / gcd, j = s / gcd; an array may not
// reach that far along both (for matrices this is exact). And no array has more elements than its span has places.
inline Status check_written(const ShapeDesc &d, const char *name) {
    if (d.length < 2) return kOk;
    unsigned long long reach = 0;
    for (int i = 0; i < d.rank; i++) {
        if (d.shape[i] < 2) continue;
        if (d.stride[i] == 0) return bad_arg(std::string(name) + ": a result cannot have a stride of 0");
        const unsigned long long s = d.stride[i] < 0 ? 0 - (unsigned long long) d.stride[i] : (unsigned long long) d.stride[i];
        reach += s * (unsigned long long) (d.shape[i] - 1);
        for (int j = 0; j < i; j++) {
            if (d.shape[j] < 2) continue;
            const unsigned long long t = d.stride[j] < 0 ? 0 - (unsigned long long) d.stride[j] : (unsigned long long) d.stride[j];
            const unsigned long long g = std::gcd(s, t);
            if (t / g < (unsigned long long) d.shape[i] && s / g < (unsigned long long) d.shape[j])
                return bad_arg(std::string(name) + ": a result cannot have elements that share their place");
        }
    }
    if (reach < (unsigned long long) (d.length - 1)) return bad_arg(std::string(name) + ": a result cannot have elements that share their place");
    return kOk;
}
inline bool equal_shape(const ShapeDesc &a, const ShapeDesc &b) {
    if (a.rank != b.rank) return false;
    for (int i = 0; i < a.rank; i++) if (a.shape[i] != b.shape[i]) return false;
    return true;
}

}  // namespace nd4jb200
