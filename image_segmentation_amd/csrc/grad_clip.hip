// Global norm of a list of tensors and clipping by it:  total = |scale| (sum g^2)^(1/2)  or  |scale| max |g|,
//   c = min(1, max_norm / (total + 1e-6)),   out = c scale g
//
// Memory-bound: one read for the norm, then a read and a write where anything changes (in place with c = 1 the second pass ends at
// once).  The list travels by value in the kernels' arguments, so a call needs no device table and can be captured; tensors are cut
// into chunks and a workgroup takes one chunk.  Squares are summed in fp64 (free beside the loads: 136 us for 212 M bf16 values against
// 133 in fp32): neither 1e-30 nor 1e30 leaves the range, and the norm does not depend on how the list is cut beyond the last bit of an
// fp64 sum.  Chunk sums are joined in a fixed order: same bits every time.
// 599 tensors, 212 M bf16 values clipped into fp32: norm 120 us (3.5 TB/s; 129 in launches of 128 tensors), joining 6, scaling 257 (4.9 TB/s;
// a copy: 5.07).  Lists of a few hundred tensors are bound by the host's reading of them: 311 tensors, 69 M fp32 values with c = 1: 105 us,
// 61 of them the kernels'.
#include <algorithm>
#include <vector>

#include "kernels.hpp"

namespace lsam {
namespace {
constexpr int NT = 256;
constexpr int SELF_JOIN = 1024;          // up to so many chunk sums the second pass joins them itself: two launches instead of three

// Tensors of a launch, as many as stay below the 4 KB that kernel arguments may take: 208 that are read (and written in place), 128 with an
// output apart.
template <bool APART> struct Table {
    static constexpr int TAB = APART ? 128 : 208;
    const void* src[TAB];
    void* dst[APART ? TAB : 1];
    unsigned n[TAB];          // elements; longer tensors take several entries
    int first[TAB];           // first chunk of the entry, counted in this launch
    unsigned char kind[TAB];  // bit 0: src bf16, bit 1: dst bf16
    int count, chunks, chunk, base;   // entries, chunks of this launch, elements a chunk, chunks before this launch
};
static_assert(sizeof(Table<false>) <= 3700 && sizeof(Table<true>) <= 3700, "kernel arguments");

template <typename Tab> __device__ __forceinline__ int entry_of(const Tab& t, int c) {   // last entry whose first chunk is <= c
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Zero-initialised where used.  Norm: 2 sums squares in fp64; inf takes the largest bit pattern of |g|, in which NaN is above infinity
template <bool INF> struct Acc {
    double s;
    unsigned m;
    __device__ __forceinline__ void add(float v) {
        if constexpr (INF) {
            const unsigned b = __builtin_bit_cast(unsigned, v) & 0x7FFFFFFFu;
            m = b > m ? b : m;
        } else s = fma((double)v, (double)v, s);
    }
    __device__ __forceinline__ void join(const Acc& o) {
        if constexpr (INF) m = o.m > m ? o.m : m;
        else s += o.s;
    }
    __device__ __forceinline__ Acc shifted(int o) const {
        Acc r{};
        if constexpr (INF) r.m = __shfl_xor(m, o);
        else r.s = __shfl_xor(s, o);
        return r;
    }
    __device__ __forceinline__ double value() const { return INF ? (double)__builtin_bit_cast(float, m) : s; }
    __device__ __forceinline__ void take(double v) {
        if constexpr (INF) m = __builtin_bit_cast(unsigned, (float)v) & 0x7FFFFFFFu;
        else s = v;
    }
};

template <bool INF> __device__ __forceinline__ Acc<INF> block_join(Acc<INF> a, Acc<INF>* red) {   // result in every thread
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
#pragma unroll
    for (int o = 32; o; o >>= 1) a.join(a.shifted(o));
    if (lane == 0) red[wave] = a;
    __syncthreads();
    Acc<INF> r = red[0];
    for (int w = 1; w < nw; ++w) r.join(red[w]);
    return r;
}

template <typename T, bool INF> __device__ __forceinline__ void chunk_norm(const T* p, int n, Acc<INF>& a) {
    constexpr int V = 16 / (int)sizeof(T);
    const int tid = threadIdx.x;
    int lead = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
    lead = min(lead, n);
    if (tid < lead) a.add(to_f(p[tid]));
    const T* q = p + lead;
    const int nv = (n - lead) / V;
#pragma unroll 4
    for (int i = tid; i < nv; i += NT) {
        const uint4 u = reinterpret_cast<const uint4*>(q)[i];
        T e[V];
        __builtin_memcpy(e, &u, 16);
#pragma unroll
        for (int j = 0; j < V; ++j) a.add(to_f(e[j]));
    }
    const int rest = lead + nv * V;
    if (rest + tid < n) a.add(to_f(p[rest + tid]));
}

template <bool INF> __global__ __launch_bounds__(NT) void clip_norm_kernel(const Table<false> t, double* __restrict__ part) {
    __shared__ Acc<INF> red[NT / 64];
    const int c = blockIdx.x, e = entry_of(t, c);
    const unsigned o = (unsigned)(c - t.first[e]) * (unsigned)t.chunk;
    const int n = (int)min((unsigned)t.chunk, t.n[e] - o);
    Acc<INF> a{};
    if (t.kind[e] & 1) chunk_norm<bf16, INF>(static_cast<const bf16*>(t.src[e]) + o, n, a);
    else chunk_norm<float, INF>(static_cast<const float*>(t.src[e]) + o, n, a);
    a = block_join<INF>(a, red);
    if (threadIdx.x == 0) part[t.base + c] = a.value();
}

struct Limit { double max_norm, scale; };

__device__ __forceinline__ void norm_and_factor(double sum, bool inf, Limit l, float& norm, float& factor) {
    const double total = (inf ? sum : sqrt(sum)) * fabs(l.scale);
    const double c = l.max_norm / (total + 1e-6);
    norm = (float)total;
    factor = (float)((c < 1. || c != c ? c : 1.) * l.scale);   // NaN stays: what is not finite is not hidden
}

template <bool INF> __device__ __forceinline__ double join_parts(const double* part, int parts, Acc<INF>* red) {
    Acc<INF> a{};
    for (int i = threadIdx.x; i < parts; i += blockDim.x) {
        Acc<INF> b{};
        b.take(part[i]);
        a.join(b);
    }
    return block_join<INF>(a, red).value();
}

template <bool INF> __global__ __launch_bounds__(1024) void clip_join_kernel(const double* __restrict__ part, int parts, Limit l,
                                                                             float* __restrict__ out) {
    __shared__ Acc<INF> red[16];
    const double s = join_parts<INF>(part, parts, red);
    if (threadIdx.x == 0) norm_and_factor(s, INF, l, out[0], out[1]);
}

template <typename S, typename D> __device__ __forceinline__ void chunk_scale(const S* s, D* d, int n, float f) {
    constexpr int V = sizeof(S) == 4 || sizeof(D) == 4 ? 4 : 8;   // elements of 16 bytes of the wider type
    using SV = __attribute__((ext_vector_type(V))) S;
    using DV = __attribute__((ext_vector_type(V))) D;
    const int tid = threadIdx.x;
    // elements up to where both are aligned to their vectors; never, when their offsets differ
    const int ls = (int)((sizeof(SV) - (reinterpret_cast<uintptr_t>(s) & (sizeof(SV) - 1))) & (sizeof(SV) - 1)) / (int)sizeof(S);
    const int ld = (int)((sizeof(DV) - (reinterpret_cast<uintptr_t>(d) & (sizeof(DV) - 1))) & (sizeof(DV) - 1)) / (int)sizeof(D);
    if (ls != ld) {
#pragma unroll 4
        for (int i = tid; i < n; i += NT) d[i] = from_f<D>(to_f(s[i]) * f);
        return;
    }
    const int lead = min(ls, n), nv = (n - lead) / V, rest = lead + nv * V;
    if (tid < lead) d[tid] = from_f<D>(to_f(s[tid]) * f);
#pragma unroll 4
    for (int i = tid; i < nv; i += NT) {
        const SV v = reinterpret_cast<const SV*>(s + lead)[i];
        DV w;
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = from_f<D>(to_f(v[j]) * f);
        reinterpret_cast<DV*>(d + lead)[i] = w;
    }
    if (rest + tid < n) d[rest + tid] = from_f<D>(to_f(s[rest + tid]) * f);
}

// `parts` > 0: joins the chunk sums itself (every workgroup the same way) and the first one reports norm and factor
template <bool INF, bool APART>
__global__ __launch_bounds__(NT) void clip_scale_kernel(const Table<APART> t, const double* __restrict__ part, int parts, Limit l,
                                                        float* __restrict__ out) {
    __shared__ Acc<INF> red[NT / 64];
    float norm, f;
    if (parts > 0) {
        norm_and_factor(join_parts<INF>(part, parts, red), INF, l, norm, f);
        if (blockIdx.x == 0 && t.base == 0 && threadIdx.x == 0) {
            out[0] = norm;
            out[1] = f;
        }
    } else f = out[1];
    if (!APART && f == 1.f) return;   // nothing changes
    const int c = blockIdx.x, e = entry_of(t, c), kind = t.kind[e];
    const void* src = t.src[e];
    void* dst = APART ? t.dst[e] : const_cast<void*>(src);
    if (f == 1.f && src == dst) return;
    const unsigned o = (unsigned)(c - t.first[e]) * (unsigned)t.chunk;
    const int n = (int)min((unsigned)t.chunk, t.n[e] - o);
    if (kind == 0) chunk_scale(static_cast<const float*>(src) + o, static_cast<float*>(dst) + o, n, f);
    else if (kind == 3) chunk_scale(static_cast<const bf16*>(src) + o, static_cast<bf16*>(dst) + o, n, f);
    else if constexpr (APART) {   // in place the types are one
        if (kind == 1) chunk_scale(static_cast<const bf16*>(src) + o, static_cast<float*>(dst) + o, n, f);
        else chunk_scale(static_cast<const float*>(src) + o, static_cast<bf16*>(dst) + o, n, f);
    }
}

constexpr long ENTRY = 1l << 30;   // elements an entry of the table may have

// elements a chunk: about 2048 workgroups, 2 Ki to 16 Ki elements.  212 M bf16 values into fp32: both passes 396 us with 16 Ki, 431 with
// 32 Ki, 470 with 64 Ki
int chunk_of(long total) {
    int c = 2048;
    while (c < 16384 && total / c > 2048) c *= 2;
    return c;
}
long chunks_of(const long long* n, int count, int chunk) {
    long k = 0;
    for (int i = 0; i < count; ++i) k += (long)((n[i] + chunk - 1) / chunk);
    return k;
}
long total_of(const long long* n, int count) {
    long t = 0;
    for (int i = 0; i < count; ++i) t += (long)n[i];
    return t;
}

// the list cut into tables
template <bool APART>
std::vector<Table<APART>> tables(const unsigned long long* src, const unsigned long long* dst, const long long* n, const unsigned char* kind, int count,
                                 int chunk) {
    std::vector<Table<APART>> tabs;
    long chunks = 0;
    for (int i = 0; i < count; ++i)
        for (long o = 0; o < (long)n[i]; o += ENTRY) {
            if (tabs.empty() || tabs.back().count == Table<APART>::TAB || tabs.back().chunks > (1 << 24)) {
                tabs.emplace_back();
                Table<APART>& f = tabs.back();
                f.count = f.chunks = 0;
                f.chunk = chunk;
                f.base = (int)chunks;
            }
            Table<APART>& t = tabs.back();
            const long left = (long)n[i] - o, take = left < ENTRY ? left : ENTRY;
            t.src[t.count] = reinterpret_cast<const void*>(src[i] + (unsigned long long)o * (kind[i] & 1 ? 2 : 4));
            if constexpr (APART) t.dst[t.count] = reinterpret_cast<void*>(dst[i] + (unsigned long long)o * (kind[i] & 2 ? 2 : 4));
            t.n[t.count] = (unsigned)take;
            t.first[t.count] = t.chunks;
            t.kind[t.count++] = kind[i];
            const int k = (int)((take + chunk - 1) / chunk);
            t.chunks += k;
            chunks += k;
        }
    return tabs;
}

template <bool INF, bool APART>
int scale_all(const std::vector<Table<APART>>& tabs, const double* part, int parts, Limit l, float* out, hipStream_t s) {
    for (const Table<APART>& t : tabs) {
        clip_scale_kernel<INF, APART><<<t.chunks, NT, 0, s>>>(t, part, parts, l, out);
        LSAM_LAUNCH_CHECK();
    }
    return LSAM_OK;
}
template <bool INF>
int run(const std::vector<Table<false>>& read, const std::vector<Table<true>>& apart, bool scale, double* part, int parts, Limit l, float* out,
        hipStream_t s) {
    for (const Table<false>& t : read) {
        clip_norm_kernel<INF><<<t.chunks, NT, 0, s>>>(t, part);
        LSAM_LAUNCH_CHECK();
    }
    const bool self = scale && parts > 0 && parts <= SELF_JOIN;
    if (!self) {
        clip_join_kernel<INF><<<1, 1024, 0, s>>>(part, parts, l, out);
        LSAM_LAUNCH_CHECK();
    }
    if (!scale) return LSAM_OK;
    return apart.empty() ? scale_all<INF>(read, part, self ? parts : 0, l, out, s) : scale_all<INF>(apart, part, self ? parts : 0, l, out, s);
}
}  // namespace

size_t clip_ws_bytes(const long long* n, int count) {
    if (!n) return sizeof(double);
    const long k = chunks_of(n, count, chunk_of(total_of(n, count)));
    return (size_t)(k > 0 ? k : 1) * sizeof(double);
}

int launch_clip_grads(const unsigned long long* src, const unsigned long long* dst, const long long* n, const unsigned char* kind, int count,
                      double max_norm, int inf, double scale, float* out, void* ws, size_t ws_bytes, hipStream_t s) {
    LSAM_REQUIRE(count >= 0 && (count == 0 || (src && dst && n && kind)) && out && ws, LSAM_ERR_BAD_ARG, "clip_grads: null operand");
    LSAM_REQUIRE(max_norm >= 0. && scale == scale, LSAM_ERR_BAD_ARG, "clip_grads: max_norm %g, scale %g", max_norm, scale);
    LSAM_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 7) == 0, LSAM_ERR_BAD_ARG, "clip_grads: workspace off its 8-byte alignment");
    for (int i = 0; i < count; ++i) {
        LSAM_REQUIRE(n[i] >= 0 && kind[i] < 4, LSAM_ERR_BAD_ARG, "clip_grads: tensor %d: %lld elements, kind %d", i, n[i], kind[i]);
        LSAM_REQUIRE(n[i] == 0 || (src[i] && dst[i] && src[i] % (kind[i] & 1 ? 2 : 4) == 0 && dst[i] % (kind[i] & 2 ? 2 : 4) == 0), LSAM_ERR_BAD_ARG,
                     "clip_grads: tensor %d: null or misaligned", i);
    }
    LSAM_REQUIRE(clip_ws_bytes(n, count) <= ws_bytes, LSAM_ERR_WORKSPACE, "clip_grads: workspace too small");
    const bool scaled = !(max_norm == (double)INFINITY && scale == 1.) || !std::equal(src, src + count, dst);
    if (scaled) {
        // what is written may not be another tensor's (or, shifted, its own) input or output: workgroups would race
        struct Span { unsigned long long lo, hi; int i; };
        std::vector<Span> w;
        w.reserve(count);
        for (int i = 0; i < count; ++i)
            if (n[i]) w.push_back({dst[i], dst[i] + (unsigned long long)n[i] * (kind[i] & 2 ? 2 : 4), i});
        const auto below = [](const Span& a, const Span& b) { return a.lo < b.lo; };
        if (!std::is_sorted(w.begin(), w.end(), below)) std::sort(w.begin(), w.end(), below);
        for (size_t k = 1; k < w.size(); ++k)
            LSAM_REQUIRE(w[k].lo >= w[k - 1].hi, LSAM_ERR_BAD_ARG, "clip_grads: tensors %d and %d share memory", w[k - 1].i, w[k].i);
        for (int i = 0; i < count; ++i) {
            const bool same = src[i] == dst[i] && (kind[i] == 0 || kind[i] == 3);
            if (!n[i] || same) continue;
            const unsigned long long lo = src[i], hi = lo + (unsigned long long)n[i] * (kind[i] & 1 ? 2 : 4);
            auto it = std::upper_bound(w.begin(), w.end(), lo, [](unsigned long long v, const Span& a) { return v < a.hi; });
            LSAM_REQUIRE(it == w.end() || it->lo >= hi, LSAM_ERR_BAD_ARG, "clip_grads: tensor %d is written as tensor %d", i, it->i);
        }
    }
    const int chunk = chunk_of(total_of(n, count));
    const long chunks = chunks_of(n, count, chunk);
    LSAM_REQUIRE(chunks < (1l << 30), LSAM_ERR_UNSUPPORTED, "clip_grads: too many elements");
    bool apart = false;
    for (int i = 0; i < count; ++i) apart |= scaled && n[i] && (src[i] != dst[i] || (kind[i] != 0 && kind[i] != 3));
    const auto read = tables<false>(src, dst, n, kind, count, chunk);
    const auto other = apart ? tables<true>(src, dst, n, kind, count, chunk) : std::vector<Table<true>>();
    const Limit l{max_norm, scale};
    return inf ? run<true>(read, other, scaled, static_cast<double*>(ws), (int)chunks, l, out, s)
               : run<false>(read, other, scaled, static_cast<double*>(ws), (int)chunks, l, out, s);
}
}  // namespace lsam
