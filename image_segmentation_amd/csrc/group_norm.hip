// Group norm with an activation over channels-last maps, forward and backward.
//
//   xhat = (x - mean_ng) rstd_ng,  h = xhat gamma_c + beta_c,  y = act(h)          mean / variance over the P pixels x C/G channels
//   dh = dy act'(h),  dgamma_c = sum_np dh xhat,  dbeta_c = sum_np dh,
//   dx = rstd (gamma dh - (S1 + xhat S2) / m),  S1 = sum_group gamma dh,  S2 = sum_group gamma dh xhat,  m = P C/G
//
// Memory-bound both ways.  A workgroup walks a range of pixels with whole rows of channels: consecutive lanes take consecutive
// 16-byte pieces of a row, a thread keeps to its channels, so what a channel needs stays in its registers and the sums over pixels
// need no exchange until the range ends.  Sums over ranges are joined in a fixed order by the next kernel: same bits every time.
//
// Two passes each way: 3 reads and writes of the map forward, 5 backward, bound by HBM.  Measured on 16 x 256 x 256 x 256 bf16 with GELU
// (536 MB a map): statistics 124 us (4.3 TB/s), normalising 228 (4.7), the backward's sums 283 (3.8), its dx 342 (4.7); 900 us with the
// host's part, where a copy's 5.07 TB/s would allow 847 (plain form 14.3 ms).
#include "kernels.hpp"

namespace lsam {
namespace {
constexpr int NT = 256, MAXC = 8192;

// Thread layout over a row of C channels: `cw` threads side by side take V channels each, `rw` pixels at a time, in `blocks` column
// blocks when a row is wider than the workgroup.
struct Lay {
    int cols, cw, rw, blocks;
    __host__ __device__ Lay(int C, int V) {
        cols = C / V;
        blocks = (cols + NT - 1) / NT;
        cw = (cols + blocks - 1) / blocks;
        rw = NT / cw;
    }
};

template <typename T, int V> __device__ __forceinline__ void load(const T* p, float (&v)[V]) {
    if constexpr (V == 1) v[0] = to_f(*p);
    else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        T e[V];
        __builtin_memcpy(e, &u, 16);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_f(e[j]);
    }
}
template <typename T, int V> __device__ __forceinline__ void store(T* p, const float (&v)[V]) {
    if constexpr (V == 1) *p = from_f<T>(v[0]);
    else {
        T e[V];
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = from_f<T>(v[j]);
        uint4 u;
        __builtin_memcpy(&u, e, 16);
        *reinterpret_cast<uint4*>(p) = u;
    }
}

__device__ __forceinline__ float sigmoid(float h) { return __builtin_amdgcn_rcpf(1.f + __expf(-h)); }
// Phi(h), the normal distribution's, and e = exp(-h^2 / 2) by the way.  EXACT: erff, for fp32 results; else Abramowitz & Stegun 7.1.26
// (|error| < 1.5e-7), a polynomial in t = 1 / (1 + p |x|), x = h / sqrt 2, times that same exponential: half the instructions, and a map's
// pass with GELU is bound by them.  As a fraction of Phi the error passes half a step of bf16 (2^-9) below h = -5.2, where |h Phi| < 6e-7
// (0.4 % at -6, 1 % at -8, 4 % at -13, the last before the values leave the range).
template <bool EXACT> __device__ __forceinline__ float phi(float h, float& e) {
    e = __builtin_amdgcn_exp2f(h * h * -0.72134752044448170f);
    if constexpr (EXACT) return 0.5f * (1.f + erff(h * 0.70710678118654752f));
    const float t = __builtin_amdgcn_rcpf(fmaf(0.23164189f, fabsf(h), 1.f));
    float y = fmaf(0.5307027145f, t, -0.7265760135f);   // half of 7.1.26's coefficients
    y = fmaf(y, t, 0.7107068705f);
    y = fmaf(y, t, -0.142248368f);
    y = fmaf(y, t, 0.127414796f);
    y = y * t * e;
    return h < 0.f ? y : 1.f - y;
}
template <bool EXACT> __device__ __forceinline__ float act_fwd(int act, float h) {
    if (act == LSAM_ACT_RELU) return h < 0.f ? 0.f : h;
    if (act == LSAM_ACT_SILU) return h * sigmoid(h);
    if (act == LSAM_ACT_GELU) {
        float e;
        return h * phi<EXACT>(h, e);
    }
    return h;
}
template <bool EXACT> __device__ __forceinline__ float act_slope(int act, float h) {
    if (act == LSAM_ACT_RELU) return h <= 0.f ? 0.f : 1.f;
    if (act == LSAM_ACT_SILU) {
        const float q = sigmoid(h);
        return q * fmaf(h, 1.f - q, 1.f);
    }
    if (act == LSAM_ACT_GELU) {
        float e;
        const float f = phi<EXACT>(h, e);
        return fmaf(0.39894228040143268f * h, e, f);
    }
    return 1.f;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// Mean and M2 = sum (x - mean)^2 of `k` pieces with counts n_i, means m_i, M2_i, one wave: mean first, then the spread around it.
template <typename F> __device__ __forceinline__ void join(int k, int lane, F piece, float& mean, float& m2, float& count) {
    float n = 0.f, s = 0.f;
    for (int i = lane; i < k; i += 64) {
        float c, m, q;
        piece(i, c, m, q);
        n += c;
        s += c * m;
    }
    count = wave_sum(n);
    mean = wave_sum(s) / count;
    float v = 0.f;
    for (int i = lane; i < k; i += 64) {
        float c, m, q;
        piece(i, c, m, q);
        v += q + c * (m - mean) * (m - mean);
    }
    m2 = wave_sum(v);
}

struct GnArgs {
    const void* x; long sx, px;    // sample and pixel strides (elements)
    const void* dy; long sy, py;
    const float *gamma, *beta;     // or null: 1, 0
    int N, P, C, G, act, splits, rows;   // rows: pixels a split
    float eps;
    float* part;                   // fwd: [N][splits][G][2] (mean, M2); bwd: [N][splits][C][2] (sum dh, sum dh (x - mean))
    float* stats;                  // [N][G][2] mean, rstd
    float* chan;                   // bwd: [N][C][2] the sums over the splits, the second one times rstd: sum dh xhat
    float* coef;                   // bwd: [N][G][2] rstd S1 / m, rstd^2 S2 / m
    void* out;                     // [N][P][C]
    float *dgamma, *dbeta;
    int cb;                        // one-pass kernels: channels a workgroup
    bool keep;                     // fwd: stats are the caller's, not workspace
};

// per-range statistics.  A thread takes its first pixel as the pivot of its channels: sums of (x - pivot) and their squares cannot
// cancel by more than the number of its pixels, however far the mean is from zero.
template <typename T, int V>
__global__ __launch_bounds__(NT) void gn_stats_kernel(const GnArgs p) {
    extern __shared__ float sm[];              // mean[C], m2[C], then the threads' pieces
    float* cm = sm;
    float* cq = sm + p.C;
    float* tm = sm + 2 * p.C;
    float* tq = tm + NT * V;
    const Lay l(p.C, V);
    const int tid = threadIdx.x, tx = tid % l.cw, ty = tid / l.cw, lane = tid & 63;
    const int n = blockIdx.x / p.splits, sp = blockIdx.x - n * p.splits;
    const int p0 = sp * p.rows, p1 = min(p.P, p0 + p.rows), cnt = p1 - p0;
    const T* x = static_cast<const T*>(p.x) + n * p.sx;
    for (int b = 0; b < l.blocks; ++b) {
        const int col = b * l.cw + tx;
        const bool on = ty < l.rw && col < l.cols && p0 + ty < p1;
        float k[V], s[V], q[V];
        int mine = 0;
        if (on) {
            const T* xp = x + (long)(p0 + ty) * p.px + col * V;
            load<T, V>(xp, k);
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = q[j] = 0.f;
            mine = (cnt - ty + l.rw - 1) / l.rw;
            const long step = (long)l.rw * p.px;
#pragma unroll 4
            for (int i = 1; i < mine; ++i) {
                float v[V];
                load<T, V>(xp + i * step, v);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[j] - k[j];
                    s[j] += d;
                    q[j] = fmaf(d, d, q[j]);
                }
            }
        }
        if (b) __syncthreads();
        if (ty < l.rw) {
            const float inv = mine ? 1.f / (float)mine : 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                tm[(ty * l.cw + tx) * V + j] = on ? fmaf(s[j], inv, k[j]) : 0.f;
                tq[(ty * l.cw + tx) * V + j] = on ? fmaxf(0.f, q[j] - s[j] * s[j] * inv) : 0.f;
            }
        }
        __syncthreads();
        for (int c = tid; c < l.cw * V && b * l.cw * V + c < p.C; c += NT) {
            float sum = 0.f, spread = 0.f;
            for (int r = 0; r < l.rw && r < cnt; ++r) sum += tm[r * l.cw * V + c] * (float)((cnt - r + l.rw - 1) / l.rw);
            const float mean = sum / (float)cnt;
            for (int r = 0; r < l.rw && r < cnt; ++r) {
                const float d = tm[r * l.cw * V + c] - mean;
                spread += tq[r * l.cw * V + c] + d * d * (float)((cnt - r + l.rw - 1) / l.rw);
            }
            cm[b * l.cw * V + c] = mean;
            cq[b * l.cw * V + c] = spread;
        }
    }
    __syncthreads();
    const int cpg = p.C / p.G;
    auto put = [&](int g, float mean, float m2) {
        if (p.splits == 1) {   // the whole sample: done
            p.stats[((size_t)n * p.G + g) * 2] = mean;
            p.stats[((size_t)n * p.G + g) * 2 + 1] = 1.f / sqrtf(m2 / ((float)cnt * (float)cpg) + p.eps);
        } else {
            float* o = p.part + ((size_t)blockIdx.x * p.G + g) * 2;
            o[0] = mean;
            o[1] = m2;
        }
    };
    if (cpg <= 32) {   // a thread a group; a wave a group, one after another, costs more than the range's loads (16 x 64 x 64 x 256: 19 us)
        for (int g = tid; g < p.G; g += NT) {
            float mean = 0.f, m2 = 0.f;
            for (int c = 0; c < cpg; ++c) mean += cm[g * cpg + c];
            mean /= (float)cpg;
            for (int c = 0; c < cpg; ++c) {
                const float d = cm[g * cpg + c] - mean;
                m2 += fmaf((float)cnt * d, d, cq[g * cpg + c]);
            }
            put(g, mean, m2);
        }
    } else {
        for (int g = tid >> 6; g < p.G; g += NT / 64) {
            float mean, m2, count;
            join(cpg, lane, [&](int i, float& c, float& m, float& q) { c = (float)cnt; m = cm[g * cpg + i]; q = cq[g * cpg + i]; }, mean, m2, count);
            if (lane == 0) put(g, mean, m2);
        }
    }
}

// a wave a (sample, group): joins its ranges
__global__ __launch_bounds__(NT) void gn_join_kernel(const GnArgs p) {
    const int id = blockIdx.x * (NT / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (id >= p.N * p.G) return;
    const int n = id / p.G, g = id - n * p.G;
    const float cpg = (float)(p.C / p.G);
    float mean, m2, count;
    join(p.splits, lane, [&](int i, float& c, float& m, float& q) {
        const float* o = p.part + ((size_t)(n * p.splits + i) * p.G + g) * 2;
        c = (float)(min(p.P, (i + 1) * p.rows) - i * p.rows) * cpg;
        m = o[0];
        q = o[1];
    }, mean, m2, count);
    if (lane == 0) {
        p.stats[2 * (size_t)id] = mean;
        p.stats[2 * (size_t)id + 1] = 1.f / sqrtf(m2 / count + p.eps);
    }
}

// what a thread needs of its channels: h = (x - mean) slope + beta, slope = rstd gamma
template <int V> struct Chan {
    float mean[V], slope[V], beta[V];
    __device__ __forceinline__ void get(const GnArgs& p, int n, int c0) {
        const float* st = p.stats + (size_t)n * p.G * 2;
        const int cpg = p.C / p.G;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int g = (c0 + j) / cpg;
            mean[j] = st[2 * g];
            slope[j] = st[2 * g + 1] * (p.gamma ? p.gamma[c0 + j] : 1.f);
            beta[j] = p.beta ? p.beta[c0 + j] : 0.f;
        }
    }
};

template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_apply_kernel(const GnArgs p) {
    const Lay l(p.C, V);
    const int tid = threadIdx.x, tx = tid % l.cw, ty = tid / l.cw;
    const int n = blockIdx.x / p.splits, sp = blockIdx.x - n * p.splits;
    const int p0 = sp * p.rows, p1 = min(p.P, p0 + p.rows);
    const T* x = static_cast<const T*>(p.x) + n * p.sx;
    T* y = static_cast<T*>(p.out) + (size_t)n * p.P * p.C;
    for (int b = 0; b < l.blocks; ++b) {
        const int col = b * l.cw + tx;
        if (ty >= l.rw || col >= l.cols) continue;
        Chan<V> ch;
        ch.get(p, n, col * V);
#pragma unroll 4
        for (int i = p0 + ty; i < p1; i += l.rw) {
            float v[V];
            load<T, V>(x + (long)i * p.px + col * V, v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = act_fwd<sizeof(T) == 4>(ACT, fmaf(v[j] - ch.mean[j], ch.slope[j], ch.beta[j]));
            store<T, V>(y + (size_t)i * p.C + col * V, v);
        }
    }
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_bwd_sums_kernel(const GnArgs p) {
    extern __shared__ float sm[];
    const Lay l(p.C, V);
    const int tid = threadIdx.x, tx = tid % l.cw, ty = tid / l.cw;
    const int n = blockIdx.x / p.splits, sp = blockIdx.x - n * p.splits;
    const int p0 = sp * p.rows, p1 = min(p.P, p0 + p.rows);
    const T* x = static_cast<const T*>(p.x) + n * p.sx;
    const T* dy = static_cast<const T*>(p.dy) + n * p.sy;
    float *ta = sm, *tb = sm + NT * V;
    for (int b = 0; b < l.blocks; ++b) {
        const int col = b * l.cw + tx;
        float a[V], c[V];
#pragma unroll
        for (int j = 0; j < V; ++j) a[j] = c[j] = 0.f;
        if (ty < l.rw && col < l.cols) {
            Chan<V> ch;
            ch.get(p, n, col * V);
#pragma unroll 2
            for (int i = p0 + ty; i < p1; i += l.rw) {
                float v[V], d[V];
                load<T, V>(x + (long)i * p.px + col * V, v);
                load<T, V>(dy + (long)i * p.py + col * V, d);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = v[j] - ch.mean[j];
                    const float dh = d[j] * act_slope<sizeof(T) == 4>(ACT, fmaf(u, ch.slope[j], ch.beta[j]));
                    a[j] += dh;
                    c[j] = fmaf(dh, u, c[j]);
                }
            }
        }
        if (b) __syncthreads();
        if (ty < l.rw) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ta[(ty * l.cw + tx) * V + j] = a[j];
                tb[(ty * l.cw + tx) * V + j] = c[j];
            }
        }
        __syncthreads();
        for (int k = tid; k < l.cw * V && b * l.cw * V + k < p.C; k += NT) {
            float s = 0.f, t = 0.f;
            for (int r = 0; r < l.rw; ++r) {
                s += ta[r * l.cw * V + k];
                t += tb[r * l.cw * V + k];
            }
            float* o = p.part + ((size_t)blockIdx.x * p.C + b * l.cw * V + k) * 2;
            o[0] = s;
            o[1] = t;
        }
    }
}

// one workgroup a (sample, group): its channels' sums over the ranges, and the two group sums
__global__ __launch_bounds__(NT) void gn_bwd_join_kernel(const GnArgs p) {
    __shared__ float r1[NT / 64], r2[NT / 64];
    const int n = blockIdx.x / p.G, g = blockIdx.x - n * p.G, cpg = p.C / p.G, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float rstd = p.stats[2 * (size_t)blockIdx.x + 1];
    float s1 = 0.f, s2 = 0.f;
    for (int c = wave; c < cpg; c += NT / 64) {   // a wave a channel, lanes over the ranges
        const int ch = g * cpg + c;
        float a = 0.f, b = 0.f;
        for (int s = lane; s < p.splits; s += 64) {
            const float* o = p.part + ((size_t)(n * p.splits + s) * p.C + ch) * 2;
            a += o[0];
            b += o[1];
        }
        a = wave_sum(a);
        b = wave_sum(b) * rstd;
        if (lane == 0) {
            p.chan[((size_t)n * p.C + ch) * 2] = a;
            p.chan[((size_t)n * p.C + ch) * 2 + 1] = b;
        }
        const float gm = p.gamma ? p.gamma[ch] : 1.f;
        s1 = fmaf(gm, a, s1);
        s2 = fmaf(gm, b, s2);
    }
    if (lane == 0) { r1[wave] = s1; r2[wave] = s2; }
    __syncthreads();
    if (threadIdx.x == 0) {
        float a = 0.f, b = 0.f;
        for (int w = 0; w < NT / 64; ++w) { a += r1[w]; b += r2[w]; }
        const float m = (float)p.P * (float)cpg;
        p.coef[2 * (size_t)blockIdx.x] = rstd * a / m;
        p.coef[2 * (size_t)blockIdx.x + 1] = rstd * rstd * b / m;
    }
}

__device__ __forceinline__ void params(const GnArgs& p, int c) {   // dgamma, dbeta of channel c: the samples' sums, in their order
    if (c >= p.C) return;
    float a = 0.f, b = 0.f;
#pragma unroll 4
    for (int n = 0; n < p.N; ++n) {
        a += p.chan[((size_t)n * p.C + c) * 2];
        b += p.chan[((size_t)n * p.C + c) * 2 + 1];
    }
    if (p.dbeta) p.dbeta[c] = a;
    if (p.dgamma) p.dgamma[c] = b;
}
__global__ __launch_bounds__(NT) void gn_params_kernel(const GnArgs p) { params(p, blockIdx.x * NT + threadIdx.x); }

// the same over many samples (rows of features): 16 channels a workgroup, 64 threads a channel
constexpr int FEW_SAMPLES = 64;
__global__ __launch_bounds__(1024) void gn_params_many_kernel(const GnArgs p) {
    __shared__ float2 sh[64][16];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
    float2 s = make_float2(0.f, 0.f);
    if (c < p.C) {
#pragma unroll 8
        for (int n = y; n < p.N; n += 64) {
            const float2 v = *reinterpret_cast<const float2*>(p.chan + ((size_t)n * p.C + c) * 2);
            s.x += v.x;
            s.y += v.y;
        }
    }
    sh[y][x] = s;
    for (int h = 32; h; h >>= 1) {
        __syncthreads();
        if (y < h) {
            sh[y][x].x += sh[y + h][x].x;
            sh[y][x].y += sh[y + h][x].y;
        }
    }
    if (y || c >= p.C) return;
    if (p.dbeta) p.dbeta[c] = sh[0][x].x;
    if (p.dgamma) p.dgamma[c] = sh[0][x].y;
}
int sum_params(const GnArgs& p, hipStream_t s) {
    if (!p.dgamma && !p.dbeta) return LSAM_OK;
    // 300,000 rows of 256: 1.1 ms, 35.7 with a thread a channel
    if (p.N > FEW_SAMPLES) gn_params_many_kernel<<<cdiv(p.C, 16), 1024, 0, s>>>(p);
    else gn_params_kernel<<<cdiv(p.C, NT), NT, 0, s>>>(p);
    LSAM_LAUNCH_CHECK();
    return LSAM_OK;
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(NT) void gn_bwd_apply_kernel(const GnArgs p) {
    const int tid = threadIdx.x;
    if ((int)blockIdx.x >= p.N * p.splits) {   // the workgroups behind the maps'
        params(p, ((int)blockIdx.x - p.N * p.splits) * NT + tid);
        return;
    }
    const Lay l(p.C, V);
    const int tx = tid % l.cw, ty = tid / l.cw, cpg = p.C / p.G;
    const int n = blockIdx.x / p.splits, sp = blockIdx.x - n * p.splits;
    const int p0 = sp * p.rows, p1 = min(p.P, p0 + p.rows);
    const T* x = static_cast<const T*>(p.x) + n * p.sx;
    const T* dy = static_cast<const T*>(p.dy) + n * p.sy;
    T* dx = static_cast<T*>(p.out) + (size_t)n * p.P * p.C;
    for (int b = 0; b < l.blocks; ++b) {
        const int col = b * l.cw + tx;
        if (ty >= l.rw || col >= l.cols) continue;
        Chan<V> ch;
        ch.get(p, n, col * V);
        float c1[V], c2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float* o = p.coef + ((size_t)n * p.G + (col * V + j) / cpg) * 2;
            c1[j] = o[0];
            c2[j] = o[1];
        }
#pragma unroll 2
        for (int i = p0 + ty; i < p1; i += l.rw) {
            float v[V], d[V];
            load<T, V>(x + (long)i * p.px + col * V, v);
            load<T, V>(dy + (long)i * p.py + col * V, d);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float u = v[j] - ch.mean[j];
                const float dh = d[j] * act_slope<sizeof(T) == 4>(ACT, fmaf(u, ch.slope[j], ch.beta[j]));
                v[j] = fmaf(dh, ch.slope[j], -fmaf(u, c2[j], c1[j]));
            }
            store<T, V>(dx + (size_t)i * p.C + col * V, v);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// One pass: where a sample's pixels times a block of whole groups fit a workgroup's registers (1024 threads x UMAX pieces), x (and dy)
// are read once, the sums go through LDS, and the result is formed from the registers.  One launch where the passes above take three:
// these sizes are bound by launches, not by bytes.  Neighbouring blocks of a sample, which share cache lines, run on one XCD.
// 16 x 64 x 64 x 256 bf16 forward: 22 us, 33 by the passes above; 4 x 43 x 57 x 105 fp32 forward and backward: 120 to 124 us, kernels 39.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int ST = 1024;

// column sums of a[rows][cols] into a[0][*]: halving, a fixed order
__device__ __forceinline__ void fold(float* a, int rows, int cols) {
    for (int n = rows; n > 1;) {
        const int h = (n + 1) / 2;
        for (int i = threadIdx.x; i < (n - h) * cols; i += ST) a[i] += a[i + h * cols];
        __syncthreads();
        n = h;
    }
}

// put(g, sum of f(c) over the cpg channels c of group g) for the groups 0 .. gb: a thread a group, a wave where it has many channels (1024 summed
// by one thread: the sum off by 7 units of its last place, by 0.5 in a wave)
template <typename F, typename P> __device__ __forceinline__ void group_sums(int gb, int cpg, F f, P put) {
    if (cpg <= 32) {
        for (int g = threadIdx.x; g < gb; g += ST) {
            float a = 0.f;
            for (int c = 0; c < cpg; ++c) a += f(g * cpg + c);
            put(g, a);
        }
    } else {
        for (int g = threadIdx.x >> 6; g < gb; g += ST / 64) {
            float a = 0.f;
            for (int c = threadIdx.x & 63; c < cpg; c += 64) a += f(g * cpg + c);
            a = wave_sum(a);
            if ((threadIdx.x & 63) == 0) put(g, a);
        }
    }
}

template <typename T, int V> struct Piece { using type = uint4; };
template <> struct Piece<float, 1> { using type = float; };
template <> struct Piece<bf16, 1> { using type = bf16; };
template <typename T, int V> __device__ __forceinline__ void widen(const typename Piece<T, V>::type& r, float (&v)[V]) {
    T e[V];
    __builtin_memcpy(e, &r, sizeof(e));
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_f(e[j]);
}

template <typename T, int V, int UMAX, int ACT> __global__ __launch_bounds__(ST) void gn_one_fwd_kernel(const GnArgs p) {
    extern __shared__ float sm[];   // [rw][cb] sums, then [cb / cpg][2] mean, rstd
    using R = typename Piece<T, V>::type;
    const int cw = p.cb / V, rw = ST / cw, tid = threadIdx.x, tx = tid % cw, ty = tid / cw, cpg = p.C / p.G, gb = p.cb / cpg;
    const int rows = min(rw, p.P);   // thread rows that have a pixel
    const int blocks = p.C / p.cb, id = xcd_remap(blockIdx.x, gridDim.x), n = id / blocks, c0 = (id - n * blocks) * p.cb;
    float* grp = sm + ST * V;
    const T* x = static_cast<const T*>(p.x) + n * p.sx + c0 + tx * V;
    const int mine = ty < rw && ty < p.P ? (p.P - ty + rw - 1) / rw : 0;
    R r[UMAX];
#pragma unroll
    for (int u = 0; u < UMAX; ++u)
        if (u < mine) r[u] = *reinterpret_cast<const R*>(x + (long)(ty + u * rw) * p.px);
    float s[V], m[V], v[V];
    auto total = [&](auto f) {   // sum of f over this thread's pixels, a channel each, and over the workgroup's
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = 0.f;
#pragma unroll
        for (int u = 0; u < UMAX; ++u)
            if (u < mine) {
                widen<T, V>(r[u], v);
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] += f(v[j], j);
            }
        if (ty < rows) {
#pragma unroll
            for (int j = 0; j < V; ++j) sm[tid * V + j] = s[j];
        }
        __syncthreads();
        fold(sm, rows, p.cb);
    };
    const float cnt = (float)p.P * (float)cpg;
    total([](float a, int) { return a; });
    auto sum = [&](int c) { return sm[c]; };
    group_sums(gb, cpg, sum, [&](int g, float a) { grp[2 * g] = a / cnt; });
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) m[j] = grp[2 * ((tx * V + j) / cpg)];
    total([&](float a, int j) { return (a - m[j]) * (a - m[j]); });
    group_sums(gb, cpg, sum, [&](int g, float a) {
        const float rstd = 1.f / sqrtf(a / cnt + p.eps);
        grp[2 * g + 1] = rstd;
        if (p.stats) {
            float* o = p.stats + ((size_t)n * p.G + c0 / cpg + g) * 2;
            o[0] = grp[2 * g];
            o[1] = rstd;
        }
    });
    __syncthreads();
    if (!mine) return;
    float sl[V], be[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = tx * V + j;
        sl[j] = grp[2 * (c / cpg) + 1] * (p.gamma ? p.gamma[c0 + c] : 1.f);
        be[j] = p.beta ? p.beta[c0 + c] : 0.f;
    }
    T* y = static_cast<T*>(p.out) + (size_t)n * p.P * p.C + c0 + tx * V;
#pragma unroll
    for (int u = 0; u < UMAX; ++u)
        if (u < mine) {
            widen<T, V>(r[u], v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = act_fwd<sizeof(T) == 4>(ACT, fmaf(v[j] - m[j], sl[j], be[j]));
            store<T, V>(y + (size_t)(ty + u * rw) * p.C, v);
        }
}

template <typename T, int V, int UMAX, int ACT> __global__ __launch_bounds__(ST) void gn_one_bwd_kernel(const GnArgs p) {
    extern __shared__ float sm[];   // [rw][cb] sums of dh, then of dh (x - mean); [cb] the first ones' result; [cb / cpg][2] coefficients
    using R = typename Piece<T, V>::type;
    const int cw = p.cb / V, rw = ST / cw, tid = threadIdx.x, tx = tid % cw, ty = tid / cw, cpg = p.C / p.G, gb = p.cb / cpg;
    const int rows = min(rw, p.P);   // thread rows that have a pixel
    const int blocks = p.C / p.cb, id = xcd_remap(blockIdx.x, gridDim.x), n = id / blocks, c0 = (id - n * blocks) * p.cb;
    float *sa = sm + ST * V, *grp = sa + p.cb;
    const T* x = static_cast<const T*>(p.x) + n * p.sx + c0 + tx * V;
    const T* dy = static_cast<const T*>(p.dy) + n * p.sy + c0 + tx * V;
    const int mine = ty < rw && ty < p.P ? (p.P - ty + rw - 1) / rw : 0;
    R r[UMAX], q[UMAX];
#pragma unroll
    for (int u = 0; u < UMAX; ++u)
        if (u < mine) {
            r[u] = *reinterpret_cast<const R*>(x + (long)(ty + u * rw) * p.px);
            q[u] = *reinterpret_cast<const R*>(dy + (long)(ty + u * rw) * p.py);
        }
    Chan<V> ch;
    ch.get(p, n, c0 + tx * V);
    float a[V], b[V], v[V], d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = b[j] = 0.f;
#pragma unroll
    for (int u = 0; u < UMAX; ++u)
        if (u < mine) {
            widen<T, V>(r[u], v);
            widen<T, V>(q[u], d);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float w = v[j] - ch.mean[j];
                const float dh = d[j] * act_slope<sizeof(T) == 4>(ACT, fmaf(w, ch.slope[j], ch.beta[j]));
                a[j] += dh;
                b[j] = fmaf(dh, w, b[j]);
            }
        }
    if (ty < rows) {
#pragma unroll
        for (int j = 0; j < V; ++j) sm[tid * V + j] = a[j];
    }
    __syncthreads();
    fold(sm, rows, p.cb);
    for (int c = tid; c < p.cb; c += ST) sa[c] = sm[c];
    __syncthreads();
    if (ty < rows) {
#pragma unroll
        for (int j = 0; j < V; ++j) sm[tid * V + j] = b[j];
    }
    __syncthreads();
    fold(sm, rows, p.cb);
    const float m = (float)p.P * (float)cpg;
    const float* st = p.stats + ((size_t)n * p.G + c0 / cpg) * 2;
    for (int c = tid; c < p.cb; c += ST) {
        const float t = sm[c] * st[2 * (c / cpg) + 1];
        if (p.N == 1) {
            if (p.dbeta) p.dbeta[c0 + c] = sa[c];
            if (p.dgamma) p.dgamma[c0 + c] = t;
        } else {
            float* o = p.chan + ((size_t)n * p.C + c0 + c) * 2;
            o[0] = sa[c];
            o[1] = t;
        }
    }
    auto gamma = [&](int c) { return p.gamma ? p.gamma[c0 + c] : 1.f; };
    group_sums(gb, cpg, [&](int c) { return gamma(c) * sa[c]; }, [&](int g, float a) { grp[2 * g] = st[2 * g + 1] * a / m; });
    group_sums(gb, cpg, [&](int c) { return gamma(c) * sm[c]; }, [&](int g, float a) { grp[2 * g + 1] = st[2 * g + 1] * st[2 * g + 1] * (st[2 * g + 1] * a) / m; });
    __syncthreads();
    if (!mine || !p.out) return;   // no map wanted: the parameters' sums were all
    float c1[V], c2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        c1[j] = grp[2 * ((tx * V + j) / cpg)];
        c2[j] = grp[2 * ((tx * V + j) / cpg) + 1];
    }
    T* dx = static_cast<T*>(p.out) + (size_t)n * p.P * p.C + c0 + tx * V;
#pragma unroll
    for (int u = 0; u < UMAX; ++u)
        if (u < mine) {
            widen<T, V>(r[u], v);
            widen<T, V>(q[u], d);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float w = v[j] - ch.mean[j];
                const float dh = d[j] * act_slope<sizeof(T) == 4>(ACT, fmaf(w, ch.slope[j], ch.beta[j]));
                v[j] = fmaf(dh, ch.slope[j], -fmaf(w, c2[j], c1[j]));
            }
            store<T, V>(dx + (size_t)(ty + u * rw) * p.C, v);
        }
}

// channels a workgroup of the one-pass kernels, 0 where they do not apply: the fewest whole groups that make whole pieces and 32 bytes of a
// pixel, or 16 where that is too much for `umax` pieces a thread; more of them where the launch would come to 2^32 threads, which the
// runtime cuts short without an error (rows of features: 262,144 samples of 256 channels)
int one_pass(const GnArgs& p, int V, int esz, int umax) {
    const int cpg = p.C / p.G;
    for (int least : {32, 16}) {
        int cb = cpg;
        while (cb < p.C && (p.C % cb || cb % V || cb * esz < least || (long)p.N * (p.C / cb) >= (1l << 32) / ST)) cb += cpg;
        if (cb % V || cb / V > ST) return 0;
        if (cdiv(p.P, ST / (cb / V)) <= umax) return cb;
    }
    return 0;
}

// pixels a range: enough ranges for `wgs` workgroups a compute unit, at least eight pixels a thread where there are that many
void ranges(GnArgs& p, int V, int wgs) {
    const Lay l(p.C, V);
    int s = (wgs * 256 + p.N - 1) / p.N;
    const int most = cdiv(p.P, l.rw * 8);
    if (s > most) s = most;
    if (s < 1) s = 1;
    p.rows = cdiv(cdiv(p.P, s), l.rw) * l.rw;
    p.splits = cdiv(p.P, p.rows);
}
// measured on 16 x 256 x 256 x 256 bf16, GELU: the statistics 128 us with 4, 155 with 8, 169 with 2; normalising 241 us with 4, 224 with
// 8; the backward's sums 286 and 279, its dx 350 and 336
constexpr int WG_STATS = 4, WG_REST = 8;
int vec_of(int esz, const GnArgs& p, bool with_dy) {
    const int V = 16 / esz;
    const bool ok = p.C % V == 0 && p.px % V == 0 && p.sx % V == 0 && aligned16(p.x) && (!p.out || aligned16(p.out)) &&
                    (!with_dy || (p.py % V == 0 && p.sy % V == 0 && aligned16(p.dy)));
    return ok ? V : 1;
}
template <typename T, int V> int run_fwd(GnArgs& p, hipStream_t s) {
    constexpr int UF = V == 8 ? 8 : V > 1 ? 16 : 32;   // what 128 registers hold without spilling
    p.cb = one_pass(p, V, sizeof(T), UF);
    if (p.cb) {
        if (!p.keep) p.stats = nullptr;
        auto k = p.act == LSAM_ACT_RELU   ? gn_one_fwd_kernel<T, V, UF, LSAM_ACT_RELU>
                 : p.act == LSAM_ACT_SILU ? gn_one_fwd_kernel<T, V, UF, LSAM_ACT_SILU>
                 : p.act == LSAM_ACT_GELU ? gn_one_fwd_kernel<T, V, UF, LSAM_ACT_GELU>
                                          : gn_one_fwd_kernel<T, V, UF, LSAM_ACT_NONE>;
        k<<<p.N * (p.C / p.cb), ST, (ST * V + 2 * p.cb) * sizeof(float), s>>>(p);
        LSAM_LAUNCH_CHECK();
        return LSAM_OK;
    }
    ranges(p, V, WG_STATS);
    gn_stats_kernel<T, V><<<p.N * p.splits, NT, (2 * p.C + 2 * NT * V) * sizeof(float), s>>>(p);
    LSAM_LAUNCH_CHECK();
    if (p.splits > 1) {
        gn_join_kernel<<<cdiv(p.N * p.G, NT / 64), NT, 0, s>>>(p);
        LSAM_LAUNCH_CHECK();
    }
    ranges(p, V, WG_REST);
    auto k = p.act == LSAM_ACT_RELU   ? gn_apply_kernel<T, V, LSAM_ACT_RELU>
             : p.act == LSAM_ACT_SILU ? gn_apply_kernel<T, V, LSAM_ACT_SILU>
             : p.act == LSAM_ACT_GELU ? gn_apply_kernel<T, V, LSAM_ACT_GELU>
                                      : gn_apply_kernel<T, V, LSAM_ACT_NONE>;
    k<<<p.N * p.splits, NT, 0, s>>>(p);
    LSAM_LAUNCH_CHECK();
    return LSAM_OK;
}
template <typename T, int V> int run_bwd(GnArgs& p, hipStream_t s) {
    constexpr int UB = V == 8 ? 4 : V > 1 ? 8 : 32;
    p.cb = one_pass(p, V, sizeof(T), UB);
    if (p.cb) {
        auto k = p.act == LSAM_ACT_RELU   ? gn_one_bwd_kernel<T, V, UB, LSAM_ACT_RELU>
                 : p.act == LSAM_ACT_SILU ? gn_one_bwd_kernel<T, V, UB, LSAM_ACT_SILU>
                 : p.act == LSAM_ACT_GELU ? gn_one_bwd_kernel<T, V, UB, LSAM_ACT_GELU>
                                          : gn_one_bwd_kernel<T, V, UB, LSAM_ACT_NONE>;
        k<<<p.N * (p.C / p.cb), ST, (ST * V + 3 * p.cb) * sizeof(float), s>>>(p);
        LSAM_LAUNCH_CHECK();
        return p.N > 1 ? sum_params(p, s) : LSAM_OK;
    }
    ranges(p, V, WG_REST);
    auto k = p.act == LSAM_ACT_RELU   ? gn_bwd_sums_kernel<T, V, LSAM_ACT_RELU>
             : p.act == LSAM_ACT_SILU ? gn_bwd_sums_kernel<T, V, LSAM_ACT_SILU>
             : p.act == LSAM_ACT_GELU ? gn_bwd_sums_kernel<T, V, LSAM_ACT_GELU>
                                      : gn_bwd_sums_kernel<T, V, LSAM_ACT_NONE>;
    k<<<p.N * p.splits, NT, 2 * NT * V * sizeof(float), s>>>(p);
    LSAM_LAUNCH_CHECK();
    gn_bwd_join_kernel<<<p.N * p.G, NT, 0, s>>>(p);
    LSAM_LAUNCH_CHECK();
    if (!p.out) return sum_params(p, s);   // 16 x 256 x 256 x 256 bf16: the second pass is more than half of the backward
    if (p.N > FEW_SAMPLES) LSAM_TRY(sum_params(p, s));
    auto a = p.act == LSAM_ACT_RELU   ? gn_bwd_apply_kernel<T, V, LSAM_ACT_RELU>
             : p.act == LSAM_ACT_SILU ? gn_bwd_apply_kernel<T, V, LSAM_ACT_SILU>
             : p.act == LSAM_ACT_GELU ? gn_bwd_apply_kernel<T, V, LSAM_ACT_GELU>
                                      : gn_bwd_apply_kernel<T, V, LSAM_ACT_NONE>;
    a<<<p.N * p.splits + (p.N > FEW_SAMPLES ? 0 : cdiv(p.C, NT)), NT, 0, s>>>(p);
    LSAM_LAUNCH_CHECK();
    return LSAM_OK;
}

int gn_check(int N, int P, int C, int G, int act, long sx, long px) {
    LSAM_REQUIRE(N >= 0 && P >= 0 && C > 0 && G > 0 && C % G == 0, LSAM_ERR_BAD_ARG,
                 "group_norm_act: %d samples, %d pixels, %d channels in %d groups", N, P, C, G);
    LSAM_REQUIRE(C <= MAXC && (long)N * G < (1l << 24) && N < (1 << 20) && P < (1 << 30), LSAM_ERR_UNSUPPORTED,
                 "group_norm_act: %d samples, %d pixels, %d channels, %d groups", N, P, C, G);
    LSAM_REQUIRE(act >= LSAM_ACT_NONE && act <= LSAM_ACT_GELU, LSAM_ERR_BAD_ARG, "group_norm_act: activation %d", act);
    LSAM_REQUIRE(px >= 0 && sx >= 0, LSAM_ERR_BAD_ARG, "group_norm_act: strides %ld, %ld", sx, px);
    return LSAM_OK;
}
}  // namespace

// what ranges() may come to in any layout: at most 2048 / N + 1 ranges a sample, and P / 8 of them
size_t gn_ws_bytes(int N, int P, int C, int G, int backward) {
    const size_t n = N > 0 ? N : 1;
    size_t split_rows = n + WG_REST * 256;
    const size_t most = n * (size_t)(P > 0 ? cdiv(P, 8) : 1);
    if (split_rows > most) split_rows = most;
    return (backward ? split_rows * C * 2 + n * C * 2 + n * G * 2 : split_rows * G * 2 + n * G * 2) * sizeof(float);
}

template <typename T>
int launch_group_norm_act_fwd(const void* x, long sx, long px, const float* gamma, const float* beta, int N, int P, int C, int G, float eps, int act,
                              void* y, float* stats, void* ws, size_t ws_bytes, hipStream_t s) {
    LSAM_TRY(gn_check(N, P, C, G, act, sx, px));
    if (N == 0 || P == 0) return LSAM_OK;
    LSAM_REQUIRE(x && y && ws && aligned16(ws), LSAM_ERR_BAD_ARG, "group_norm_act: null operand or workspace off its 16-byte alignment");
    LSAM_REQUIRE(ws_bytes >= gn_ws_bytes(N, P, C, G, 0), LSAM_ERR_WORKSPACE, "group_norm_act: workspace too small");
    GnArgs p{};
    p.x = x; p.sx = sx; p.px = px; p.gamma = gamma; p.beta = beta; p.N = N; p.P = P; p.C = C; p.G = G; p.act = act; p.eps = eps;
    p.keep = stats != nullptr;
    p.stats = stats ? stats : static_cast<float*>(ws);
    p.part = static_cast<float*>(ws) + (size_t)N * G * 2;
    p.out = y;
    const int V = vec_of(sizeof(T), p, false);
    return V > 1 ? run_fwd<T, 16 / sizeof(T)>(p, s) : run_fwd<T, 1>(p, s);
}

template <typename T>
int launch_group_norm_act_bwd(const void* dy, long sy, long py, const void* x, long sx, long px, const float* gamma, const float* beta,
                              const float* stats, int N, int P, int C, int G, int act, bool want_dx, void* dx, float* dgamma, float* dbeta,
                              void* ws, size_t ws_bytes, hipStream_t s) {
    LSAM_TRY(gn_check(N, P, C, G, act, sx, px));
    LSAM_TRY(gn_check(N, P, C, G, act, sy, py));
    GnArgs p{};
    p.N = N; p.P = P; p.C = C; p.G = G; p.act = act;
    LSAM_REQUIRE(ws && aligned16(ws), LSAM_ERR_BAD_ARG, "group_norm_act: null workspace or off its 16-byte alignment");
    LSAM_REQUIRE(ws_bytes >= gn_ws_bytes(N, P, C, G, 1), LSAM_ERR_WORKSPACE, "group_norm_act: workspace too small");
    p.x = x; p.sx = sx; p.px = px; p.dy = dy; p.sy = sy; p.py = py; p.gamma = gamma; p.beta = beta; p.stats = const_cast<float*>(stats);
    p.out = want_dx ? dx : nullptr; p.dgamma = dgamma; p.dbeta = dbeta;
    if (!want_dx && !dgamma && !dbeta) return LSAM_OK;
    p.chan = static_cast<float*>(ws);
    p.coef = p.chan + (size_t)(N > 0 ? N : 1) * C * 2;
    p.part = p.coef + (size_t)(N > 0 ? N : 1) * G * 2;
    if (N == 0 || P == 0) {   // nothing but zero sums: the workgroups behind no maps
        p.N = 0;
        p.splits = 1;
        gn_bwd_apply_kernel<T, 1, LSAM_ACT_NONE><<<cdiv(C, NT), NT, 0, s>>>(p);
        LSAM_LAUNCH_CHECK();
        return LSAM_OK;
    }
    LSAM_REQUIRE(x && dy && (dx || !want_dx) && stats, LSAM_ERR_BAD_ARG, "group_norm_act: null operand");
    const int V = vec_of(sizeof(T), p, true);
    return V > 1 ? run_bwd<T, 16 / sizeof(T)>(p, s) : run_bwd<T, 1>(p, s);
}
#define GN_INST(T)                                                                                                                              \
    template int launch_group_norm_act_fwd<T>(const void*, long, long, const float*, const float*, int, int, int, int, float, int, void*,       \
                                              float*, void*, size_t, hipStream_t);                                                             \
    template int launch_group_norm_act_bwd<T>(const void*, long, long, const void*, long, long, const float*, const float*, const float*, int,  \
                                              int, int, int, int, bool, void*, float*, float*, void*, size_t, hipStream_t);
GN_INST(float)
GN_INST(bf16)
}  // namespace lsam
