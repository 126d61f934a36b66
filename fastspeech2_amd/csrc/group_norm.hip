// Group norm of packed ragged rows with an activation, and its backward.  Utterance b owns rows cu[b] .. cu[b + 1] of
// x [M, C] (channels last); mean and variance are taken over (its rows) x (the C / G channels of a group):
//   xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps);  y = dropout(act(gamma xhat + beta))
//   dz = dropout(dy) act'(gamma xhat + beta),  dh = gamma dz
//   dx = rstd (dh - mean_g(dh) - xhat mean_g(dh xhat));  dgamma = sum dz xhat,  dbeta = sum dz
// Unlike BatchNorm (batchnorm.hip) no utterance sees another: a batch row equals the utterance alone.
//
// Memory-bound: the floor is one read of the inputs and one write of the output.  A workgroup owns a STRIP of whole groups (at least
// GN_STRIP_BYTES of a row) of one utterance and holds its rows in REGISTERS: it reads them once, takes the mean, then the centred
// squares (two passes over registers, no cancellation), and writes.  An utterance too long for the registers is cut into chunks: a first
// kernel leaves (mean, centred squares) of every chunk, or the backward's sums; behind the join of these a last one reads the rows again and applies.
// Chunks merge by M2 = sum M2_i + n_i (mean_i - mean)^2 in a fixed order; no atomics.
//
// Measured, 32 utterances x 800 rows x 256 channels in 16 groups, tanh: forward fp32 -> bf16 14.5 us for 39 MB (2.7 TB/s); backward
// 19.2 us for 65 MB (3.4 TB/s), 3.9 of it the sums of dgamma and dbeta; 256 x 800 x 80, bf16 backward: 34.9 us for 97 MB (2.8 TB/s).
// What is left: all workgroups read, reduce and write at the same time, so the memory waits while they reduce (of the 34 us of the
// last, 15 are the read at 4.2 TB/s, 4 the sums, 15 the write).  Activation and dropout are chosen by the vector of values: by the
// value, with its branches, the three took 15.4, 22.5 and 47.4 us.
#include "common.h"

namespace fs2 {

// Threads of a workgroup: 512 where it holds a whole utterance's strip, 256 where it streams a chunk: small groups overlap each other's
// phases (64 x 6000 rows x 80 channels, bf16 backward 85 us with 256 and 93 with 512 threads; 32 x 6000 x 256 fp32 forward 149 and 165; one
// utterance of 6000 13.3 and 15.1; all with the chunks joined by a launch of its own).
constexpr int GN_WHOLE_THREADS = 512, GN_CHUNK_THREADS = 256;
constexpr int GN_CHUNK_ROWS = 8;          // rows per thread of a chunk
constexpr int GN_HOLD = 4;                // rows per thread in registers at a time, in a chunk
constexpr int GN_STRIP_BYTES = 64;        // 32 x 800 rows x 256 channels, fp32: forward 16.0 us (128: 18.2), one utterance 9.0 (12.8)

struct GnArgs {
    const void* x;           // [M, ldx]
    const int* cu;           // [B + 1]
    const float* gamma;
    const float* beta;
    void* out;               // [M, ldo]
    float* stats;            // [B][G][2] mean, rstd
    const void* dout;        // [M, ldd]
    void* dx;                // [M, ldg]
    float* part;             // forward chunks: [B][nchunk][G][2] mean, M2; backward: [B][nchunk][2][C] sums of dz, dz xhat
    float* gpart;            // backward chunks: [B][nchunk][G][2] sums of dh, dh xhat
    float* gsum;             // backward of chunked utterances: [B][G][2] means of the same
    int M, max_len, C, G, cg, ldx, ldo, ldd, ldg, act, nchunk, nstrip;
    int units;               // B * nchunk
    int W, LX, LY;           // channels of a strip, lanes per row, rows per pass of the workgroup
    float inv_lx, inv_cg;    // 1 / LX, 1 / cg
    float eps;
    Dropout drop;
};

// ---- activations: 0 none, 1 ReLU, 2 tanh, 3 SiLU -------------------------------------------------------------------
// tanh z = z P(z^2) / Q(z^2), P and Q of degree 4 fitted to 0.1 u of it for |z| <= 8 (u = 2^-24; beyond, where 1 - tanh < 4 u, z^2 stays at 64 and
// the quotient is cut at 1): 7 u with the rounding, in as many operations as 1 - 2 / (1 + e^2z), which keeps no relative accuracy near 0.
// Slopes and sigmoid from e = exp(-2|z|) or exp(-|z|) <= 1 and one reciprocal: nothing overflows, and they keep their relative accuracy
// where the activation saturates: tanh' = 4 e / (1 + e)^2 to (4 |z| + 10) u; sigmoid to 8 u of either sign, the exponent's own rounding
// added back, and silu to 9 u.
__device__ __forceinline__ float gn_tanh(float z) {
    const float u = fminf(z * z, 64.0f);
    float p = fmaf(1.523053150265241e-8f, u, 2.1894744349992834e-5f), q = fmaf(8.522493430973554e-7f, u, 3.411300422158092e-4f);
    p = fmaf(fmaf(fmaf(p, u, 3.571603214368224e-3f), u, 0.13444502651691437f), u, 1.0f);
    q = fmaf(fmaf(fmaf(q, u, 2.616446278989315e-2f), u, 0.4677782952785492f), u, 1.0f);
    const float t = z * p * __builtin_amdgcn_rcpf(q);
    return __builtin_elementwise_maximum(__builtin_elementwise_minimum(t, 1.0f), -1.0f);         // (these keep a NaN)
}
__device__ __forceinline__ float gn_tanh_slope(float z) {
    const float e = __builtin_amdgcn_exp2f(fabsf(z) * -2.8853900817779268f), r = __builtin_amdgcn_rcpf(1.0f + e);
    return 4.0f * e * (r * r);
}
// sigmoid(z) and sigmoid(-z)
__device__ __forceinline__ void gn_sigmoid(float z, float& s, float& other) {
    const float a = fminf(fabsf(z), 128.0f), x = a * -1.4426950408889634f;            // (e is 0 from 104 on)
    float e = __builtin_amdgcn_exp2f(x);
    // a log2(e) - what x has of it, its rounding and the constant's: log2(e) = 1.44269502162933 + 1.92596e-8
    e = fmaf(e, fmaf(a, -1.3349758e-8f, fmaf(a, -1.4426950408889634f, -x) * 0.6931471805599453f), e);
    const float r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    s = z >= 0.f ? r : er;
    other = z >= 0.f ? er : r;
}
// act of V values, or act' times u: one (uniform) branch for the vector
template <int V> __device__ __forceinline__ void gn_act(int act, float (&z)[V]) {
    if (act == 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = z[j] > 0.f ? z[j] : (z[j] == z[j] ? 0.f : z[j]);
    } else if (act == 2) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = gn_tanh(z[j]);
    } else if (act == 3) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float g, h;
            gn_sigmoid(z[j], g, h);
            z[j] = z[j] == -INFINITY ? 0.f : z[j] * g;
        }
    }
}
template <int V> __device__ __forceinline__ void gn_slope(int act, const float (&z)[V], float (&u)[V]) {
    if (act == 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = z[j] > 0.f ? u[j] : u[j] * 0.f;
    } else if (act == 2) {
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] *= gn_tanh_slope(z[j]);
    } else if (act == 3) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float g, h;
            gn_sigmoid(z[j], g, h);
            u[j] *= g * fmaf(z[j], h, 1.0f);
        }
    }
}
template <int V> __device__ __forceinline__ void gn_drop(const Dropout& drop, int row, int c0, float (&z)[V]) {
    if (drop.thresh) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] *= drop_mul(drop, (uint32_t)row, (uint32_t)(c0 + j));
    }
}

// ---- V consecutive channels of a row: raw registers and their values ---------------------------------------------------
template <typename T, int V> struct GnVec {
    uint32_t w[V * sizeof(T) / 4];
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[j]);
        return __builtin_bit_cast(float, j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
    }
    // the registers as they are: keeps the compiler from holding the widened values of a bf16 vector between two passes
    __device__ __forceinline__ void keep_raw() {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < (int)(V * sizeof(T) / 4); ++j) asm volatile("" : "+v"(w[j]));
        }
    }
};
template <typename T, int V> __device__ __forceinline__ GnVec<T, V> gn_load(const T* p) {
    GnVec<T, V> r;
    constexpr int N = V * sizeof(T) / 4;
    if constexpr (N == 2) {
        const uint2 t = *(const uint2*)p;
        r.w[0] = t.x; r.w[1] = t.y;
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const vec16 t = *((const vec16*)p + j / 4);
            r.w[j] = t.x; r.w[j + 1] = t.y; r.w[j + 2] = t.z; r.w[j + 3] = t.w;
        }
    }
    return r;
}
template <typename T, int V> __device__ __forceinline__ void gn_store(T* p, const float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; j += 4) store4<T>(p + j, (f32x4){f[j], f[j + 1], f[j + 2], f[j + 3]});
}

struct GnPlace { int b, chunk, strip, r0, len, x, y, c0; bool on; };
// n / d for 0 <= n < 2^13, d >= 1: the error of the fp32 quotient stays below the half that is added
__device__ __forceinline__ int gn_div(int n, float inv) { return (int)(((float)n + 0.5f) * inv); }

// workgroup -> (utterance, chunk, strip): the strips of one chunk share cache lines of its rows, so they are dealt to one XCD
// (workgroup ids go round-robin over the 8).  Thread -> (lane x of the strip's row, row y of a pass): whole rows to a wave
// where a row has at most 64 lanes.  len: rows of THIS chunk.
template <int V, int R> __device__ __forceinline__ GnPlace gn_place(const GnArgs& a, int& total) {
    GnPlace p;
    int unit;
    if (a.units >= 8) {
        const int slot = blockIdx.x >> 3;
        unit = (blockIdx.x & 7) + 8 * (slot / a.nstrip);
        p.strip = slot % a.nstrip;
    } else {
        unit = blockIdx.x / a.nstrip;
        p.strip = blockIdx.x % a.nstrip;
    }
    total = 0;
    p.b = -1;
    if (unit >= a.units) return p;
    p.chunk = unit % a.nchunk;
    p.b = unit / a.nchunk;
    const int c0 = min(max(a.cu[p.b], 0), a.M), c1 = min(max(a.cu[p.b + 1], c0), a.M);
    total = min(c1 - c0, a.max_len);
    const int rows = a.LY * R, first = min(p.chunk * rows, total);
    p.r0 = c0 + first;
    p.len = min(total - first, rows);
    if (a.LX <= 64) {
        const int lane = threadIdx.x & 63, rw = gn_div(64, a.inv_lx), y = gn_div(lane, a.inv_lx);
        p.x = lane - y * a.LX;
        p.on = y < rw;
        p.y = (threadIdx.x >> 6) * rw + y;
    } else {
        p.y = gn_div(threadIdx.x, a.inv_lx);
        p.x = threadIdx.x - p.y * a.LX;
        p.on = p.y < a.LY;
    }
    p.c0 = p.strip * a.W + p.x * V;
    return p;
}

// Sums of a strip's columns over the workgroup's rows -> red [entries][w], w = LX * N columns (N values of a lane), entries =
// waves, or the rows of a pass where a row takes several waves.  In a wave: through its own N * 64 floats of `tmp`, every
// column read by as many lanes as there are for it, those joined by shuffles (half the LDS traffic of shuffling all N values
// over all rows).  The caller puts a barrier behind it.
template <int N> __device__ __forceinline__ void gn_put_sums(const GnArgs& a, const GnPlace& p, const float (&s)[N], float* tmp, float* red) {
    const int w = a.LX * N;
    if (a.LX > 64) {
        if (p.on) {
#pragma unroll
            for (int j = 0; j < N; ++j) red[p.y * w + p.x * N + j] = s[j];
        }
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = gn_div(64, a.inv_lx);
    float* t = tmp + wave * 64 * N;
    if constexpr (N == 1) {
        t[lane] = s[0];
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 4) *(f32x4*)(t + lane * N + j) = (f32x4){s[j], s[j + 1], s[j + 2], s[j + 3]};
    }
    __builtin_amdgcn_wave_barrier();
    if (w <= 64) {
        const float inv_w = a.inv_lx * (1.0f / N);
        int parts = min(gn_div(64, inv_w), rows);
        const int part = gn_div(lane, inv_w), c = lane - part * w;
        float v = 0.f;
        if (part < parts)
            for (int y = part; y < rows; y += parts) v += t[y * w + c];
        while (parts > 1) {                      // (uniform)
            const int half = (parts + 1) >> 1;
            const float o = __shfl(v, lane + half * w, 64);
            if (part + half < parts) v += o;
            parts = half;
        }
        if (part == 0) red[wave * w + c] = v;
    } else {
        for (int c = lane; c < w; c += 64) {
            float v = 0.f;
            for (int y = 0; y < rows; ++y) v += t[y * w + c];
            red[wave * w + c] = v;
        }
    }
    __builtin_amdgcn_wave_barrier();
}
// sum over red's entries and a group's `n` columns -> grp[group of the strip], one wave per group
template <int NT> __device__ __forceinline__ void gn_group_sums(const GnArgs& a, const float* red, int w, int n, float* grp) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ng = a.W / a.cg;
    const int entries = a.LX <= 64 ? NT / 64 : a.LY;
    for (int gi = wave; gi < ng; gi += NT / 64) {
        float t = 0.f;
        for (int c = gi * n + lane; c < gi * n + n; c += 64) {
            float u = 0.f;
#pragma unroll 4
            for (int e = 0; e < entries; ++e) u += red[e * w + c];
            t += u;
        }
        t = wave_sum(t);
        if (lane == 0) grp[gi] = t;
    }
}
// the same of two sums at once, * weight[column]
template <int NT>
__device__ __forceinline__ void gn_weighted_sums(const GnArgs& a, const float* red0, const float* red1, const float* weight, float* grp,
                                                 float* grp2) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ng = a.W / a.cg, n = a.cg;
    const int entries = a.LX <= 64 ? NT / 64 : a.LY;
    for (int gi = wave; gi < ng; gi += NT / 64) {
        float t0 = 0.f, t1 = 0.f;
        for (int c = gi * n + lane; c < gi * n + n; c += 64) {
            const float w = weight[c];
            float u0 = 0.f, u1 = 0.f;
#pragma unroll 4
            for (int e = 0; e < entries; ++e) {
                u0 += red0[e * a.W + c];
                u1 += red1[e * a.W + c];
            }
            t0 = fmaf(u0, w, t0);
            t1 = fmaf(u1, w, t1);
        }
        t0 = wave_sum(t0);
        t1 = wave_sum(t1);
        if (lane == 0) {
            grp[gi] = t0;
            grp2[gi] = t1;
        }
    }
}
// the group sums of per-channel values: a lane whose vector lies inside one group adds it up first
template <int V, int NT>
__device__ __forceinline__ void gn_reduce(const GnArgs& a, const GnPlace& p, const float (&s)[V], float* tmp, float* red, float* grp) {
    if (a.cg % V == 0) {
        float t[1] = {0.f};
#pragma unroll
        for (int j = 0; j < V; ++j) t[0] += s[j];
        gn_put_sums<1>(a, p, t, tmp, red);
        __syncthreads();
        gn_group_sums<NT>(a, red, a.LX, a.cg / V, grp);
    } else {
        gn_put_sums<V>(a, p, s, tmp, red);
        __syncthreads();
        gn_group_sums<NT>(a, red, a.W, a.cg, grp);
    }
    __syncthreads();
}

// LDS: a wave's staging, the entries of one or two sums, then two values per group of the strip
#define GN_LDS(V, NT, N)                                                   \
    __shared__ __attribute__((aligned(16))) float tmp[NT * V];             \
    __shared__ __attribute__((aligned(16))) float red[N][NT * V];          \
    extern __shared__ float gn_dyn[];                                      \
    float* grp = gn_dyn;                                                   \
    float* grp2 = gn_dyn + a.W / a.cg

template <int V> __device__ __forceinline__ void gn_params(const float* src, float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
        const f32x4 t = *(const f32x4*)(src + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[j + e] = t[e];
    }
}

// mean, rstd, gamma, beta of a lane's channels
template <int V>
__device__ __forceinline__ void gn_lane_params(const GnArgs& a, const GnPlace& p, float (&mean)[V], float (&rs)[V], float (&ga)[V],
                                               float (&be)[V]) {
    const int c0 = p.on ? p.c0 : p.strip * a.W;
    const float* st = a.stats + (size_t)p.b * a.G * 2;
    gn_params<V>(a.gamma + c0, ga);
    gn_params<V>(a.beta + c0, be);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int gi = gn_div(c0 + j, a.inv_cg);
        mean[j] = st[gi * 2];
        rs[j] = st[gi * 2 + 1];
    }
}

// y rows from x rows in registers or memory, given the groups' mean (grp) and rstd (grp2) in LDS
template <typename TX, typename TO, int V>
__device__ __forceinline__ void gn_write_row(const GnArgs& a, int row, int c0, const GnVec<TX, V>& x, const float (&mean)[V],
                                             const float (&rg)[V], const float (&be)[V]) {
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = fmaf(x.get(j) - mean[j], rg[j], be[j]);
    gn_act<V>(a.act, o);
    gn_drop<V>(a.drop, row, c0, o);
    gn_store<TO, V>((TO*)a.out + (size_t)row * a.ldo + c0, o);
}

// WHOLE: the utterance fits (nchunk == 1): statistics and output in one pass.  Else: (mean, M2) of the chunk to part.
template <typename TX, typename TO, int R, bool WHOLE>
__global__ __launch_bounds__(WHOLE ? GN_WHOLE_THREADS : GN_CHUNK_THREADS) void gn_fwd_kernel(GnArgs a) {
    constexpr int NT = WHOLE ? GN_WHOLE_THREADS : GN_CHUNK_THREADS;
    constexpr int V = 16 / (int)sizeof(TX);
    GN_LDS(V, NT, 1);
    int total;
    const GnPlace p = gn_place<V, R>(a, total);
    if (p.b < 0 || (!WHOLE && p.len == 0)) return;          // (block-uniform)
    GnVec<TX, V> x[R];
    const TX* src = (const TX*)a.x + (size_t)p.r0 * a.ldx + p.c0;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int row = p.y + k * a.LY;
        if (p.on && row < p.len) x[k] = gn_load<TX, V>(src + (size_t)row * a.ldx);
    }
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = 0.f;
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (p.on && p.y + k * a.LY < p.len) {
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += x[k].get(j);
        }
    gn_reduce<V, NT>(a, p, s, tmp, red[0], grp);
    const float inv_n = p.len > 0 ? 1.0f / ((float)p.len * (float)a.cg) : 0.f;
    float mean[V];
    int gi[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        gi[j] = p.on ? gn_div(p.x * V + j, a.inv_cg) : 0;
        mean[j] = grp[gi[j]] * inv_n;
        s[j] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < R; ++k) x[k].keep_raw();
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (p.on && p.y + k * a.LY < p.len) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = x[k].get(j) - mean[j];
                s[j] = fmaf(d, d, s[j]);
            }
        }
    gn_reduce<V, NT>(a, p, s, tmp, red[0], grp2);
    const int g0 = p.strip * (a.W / a.cg), ng = a.W / a.cg;
    if (!WHOLE) {
        float* dst = a.part + (((size_t)p.b * a.nchunk + p.chunk) * a.G + g0) * 2;
        for (int t = threadIdx.x; t < ng; t += NT) {
            dst[t * 2] = grp[t] * inv_n;
            dst[t * 2 + 1] = grp2[t];
        }
        return;
    }
    for (int t = threadIdx.x; t < ng; t += NT) {
        float* st = a.stats + ((size_t)p.b * a.G + g0 + t) * 2;
        st[0] = grp[t] * inv_n;
        st[1] = 1.0f / sqrtf(grp2[t] * inv_n + a.eps);
    }
    if (!p.on) return;
    float rg[V], be[V];
    gn_params<V>(a.gamma + p.c0, rg);
    gn_params<V>(a.beta + p.c0, be);
#pragma unroll
    for (int j = 0; j < V; ++j) rg[j] *= 1.0f / sqrtf(grp2[gi[j]] * inv_n + a.eps);
#pragma unroll
    for (int k = 0; k < R; ++k) x[k].keep_raw();
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int row = p.y + k * a.LY;
        if (row < p.len) gn_write_row<TX, TO, V>(a, p.r0 + row, p.c0, x[k], mean, rg, be);
    }
}

// Chunks -> utterance, one wave to a group: lanes take every 64th chunk, sums in 64 bits, then over the wave; a fixed order.  Up to GN_JOIN_HERE
// chunks (one load to a lane) each workgroup of the last kernel does that for itself; beyond, where a workgroup would take longer over the
// chunks than over its rows, a launch of its own does it once (3 us; 3 x 3500 rows x 512 channels in one group, 219 chunks: forward 19.8 us,
// backward 34.5; a serial join in each workgroup took 62 and 495).
constexpr int GN_JOIN_HERE = 64;
// mean = sum n_i mean_i / n,  variance = (sum M2_i + n_i (mean_i - mean)^2) / n
__device__ __forceinline__ void gn_join(const GnArgs& a, int b, int g, int rows, int total, float& mean, float& rstd) {
    const unsigned lane = threadIdx.x & 63;
    const float* src = a.part + ((size_t)b * a.nchunk * a.G + g) * 2;
    const size_t step = (size_t)a.G * 2;
    const float inv = total > 0 ? 1.0f / (float)total : 0.f;
    double t = 0.0;
#pragma unroll 4
    for (unsigned c = lane; c * rows < (unsigned)total; c += 64) t += (double)src[c * step] * (double)min(total - (int)c * rows, rows);
    mean = wave_sum((float)t) * inv;
    t = 0.0;
#pragma unroll 4
    for (unsigned c = lane; c * rows < (unsigned)total; c += 64) {
        const float d = src[c * step] - mean;
        t += (double)(d * d * ((float)min(total - (int)c * rows, rows) * (float)a.cg) + src[c * step + 1]);
    }
    rstd = 1.0f / sqrtf(wave_sum((float)t) * (inv / (float)a.cg) + a.eps);
}
// the means of dh and dh xhat
__device__ __forceinline__ void gn_join_bwd(const GnArgs& a, int b, int g, int rows, int total, float& m1, float& m2) {
    const unsigned lane = threadIdx.x & 63;
    const float* src = a.gpart + ((size_t)b * a.nchunk * a.G + g) * 2;
    const size_t step = (size_t)a.G * 2;
    double t0 = 0.0, t1 = 0.0;
#pragma unroll 4
    for (unsigned c = lane; c * rows < (unsigned)total; c += 64) {
        t0 += (double)src[c * step];
        t1 += (double)src[c * step + 1];
    }
    const float inv_n = total > 0 ? 1.0f / ((float)total * (float)a.cg) : 0.f;
    m1 = wave_sum((float)t0) * inv_n;
    m2 = wave_sum((float)t1) * inv_n;
}
// the launch for many chunks: forward to stats, backward to gsum
template <int R, bool BWD> __global__ __launch_bounds__(GN_CHUNK_THREADS) void gn_join_kernel(GnArgs a) {
    const unsigned slot = blockIdx.x * (GN_CHUNK_THREADS / 64) + (threadIdx.x >> 6);
    const int b = (int)(slot / (unsigned)a.G), g = (int)(slot - (unsigned)b * (unsigned)a.G);
    if (b >= a.units / a.nchunk) return;
    const int c0 = min(max(a.cu[b], 0), a.M), c1 = min(max(a.cu[b + 1], c0), a.M), total = min(c1 - c0, a.max_len);
    float u, v;
    if (BWD) gn_join_bwd(a, b, g, a.LY * R, total, u, v);
    else gn_join(a, b, g, a.LY * R, total, u, v);
    if ((threadIdx.x & 63) == 0) {
        float* dst = (BWD ? a.gsum : a.stats) + ((size_t)b * a.G + g) * 2;
        dst[0] = u;
        dst[1] = v;
    }
}

// chunked forward, last kernel: apply
template <typename TX, typename TO, int R>
__global__ __launch_bounds__(GN_CHUNK_THREADS) void gn_apply_kernel(GnArgs a) {
    constexpr int V = 16 / (int)sizeof(TX);
    extern __shared__ float gn_dyn[];
    const int ng = a.W / a.cg;
    float *grp = gn_dyn, *grp2 = gn_dyn + ng;
    int total;
    const GnPlace p = gn_place<V, R>(a, total);
    if (p.b < 0 || (p.len == 0 && p.chunk > 0)) return;
    const bool here = a.nchunk <= GN_JOIN_HERE;
    if (here) {
        for (int gi = threadIdx.x >> 6; gi < ng; gi += GN_CHUNK_THREADS / 64) {
            float u, v;
            gn_join(a, p.b, p.strip * ng + gi, a.LY * R, total, u, v);
            if ((threadIdx.x & 63) == 0) {
                grp[gi] = u;
                grp2[gi] = v;
                if (p.chunk == 0) {
                    float* st = a.stats + ((size_t)p.b * a.G + p.strip * ng + gi) * 2;
                    st[0] = u;
                    st[1] = v;
                }
            }
        }
        __syncthreads();
    }
    if (!p.on) return;
    const float* st = a.stats + ((size_t)p.b * a.G + p.strip * ng) * 2;
    float mean[V], rg[V], be[V];
    gn_params<V>(a.gamma + p.c0, rg);
    gn_params<V>(a.beta + p.c0, be);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int gi = gn_div(p.x * V + j, a.inv_cg);
        mean[j] = here ? grp[gi] : st[gi * 2];
        rg[j] *= here ? grp2[gi] : st[gi * 2 + 1];
    }
    const TX* src = (const TX*)a.x + (size_t)p.r0 * a.ldx + p.c0;
#pragma unroll 4
    for (int k = 0; k < R; ++k) {
        const int row = p.y + k * a.LY;
        if (row < p.len) gn_write_row<TX, TO, V>(a, p.r0 + row, p.c0, gn_load<TX, V>(src + (size_t)row * a.ldx), mean, rg, be);
    }
}

template <typename TD, int V>
__device__ __forceinline__ void gn_dz(const GnArgs& a, int row, int c0, const GnVec<TD, V>& d, const float (&xh)[V],
                                      const float (&ga)[V], const float (&be)[V], float (&dz)[V]) {
    float z[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        dz[j] = d.get(j);
        z[j] = fmaf(xh[j], ga[j], be[j]);
    }
    gn_drop<V>(a.drop, row, c0, dz);
    gn_slope<V>(a.act, z, dz);
}

// WHOLE: sums and dx in one pass; always: the chunk's channel sums of dz and dz xhat to part
template <typename TX, typename TD, typename TG, int R, bool WHOLE>
__global__ __launch_bounds__(WHOLE ? GN_WHOLE_THREADS : GN_CHUNK_THREADS) void gn_bwd_kernel(GnArgs a) {
    constexpr int NT = WHOLE ? GN_WHOLE_THREADS : GN_CHUNK_THREADS;
    constexpr int V = 16 / (int)sizeof(TX);
    GN_LDS(V, NT, 2);
    int total;
    const GnPlace p = gn_place<V, R>(a, total);
    if (p.b < 0) return;
    constexpr int HOLD = WHOLE ? R : GN_HOLD;                   // rows in registers at a time
    GnVec<TX, V> x[HOLD];
    GnVec<TD, V> d[HOLD];
    constexpr bool KEEP = WHOLE && (R <= 8 || sizeof(TX) == 4);
    float dz[KEEP ? R : 1][V];
    const TX* src = (const TX*)a.x + (size_t)p.r0 * a.ldx + p.c0;
    const TD* sd = (const TD*)a.dout + (size_t)p.r0 * a.ldd + p.c0;
    float mean[V], rs[V], ga[V], be[V];
    if (!WHOLE) gn_lane_params<V>(a, p, mean, rs, ga, be);
    float s0[V], s1[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s0[j] = s1[j] = 0.f;
#pragma unroll 1
    for (int k0 = 0; k0 < R; k0 += HOLD) {
#pragma unroll
        for (int k = 0; k < HOLD; ++k) {
            const int row = p.y + (k0 + k) * a.LY;
            if (p.on && row < p.len) {
                x[k] = gn_load<TX, V>(src + (size_t)row * a.ldx);
                d[k] = gn_load<TD, V>(sd + (size_t)row * a.ldd);
            }
        }
        if (WHOLE) gn_lane_params<V>(a, p, mean, rs, ga, be);       // behind the rows' loads
#pragma unroll
        for (int k = 0; k < HOLD; ++k) {
            const int row = p.y + (k0 + k) * a.LY;
            if (p.on && row < p.len) {
                float xh[V];
#pragma unroll
                for (int j = 0; j < V; ++j) xh[j] = (x[k].get(j) - mean[j]) * rs[j];
                gn_dz<TD, V>(a, p.r0 + row, p.c0, d[k], xh, ga, be, dz[KEEP ? k : 0]);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s0[j] += dz[KEEP ? k : 0][j];
                    s1[j] = fmaf(dz[KEEP ? k : 0][j], xh[j], s1[j]);
                }
            }
        }
    }
    gn_put_sums<V>(a, p, s0, tmp, red[0]);
    gn_put_sums<V>(a, p, s1, tmp, red[1]);
    __syncthreads();
    float* dst = a.part + ((size_t)p.b * a.nchunk + p.chunk) * 2 * a.C + p.strip * a.W;
    const int entries = a.LX <= 64 ? NT / 64 : a.LY;
    for (int c = threadIdx.x; c < a.W; c += NT) {
        float t0 = 0.f, t1 = 0.f;
#pragma unroll 8
        for (int e = 0; e < entries; ++e) {
            t0 += red[0][e * a.W + c];
            t1 += red[1][e * a.W + c];
        }
        dst[c] = t0;
        dst[a.C + c] = t1;
    }
    gn_weighted_sums<NT>(a, red[0], red[1], a.gamma + p.strip * a.W, grp, grp2);
    __syncthreads();
    if (!WHOLE) {
        const int ng = a.W / a.cg;
        float* gdst = a.gpart + (((size_t)p.b * a.nchunk + p.chunk) * a.G + p.strip * ng) * 2;
        for (int t = threadIdx.x; t < ng; t += NT) {
            gdst[t * 2] = grp[t];
            gdst[t * 2 + 1] = grp2[t];
        }
        return;
    }
    if (!p.on) return;
    const float inv_n = p.len > 0 ? 1.0f / ((float)p.len * (float)a.cg) : 0.f;
    float m1[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int gi = gn_div(p.x * V + j, a.inv_cg);
        m1[j] = grp[gi] * inv_n;
        m2[j] = grp2[gi] * inv_n;
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
        x[k].keep_raw();
        if (!KEEP) d[k].keep_raw();
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int row = p.y + k * a.LY;
        if (row < p.len) {
            float o[V], xh[V];
#pragma unroll
            for (int j = 0; j < V; ++j) xh[j] = (x[k].get(j) - mean[j]) * rs[j];
            if (!KEEP) gn_dz<TD, V>(a, p.r0 + row, p.c0, d[k], xh, ga, be, dz[0]);
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = rs[j] * (fmaf(ga[j], dz[KEEP ? k : 0][j], -m1[j]) - xh[j] * m2[j]);
            gn_store<TG, V>((TG*)a.dx + (size_t)(p.r0 + row) * a.ldg + p.c0, o);
        }
    }
}

// chunked backward, last kernel: dx from a second read
template <typename TX, typename TD, typename TG, int R>
__global__ __launch_bounds__(GN_CHUNK_THREADS) void gn_bwd_apply_kernel(GnArgs a) {
    constexpr int V = 16 / (int)sizeof(TX);
    extern __shared__ float gn_dyn[];
    const int ng = a.W / a.cg;
    float *grp = gn_dyn, *grp2 = gn_dyn + ng;
    int total;
    const GnPlace p = gn_place<V, R>(a, total);
    if (p.b < 0 || p.len == 0) return;
    const bool here = a.nchunk <= GN_JOIN_HERE;
    if (here) {
        for (int gi = threadIdx.x >> 6; gi < ng; gi += GN_CHUNK_THREADS / 64) {
            float u, v;
            gn_join_bwd(a, p.b, p.strip * ng + gi, a.LY * R, total, u, v);
            if ((threadIdx.x & 63) == 0) {
                grp[gi] = u;
                grp2[gi] = v;
            }
        }
        __syncthreads();
    }
    if (!p.on) return;
    const float* sums = a.gsum + ((size_t)p.b * a.G + p.strip * ng) * 2;
    float mean[V], rs[V], ga[V], be[V], m1[V], m2[V];
    gn_lane_params<V>(a, p, mean, rs, ga, be);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int gi = gn_div(p.x * V + j, a.inv_cg);
        m1[j] = here ? grp[gi] : sums[gi * 2];
        m2[j] = here ? grp2[gi] : sums[gi * 2 + 1];
    }
    const TX* src = (const TX*)a.x + (size_t)p.r0 * a.ldx + p.c0;
    const TD* sd = (const TD*)a.dout + (size_t)p.r0 * a.ldd + p.c0;
#pragma unroll 4
    for (int k = 0; k < R; ++k) {
        const int row = p.y + k * a.LY;
        if (row < p.len) {
            const GnVec<TX, V> x = gn_load<TX, V>(src + (size_t)row * a.ldx);
            const GnVec<TD, V> d = gn_load<TD, V>(sd + (size_t)row * a.ldd);
            float xh[V], dz[V], o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) xh[j] = (x.get(j) - mean[j]) * rs[j];
            gn_dz<TD, V>(a, p.r0 + row, p.c0, d, xh, ga, be, dz);
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = rs[j] * (fmaf(ga[j], dz[j], -m1[j]) - xh[j] * m2[j]);
            gn_store<TG, V>((TG*)a.dx + (size_t)(p.r0 + row) * a.ldg + p.c0, o);
        }
    }
}

// dgamma, dbeta: sums of the partial rows [n][2][C]; 16 columns x 64 row lanes per workgroup, f64 over the row lanes' sums
__global__ __launch_bounds__(1024) void gn_param_kernel(const float* __restrict__ part, int n, int C, float* __restrict__ dgamma,
                                                        float* __restrict__ dbeta) {
    __shared__ float red[64][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
    float t = 0.f;
    if (c < 2 * C) {
#pragma unroll 4
        for (int r = y; r < n; r += 64) t += part[(size_t)r * 2 * C + c];
    }
    red[y][x] = t;
    __syncthreads();
    if (threadIdx.x < 64) {                      // y < 4: a quarter of the row lanes each
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < 16; ++k) sum += (double)red[y * 16 + k][x];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (y == 0 && c < 2 * C) {
            if (c < C)
                dbeta[c] = (float)sum;
            else
                dgamma[c - C] = (float)sum;
        }
    }
}

// ---- geometry ------------------------------------------------------------------------------------------------------
// Strip: the narrowest run of whole groups and whole vectors that is at least GN_STRIP_BYTES wide and divides C.  R: rows per thread,
// the smallest compiled one that holds the utterance; none does: chunks of GN_CHUNK_ROWS.
// More than 8 rows per thread of a bf16 backward (128 registers of data): only for bf16 dout (the thread recomputes dz instead of
// keeping it; 4 x 1500 rows x 256 channels with fp32 dout: 27 us against 18 in chunks), and only where the workgroups fill the chip
// (512 of them, 256 x 800 x 80: 35 us against 47 in chunks; 256: 19 against 27; 64: 15, 20 and 25 us without activation, with tanh and with
// SiLU against 18, 20 and 22).  All others hold 16 rows (32 x 1600 x 256 fp32: forward 30 us against 44 in chunks, backward 47 against 77;
// one utterance 8.6 against 12.4, 10.6 against 16.1).
struct GnPlan { int W, LX, LY, R, nchunk; bool whole; };

static int gn_gcd(int a, int b) { return b ? gn_gcd(b, a % b) : a; }

// dout_dtype: of a backward, -1 for the forward
static GnPlan gn_plan(int B, int max_len, int C, int G, int x_dtype, int dout_dtype) {
    GnPlan p;
    const int V = x_dtype == 0 ? 4 : 8, es = x_dtype == 0 ? 4 : 2, cg = C / G;
    const int unit = cg / gn_gcd(cg, V) * V, units = C / unit;
    int m = 1;
    while (m < units && (m * unit * es < GN_STRIP_BYTES || units % m)) ++m;
    p.W = m * unit;
    p.LX = p.W / V;
    const bool fewer = x_dtype == 1 && dout_dtype >= 0 && (dout_dtype == 0 || (long long)B * (C / p.W) < 256);
    for (int nt = GN_WHOLE_THREADS;; nt = GN_CHUNK_THREADS) {
        p.LY = p.LX <= 64 ? nt / 64 * (64 / p.LX) : nt / p.LX;
        const int need = (int)(((long long)max_len + p.LY - 1) / p.LY);
        p.whole = nt == GN_WHOLE_THREADS && need <= (fewer ? 8 : 16);
        p.R = !p.whole ? GN_CHUNK_ROWS : (need <= 4 ? 4 : (need <= 8 ? 8 : 16));
        p.nchunk = p.whole ? 1 : (int)(((long long)max_len + p.LY * p.R - 1) / (p.LY * p.R));
        if (p.whole || nt == GN_CHUNK_THREADS) break;
    }
    return p;
}

static unsigned gn_grid(const GnArgs& a) {
    return (unsigned)(a.units >= 8 ? 8LL * a.nstrip * ((a.units + 7) / 8) : (long long)a.units * a.nstrip);
}

static unsigned gn_join_grid(const GnArgs& a) {          // a wave to every (utterance, group)
    return (unsigned)(((long long)(a.units / a.nchunk) * a.G + GN_CHUNK_THREADS / 64 - 1) / (GN_CHUNK_THREADS / 64));
}

template <typename TX, typename TO, int R> static void gn_launch_fwd(const GnArgs& a, const GnPlan& p, hipStream_t s) {
    const unsigned grid = gn_grid(a);
    const int lds = 2 * (a.W / a.cg) * (int)sizeof(float);
    if (p.whole) {
        hipLaunchKernelGGL((gn_fwd_kernel<TX, TO, R, true>), dim3(grid), dim3(GN_WHOLE_THREADS), lds, s, a);
    } else if constexpr (R == GN_CHUNK_ROWS) {
        hipLaunchKernelGGL((gn_fwd_kernel<TX, TO, R, false>), dim3(grid), dim3(GN_CHUNK_THREADS), lds, s, a);
        if (a.nchunk > GN_JOIN_HERE) hipLaunchKernelGGL((gn_join_kernel<R, false>), dim3(gn_join_grid(a)), dim3(GN_CHUNK_THREADS), 0, s, a);
        hipLaunchKernelGGL((gn_apply_kernel<TX, TO, R>), dim3(grid), dim3(GN_CHUNK_THREADS), lds, s, a);
    }
}
template <typename TX, typename TO> static void gn_launch_fwd_r(const GnArgs& a, const GnPlan& p, hipStream_t s) {
    if (p.R == 4) gn_launch_fwd<TX, TO, 4>(a, p, s);
    else if (p.R == 8) gn_launch_fwd<TX, TO, 8>(a, p, s);
    else gn_launch_fwd<TX, TO, 16>(a, p, s);
}

template <typename TX, typename TD, typename TG, int R>
static void gn_launch_bwd(const GnArgs& a, const GnPlan& p, hipStream_t s) {
    const unsigned grid = gn_grid(a);
    const int lds = 2 * (a.W / a.cg) * (int)sizeof(float);
    if (p.whole) {
        hipLaunchKernelGGL((gn_bwd_kernel<TX, TD, TG, R, true>), dim3(grid), dim3(GN_WHOLE_THREADS), lds, s, a);
    } else if constexpr (R == GN_CHUNK_ROWS) {
        hipLaunchKernelGGL((gn_bwd_kernel<TX, TD, TG, R, false>), dim3(grid), dim3(GN_CHUNK_THREADS), lds, s, a);
        if (a.nchunk > GN_JOIN_HERE) hipLaunchKernelGGL((gn_join_kernel<R, true>), dim3(gn_join_grid(a)), dim3(GN_CHUNK_THREADS), 0, s, a);
        hipLaunchKernelGGL((gn_bwd_apply_kernel<TX, TD, TG, R>), dim3(grid), dim3(GN_CHUNK_THREADS), lds, s, a);
    }
}
template <typename TX, typename TD, typename TG> static void gn_launch_bwd_r(const GnArgs& a, const GnPlan& p, hipStream_t s) {
    if (p.R == 4) gn_launch_bwd<TX, TD, TG, 4>(a, p, s);
    else if (p.R == 8) gn_launch_bwd<TX, TD, TG, 8>(a, p, s);
    else if constexpr (sizeof(TX) == 4 || sizeof(TD) == 2) gn_launch_bwd<TX, TD, TG, 16>(a, p, s);
}

static int gn_check(const char* who, const void* x, const int* cu, const float* gamma, const float* beta, const float* stats, int B,
                    int max_len, int M, int C, int groups, int ldx, int act, int x_dtype, float rate) {
    FS2_CHECK_ARG(cu && gamma && beta && stats && (x || M == 0) && B > 0 && M >= 0, "%s: bad args", who);
    FS2_CHECK_ARG(max_len >= 0 && max_len <= M && B <= (1 << 24), "%s: B=%d, max_len=%d, M=%d", who, B, max_len, M);
    FS2_CHECK_ARG(x_dtype == 0 || x_dtype == 1, "%s: x_dtype=%d (0 fp32, 1 bf16)", who, x_dtype);
    const int V = x_dtype == 0 ? 4 : 8;
    FS2_CHECK_ARG((((uintptr_t)gamma | (uintptr_t)beta) & 15) == 0, "%s: gamma or beta unaligned", who);
    FS2_CHECK_ARG(C > 0 && C <= 1024 && C % V == 0, "%s: C=%d must be a multiple of %d and at most 1024", who, C, V);
    FS2_CHECK_ARG(groups > 0 && C % groups == 0, "%s: %d channels in %d groups", who, C, groups);
    FS2_CHECK_ARG(ldx >= C && ldx % V == 0 && ((uintptr_t)x & 15) == 0, "%s: ldx=%d, or x unaligned", who, ldx);
    FS2_CHECK_ARG(act >= 0 && act <= 3, "%s: act=%d (0 none, 1 ReLU, 2 tanh, 3 SiLU)", who, act);
    FS2_CHECK_ARG(rate >= 0.f && rate < 1.f, "%s: dropout rate must be in [0, 1)", who);
    return FS2_OK;
}

static GnArgs gn_args(int B, const void* x, const int* cu, const float* gamma, const float* beta, float* stats, void* workspace,
                      int max_len, int M, int C, int groups, int ldx, int act, const GnPlan& p, Dropout drop) {
    GnArgs a = {};
    a.x = x; a.cu = cu; a.gamma = gamma; a.beta = beta; a.stats = stats; a.part = (float*)workspace;
    a.M = M; a.max_len = max_len; a.C = C; a.G = groups; a.cg = C / groups; a.ldx = ldx; a.act = act;
    a.nchunk = p.nchunk; a.nstrip = C / p.W; a.W = p.W; a.LX = p.LX; a.LY = p.LY;
    a.units = B * p.nchunk; a.inv_lx = 1.0f / (float)p.LX; a.inv_cg = 1.0f / (float)a.cg;
    a.drop = drop;
    return a;
}

}  // namespace fs2

using namespace fs2;

extern "C" long long fs2_group_norm_workspace(int B, int max_len, int C, int groups) {
    if (B <= 0 || C <= 0 || groups <= 0 || C % groups || C % 4) return 0;
    long long most = 0;
    for (int t = 0; t < (C % 8 ? 1 : 2); ++t) {
        const GnPlan p = gn_plan(B, max_len, C, groups, t, -1);
        const long long n = p.whole ? 0 : (long long)B * p.nchunk * groups * 2 * (long long)sizeof(float);
        most = n > most ? n : most;
    }
    return most;
}

extern "C" int fs2_group_norm(const void* x, const int* cu, const float* gamma, const float* beta, void* out, float* stats,
                              void* workspace, int B, int max_len, int M, int C, int groups, int ldx, int ldo, float eps, int act,
                              int x_dtype, int out_dtype, unsigned seed, unsigned site, float rate, hipStream_t stream) {
    const int rc = gn_check("fs2_group_norm", x, cu, gamma, beta, stats, B, max_len, M, C, groups, ldx, act, x_dtype, rate);
    if (rc != FS2_OK) return rc;
    FS2_CHECK_ARG((out_dtype == 0 || out_dtype == 1) && (out || M == 0) && ldo >= C && ldo % 4 == 0 && ((uintptr_t)out & 15) == 0,
                  "fs2_group_norm: out_dtype=%d, ldo=%d (a multiple of 4), or out null or unaligned", out_dtype, ldo);
    FS2_CHECK_ARG(eps > 0.f, "fs2_group_norm: eps must be positive");
    const GnPlan p = gn_plan(B, max_len, C, groups, x_dtype, -1);
    FS2_CHECK_ARG(p.whole || workspace, "fs2_group_norm: this shape needs fs2_group_norm_workspace bytes");
    FS2_CHECK_ARG((long long)B * p.nchunk * (C / p.W) < (1ll << 22), "fs2_group_norm: too many workgroups (B=%d)", B);
    GnArgs a = gn_args(B, x, cu, gamma, beta, stats, workspace, max_len, M, C, groups, ldx, act, p, fs2_make_dropout(seed, site, rate));
    a.out = out; a.ldo = ldo; a.eps = eps;
    if (x_dtype == 0 && out_dtype == 0) gn_launch_fwd_r<float, float>(a, p, stream);
    else if (x_dtype == 0) gn_launch_fwd_r<float, bf16_t>(a, p, stream);
    else if (out_dtype == 0) gn_launch_fwd_r<bf16_t, float>(a, p, stream);
    else gn_launch_fwd_r<bf16_t, bf16_t>(a, p, stream);
    FS2_CHECK_LAUNCH("fs2_group_norm");
    return FS2_OK;
}

// a chunked backward's workspace: the chunks' channel sums, their group sums, the utterances' group means
static long long gn_bwd_floats(int B, int C, int groups, const GnPlan& p) {
    const long long units = (long long)B * p.nchunk;
    return units * 2 * C + (p.whole ? 0 : (units + B) * groups * 2);
}

extern "C" long long fs2_group_norm_bwd_workspace(int B, int max_len, int C, int groups) {
    if (B <= 0 || C <= 0 || groups <= 0 || C % groups || C % 4) return 16;
    long long most = 0;
    for (int t = 0; t < (C % 8 ? 2 : 4); ++t) {
        const GnPlan p = gn_plan(B, max_len, C, groups, t >> 1, t & 1);
        const long long n = gn_bwd_floats(B, C, groups, p) * (long long)sizeof(float);
        most = n > most ? n : most;
    }
    return most;
}

extern "C" int fs2_group_norm_bwd(const void* x, const float* stats, const int* cu, const float* gamma, const float* beta,
                                  const void* dout, void* dx, float* dgamma, float* dbeta, void* workspace, int B, int max_len, int M,
                                  int C, int groups, int ldx, int ldd, int ldg, int act, int x_dtype, int dout_dtype, int dx_dtype,
                                  unsigned seed, unsigned site, float rate, hipStream_t stream) {
    const int rc = gn_check("fs2_group_norm_bwd", x, cu, gamma, beta, stats, B, max_len, M, C, groups, ldx, act, x_dtype, rate);
    if (rc != FS2_OK) return rc;
    FS2_CHECK_ARG((dout_dtype == 0 || dout_dtype == 1) && (dx_dtype == 0 || dx_dtype == 1),
                  "fs2_group_norm_bwd: dout_dtype=%d, dx_dtype=%d (0 fp32, 1 bf16)", dout_dtype, dx_dtype);
    FS2_CHECK_ARG((M == 0 || (dout && dx)) && dgamma && dbeta && workspace, "fs2_group_norm_bwd: null argument");
    FS2_CHECK_ARG(ldd >= C && ldg >= C && ldd % (x_dtype == 0 ? 4 : 8) == 0 && ldg % 4 == 0 &&
                      (((uintptr_t)dout | (uintptr_t)dx) & 15) == 0,
                  "fs2_group_norm_bwd: ldd=%d (a multiple of %d), ldg=%d (of 4), or dout or dx unaligned", ldd, x_dtype == 0 ? 4 : 8,
                  ldg);
    const GnPlan p = gn_plan(B, max_len, C, groups, x_dtype, dout_dtype);
    FS2_CHECK_ARG((long long)B * p.nchunk * (C / p.W) < (1ll << 22), "fs2_group_norm_bwd: too many workgroups (B=%d)", B);
    GnArgs a = gn_args(B, x, cu, gamma, beta, (float*)stats, workspace, max_len, M, C, groups, ldx, act, p, fs2_make_dropout(seed, site, rate));
    a.dout = dout; a.dx = dx; a.ldd = ldd; a.ldg = ldg;
    a.gpart = a.part + (size_t)a.units * 2 * C;
    a.gsum = a.gpart + (size_t)a.units * groups * 2;
#define FS2_GN(TX, TD)                                              \
    if (dx_dtype == 0) gn_launch_bwd_r<TX, TD, float>(a, p, stream); \
    else gn_launch_bwd_r<TX, TD, bf16_t>(a, p, stream)
    if (x_dtype == 0 && dout_dtype == 0) { FS2_GN(float, float); }
    else if (x_dtype == 0) { FS2_GN(float, bf16_t); }
    else if (dout_dtype == 0) { FS2_GN(bf16_t, float); }
    else { FS2_GN(bf16_t, bf16_t); }
#undef FS2_GN
    hipLaunchKernelGGL(gn_param_kernel, dim3((2 * C + 15) / 16), dim3(1024), 0, stream, a.part, B * p.nchunk, C, dgamma, dbeta);
    FS2_CHECK_LAUNCH("fs2_group_norm_bwd");
    return FS2_OK;
}
