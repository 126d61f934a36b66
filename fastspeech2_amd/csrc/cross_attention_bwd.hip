// Backward of cross attention (cross_attention.hip) and the attention mass of every key; the probabilities are recomputed tile
// by tile from q, k and the saved log-sum-exp, never stored.  With S = q k^T / sqrt(dk), P = exp2(S log2 e - lse), D the
// dropout multiplier, O = (P o D) v and upstream dO:
//   delta = sum_dv dO o O
//   dP = dO v^T o D,  dS = P o (dP - delta)
//   dq = dS k / sqrt(dk)                                          xattn_dq_kernel: one wave per 16 packed rows
//   dk = dS^T q / sqrt(dk),  dv = (P o D)^T dO                    xattn_dkv_kernel: one wave per 16 keys, over ALL packed rows
//   mass[h][key] = sum_q P                                        xattn_mass_kernel
// The packed rows of a shared head are its g query heads, so the sum over the group that dk and dv need is part of the loop.
// Every output element has one writer and every sum a fixed order: no atomics, the same bits every time.
#include "cross_attention.h"

namespace fs2 {

// ---- dq and delta: one workgroup per (utterance, shared head, 64 packed rows) -------------------------------------
template <typename T, int DK>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void xattn_dq_kernel(XArgs a) {
    typedef XTile<T, DK> TL;
    typedef typename TL::frag_t frag_t;
    constexpr int KS = TL::KS, DT = TL::DT;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];     // stage s: K tile (rotation 2), V tile (rotation 1)

    int b, kvh, blk;
    if (!fs2_pair_order_decode(a.order, b, kvh, blk)) return;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, q0, lenq);
    x_range(a.cu_k, b, a.Mk, k0, lenk);
    const int nrow = lenq * a.g;
    if (blk * 64 >= nrow) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int r = blk * 64 + wave * 16 + i;
    const int rc = min(r, nrow - 1), q = x_query(a, rc);
    const int head = kvh * a.g + rc - q * a.g, qrow = q0 + q;

    const T* __restrict__ kb = (const T*)a.k + (size_t)k0 * a.ldk + kvh * DK;
    const T* __restrict__ vb = (const T*)a.v + (size_t)k0 * a.ldv + kvh * DK;
    auto stage = [&](int kt, int st) __attribute__((always_inline)) {
        unsigned char* d = smem + st * 2 * TL::BYTES;
        TL::template stage<2, 4>(kb, a.ldk, kt * 64, lenk, d, wave, lane);
        TL::template stage<1, 4>(vb, a.ldv, kt * 64, lenk, d + TL::BYTES, wave, lane);
    };
    if (lenk > 0) stage(0, 0);

    frag_t qf[KS], dof[KS];
    float del = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int c = head * DK + ks * 32 + g * 8;
        qf[ks] = *(const frag_t*)((const T*)a.q + (size_t)qrow * a.ldq + c);
        dof[ks] = *(const frag_t*)((const T*)a.dctx + (size_t)qrow * a.ldo + c);
        const frag_t of = *(const frag_t*)((const T*)a.ctx + (size_t)qrow * a.ldo + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) del = fmaf(to_f32(dof[ks][j]), to_f32(of[j]), del);
    }
    del = rows_sum(del);
    if (g == 0 && r < nrow) a.delta[(size_t)head * a.Mq + qrow] = del;
    const float lse_q = a.lse[(size_t)head * a.Mq + qrow];

    f32x4 dq[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dq[dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    Dropout dh = a.drop;
    dh.stream += (uint32_t)head;
    const int ntiles = (lenk + 63) / 64;
    for (int kt = 0; kt < ntiles; ++kt) {
        vm_wait_barrier<0>();      // tile kt has landed; every wave is done with the other stage
        if (kt + 1 < ntiles) stage(kt + 1, (kt + 1) & 1);
        const unsigned char* Ks = smem + (kt & 1) * 2 * TL::BYTES;
        const unsigned char* Vs = Ks + TL::BYTES;
        f32x4 s[4], dp[4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) s[nt] = dp[nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            frag_t kf[4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) kf[nt] = TL::template row_frag<2>(Ks, nt * 16 + i, ks, g);
            mma16_multi<4>(kf, qf[ks], s);
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) kf[nt] = TL::template row_frag<1>(Vs, nt * 16 + i, ks, g);
            mma16_multi<4>(kf, dof[ks], dp);
        }
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = kt * 64 + nt * 16 + 4 * g + e;
                const float p = key < lenk ? __builtin_amdgcn_exp2f(fmaf(s[nt][e], a.scale_log2e, -lse_q)) : 0.f;
                float dpv = dp[nt][e];
                if (a.drop.thresh) dpv *= drop_mul(dh, (uint32_t)qrow, (uint32_t)key);
                s[nt][e] = key < lenk ? p * (dpv - del) : 0.f;
            }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const frag_t dsf = x_pack<T>(s[2 * c], s[2 * c + 1]);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) dq[dt] = mma16(TL::template col_frag<2>(Ks, c, dt, g, i), dsf, dq[dt]);
        }
    }
    if (r < nrow) {
        T* dst = (T*)a.dq + (size_t)qrow * a.ldq + head * DK + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) store4<T>(dst + dt * 16, dq[dt] * a.scale);
    }
}

// ---- dk, dv: one workgroup per (utterance, shared head, 64 keys, range of packed rows) ----------------------------
template <typename T, int DK>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void xattn_dkv_kernel(XArgs a) {
    typedef XTile<T, DK> TL;
    typedef typename TL::frag_t frag_t;
    constexpr int KS = TL::KS, DT = TL::DT;
    // stage s: Q tile, dO tile (rotation 2: read both ways), then the 64 lse and 64 delta values of those rows
    constexpr int STAGE = 2 * TL::BYTES + 512;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

    int b, kvh, blk;
    if (!fs2_pair_order_decode(a.order, b, kvh, blk)) return;
    const int split = blk % a.nsplit;
    blk /= a.nsplit;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, q0, lenq);
    x_range(a.cu_k, b, a.Mk, k0, lenk);
    if (blk * 64 >= lenk) return;
    const int nrow = lenq * a.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int key = blk * 64 + wave * 16 + i, kc = min(key, lenk - 1);
    const int ntiles = (nrow + 63) / 64, per = (ntiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(t0 + per, ntiles);

    const T* __restrict__ qb = (const T*)a.q + (size_t)q0 * a.ldq + kvh * a.g * DK;
    const T* __restrict__ db = (const T*)a.dctx + (size_t)q0 * a.ldo + kvh * a.g * DK;
    auto stage = [&](int qt, int st) __attribute__((always_inline)) {
        unsigned char* d = smem + st * STAGE;
        TL::template stage_rows<2, 4>(a, qb, a.ldq, qt * 64, nrow, d, wave, lane);
        TL::template stage_rows<2, 4>(a, db, a.ldo, qt * 64, nrow, d + TL::BYTES, wave, lane);
        if (wave < 2) {
            const int r = min(qt * 64 + lane, nrow - 1), q = x_query(a, r);
            const size_t at = (size_t)(kvh * a.g + r - q * a.g) * a.Mq + q0 + q;
            __builtin_amdgcn_global_load_lds((x_gbl_void*)((wave ? a.delta : a.lse) + at),
                                             (x_lds_void*)(d + 2 * TL::BYTES + wave * 256), 4, 0, 0);
        }
    };
    if (t0 < t1) stage(t0, 0);
    frag_t kf[KS], vf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        kf[ks] = *(const frag_t*)((const T*)a.k + (size_t)(k0 + kc) * a.ldk + kvh * DK + ks * 32 + g * 8);
        vf[ks] = *(const frag_t*)((const T*)a.v + (size_t)(k0 + kc) * a.ldv + kvh * DK + ks * 32 + g * 8);
    }
    f32x4 dk_[DT], dv_[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dk_[dt] = dv_[dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    for (int qt = t0; qt < t1; ++qt) {
        vm_wait_barrier<0>();
        const int st = (qt - t0) & 1;
        if (qt + 1 < t1) stage(qt + 1, st ^ 1);
        const unsigned char* Qs = smem + st * STAGE;
        const unsigned char* Ds = Qs + TL::BYTES;
        const float* lse_s = (const float*)(Qs + 2 * TL::BYTES);
        f32x4 s[4], dp[4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) s[nt] = dp[nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            frag_t f[4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) f[nt] = TL::template row_frag<2>(Qs, nt * 16 + i, ks, g);
            mma16_multi<4>(f, kf[ks], s);            // rows: packed rows qt 64 + 16 nt + 4 g + e, column: key i
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) f[nt] = TL::template row_frag<2>(Ds, nt * 16 + i, ks, g);
            mma16_multi<4>(f, vf[ks], dp);
        }
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            const f32x4 lse4 = *(const f32x4*)(lse_s + nt * 16 + 4 * g);
            const f32x4 del4 = *(const f32x4*)(lse_s + 64 + nt * 16 + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = qt * 64 + nt * 16 + 4 * g + e;
                const bool ok = r < nrow;
                const float p = ok ? __builtin_amdgcn_exp2f(fmaf(s[nt][e], a.scale_log2e, -lse4[e])) : 0.f;
                float mul = 1.0f;
                if (a.drop.thresh) {
                    const int rr = min(r, nrow - 1), q = x_query(a, rr);
                    Dropout dh = a.drop;
                    dh.stream += (uint32_t)(kvh * a.g + rr - q * a.g);
                    mul = drop_mul(dh, (uint32_t)(q0 + q), (uint32_t)kc);
                }
                dp[nt][e] = ok ? p * (dp[nt][e] * mul - del4[e]) : 0.f;
                s[nt][e] = p * mul;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const frag_t pf = x_pack<T>(s[2 * c], s[2 * c + 1]), dsf = x_pack<T>(dp[2 * c], dp[2 * c + 1]);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                dv_[dt] = mma16(TL::template col_frag<2>(Ds, c, dt, g, i), pf, dv_[dt]);
                dk_[dt] = mma16(TL::template col_frag<2>(Qs, c, dt, g, i), dsf, dk_[dt]);
            }
        }
    }
    if (key >= lenk) return;
    if (a.nsplit == 1) {
        T* dk = (T*)a.dk + (size_t)(k0 + key) * a.ldk + kvh * DK + 4 * g;
        T* dv = (T*)a.dv + (size_t)(k0 + key) * a.ldv + kvh * DK + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            store4<T>(dk + dt * 16, dk_[dt] * a.scale);
            store4<T>(dv + dt * 16, dv_[dt]);
        }
    } else {                          // part[split][dk, dv][Mk][KV * DK]
        const size_t w = (size_t)a.KV * DK, half = (size_t)a.Mk * w;
        float* dst = a.part + (size_t)split * 2 * half + (size_t)(k0 + key) * w + kvh * DK + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            *(f32x4*)(dst + dt * 16) = dk_[dt] * a.scale;
            *(f32x4*)(dst + half + dt * 16) = dv_[dt];
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void xattn_dkv_sum_kernel(XArgs a, int B, int dk) {
    const int w = a.KV * dk, wv = w >> 2;
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    const int rows = min(max(a.cu_k[B], 0), a.Mk);
    const long long n = (long long)rows * wv;
    if (idx >= 2 * n) return;
    const bool is_v = idx >= n;
    const long long e = is_v ? idx - n : idx;
    const int m = (int)(e / wv), c = (int)(e % wv) * 4;
    const size_t half = (size_t)a.Mk * w;
    const float* src = a.part + (is_v ? half : 0) + (size_t)m * w + c;
    f32x4 sum = *(const f32x4*)src;
    for (int s = 1; s < a.nsplit; ++s) sum += *(const f32x4*)(src + (size_t)s * 2 * half);
    if (is_v)
        store4<T>((T*)a.dv + (size_t)m * a.ldv + c, sum);
    else
        store4<T>((T*)a.dk + (size_t)m * a.ldk + c, sum);
}

// ---- mass: one workgroup per (utterance, head, KB keys, range of queries) ------------------------------------------
// The KB keys stay in LDS; the four waves stream the queries, 16 at a time, straight from memory into registers (each row is
// read once per key block).  S^T = K Q^T: a lane owns one query and 4 keys of every 16, adds its own queries' weights over the
// whole loop, and the 16 queries of a row of lanes meet only at the end.
template <typename T, int DK, int KB>
__global__ __launch_bounds__(256, 1) void xattn_mass_kernel(XArgs a) {
    typedef XTile<T, DK, KB> TL;
    typedef typename TL::frag_t frag_t;
    constexpr int KS = TL::KS, NT = KB / 16;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    int b, h, blk;
    if (!fs2_pair_order_decode(a.order, b, h, blk)) return;
    const int split = blk % a.nsplit;
    blk /= a.nsplit;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, q0, lenq);
    x_range(a.cu_k, b, a.Mk, k0, lenk);
    if (blk * KB >= lenk) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int kvh = h / a.g;
    TL::template stage<1, 4>((const T*)a.k + (size_t)k0 * a.ldk + kvh * DK, a.ldk, blk * KB, lenk, smem, wave, lane);
    const int ntiles = (lenq + 15) / 16, per = (ntiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(t0 + per, ntiles);
    f32x4 acc[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const T* __restrict__ qb = (const T*)a.q + (size_t)q0 * a.ldq + h * DK;
    const float* __restrict__ lse = a.lse + (size_t)h * a.Mq + q0;
    vm_wait_barrier<0>();
    for (int qt = t0 + wave; qt < t1; qt += 4) {
        const int q = qt * 16 + i, qc = min(q, lenq - 1);
        frag_t qf[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const frag_t*)(qb + (size_t)qc * a.ldq + ks * 32 + g * 8);
        float l = lse[qc];
        if (q >= lenq || !(fabsf(l) < INFINITY)) l = INFINITY;          // no such query: no weight
#pragma unroll
        for (int n4 = 0; n4 < NT; n4 += 4) {
            f32x4 s[4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) s[nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                frag_t kf[4];
#pragma unroll
                for (int nt = 0; nt < 4; ++nt) kf[nt] = TL::template row_frag<1>(smem, (n4 + nt) * 16 + i, ks, g);
                mma16_multi<4>(kf, qf[ks], s);
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n4 + nt][e] += __builtin_amdgcn_exp2f(fmaf(s[nt][e], a.scale_log2e, -l));
        }
    }
    __syncthreads();
    float* red = (float*)smem;          // [4][KB]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v = row16_sum(acc[nt][e]);
            if (i == 0) red[wave * KB + nt * 16 + 4 * g + e] = v;
        }
    __syncthreads();
    const int key = blk * KB + tid;
    if (tid < KB && key < lenk) {
        const float v = red[tid] + red[KB + tid] + red[2 * KB + tid] + red[3 * KB + tid];
        float* dst = a.nsplit == 1 ? a.mass : a.part + (size_t)split * a.H * a.Mk;
        dst[(size_t)h * a.Mk + k0 + key] = v;
    }
}

__global__ __launch_bounds__(256) void xattn_mass_sum_kernel(XArgs a, int B) {
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    const int rows = min(max(a.cu_k[B], 0), a.Mk);
    if (idx >= (long long)a.H * rows) return;
    const size_t at = (size_t)(idx / rows) * a.Mk + idx % rows, step = (size_t)a.H * a.Mk;
    float sum = a.part[at];
    for (int s = 1; s < a.nsplit; ++s) sum += a.part[s * step + at];
    a.mass[at] = sum;
}

constexpr int X_MASS_KB = 128;

static int x_dkv_split(int B, int max_q, int max_k, int H, int KV) {
    const long items = (long)B * KV * ((max_k + 63) / 64), tiles = ((long)max_q * (H / KV) + 63) / 64;
    if (items >= 256 || tiles < 4) return 1;
    const long want = 512 / items, most = tiles / 2, n = want < most ? want : most;
    return (int)(n < 1 ? 1 : (n > 32 ? 32 : n));
}
static int x_mass_split(int B, int max_q, int max_k, int H) {
    const long items = (long)B * H * ((max_k + X_MASS_KB - 1) / X_MASS_KB), tiles = (max_q + 15) / 16;
    if (items >= 256 || tiles < 8) return 1;
    const long want = 512 / items, most = tiles / 4, n = want < most ? want : most;
    return (int)(n < 1 ? 1 : (n > 64 ? 64 : n));
}

template <typename T, int DK>
static int launch_xattn_bwd(XArgs& a, int B, int max_q, int max_k, int dk, hipStream_t stream) {
    constexpr int lds_dq = 4 * XTile<T, DK>::BYTES, lds_dkv = lds_dq + 2 * 512;
    static unsigned long long ok_dq = 0, ok_dkv = 0;
    fs2_allow_lds((const void*)xattn_dq_kernel<T, DK>, lds_dq, &ok_dq);
    fs2_allow_lds((const void*)xattn_dkv_kernel<T, DK>, lds_dkv, &ok_dkv);
    if (max_q > 0) {
        const dim3 grid = fs2_pair_order_grid(a.order, (max_q * a.g + 63) / 64, a.KV, B, true);
        hipLaunchKernelGGL((xattn_dq_kernel<T, DK>), grid, dim3(256), lds_dq, stream, a);
        FS2_CHECK_LAUNCH("fs2_cross_attention_bwd(dq)");
    }
    if (max_k > 0) {
        const dim3 grid = fs2_pair_order_grid(a.order, ((max_k + 63) / 64) * a.nsplit, a.KV, B, true);
        hipLaunchKernelGGL((xattn_dkv_kernel<T, DK>), grid, dim3(256), lds_dkv, stream, a);
        FS2_CHECK_LAUNCH("fs2_cross_attention_bwd(dk, dv)");
        if (a.nsplit > 1) {
            const long long n = 2LL * a.Mk * (a.KV * dk / 4);
            hipLaunchKernelGGL(xattn_dkv_sum_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a, B, dk);
            FS2_CHECK_LAUNCH("fs2_cross_attention_bwd(sum)");
        }
    }
    return FS2_OK;
}

template <typename T, int DK>
static int launch_xattn_mass(XArgs& a, int B, int max_k, hipStream_t stream) {
    constexpr int lds = XTile<T, DK, X_MASS_KB>::BYTES;
    static unsigned long long ok = 0;
    fs2_allow_lds((const void*)xattn_mass_kernel<T, DK, X_MASS_KB>, lds, &ok);
    const dim3 grid = fs2_pair_order_grid(a.order, ((max_k + X_MASS_KB - 1) / X_MASS_KB) * a.nsplit, a.H, B, true);
    hipLaunchKernelGGL((xattn_mass_kernel<T, DK, X_MASS_KB>), grid, dim3(256), lds, stream, a);
    FS2_CHECK_LAUNCH("fs2_cross_attention_mass");
    if (a.nsplit > 1) {
        const long long n = (long long)a.H * a.Mk;
        hipLaunchKernelGGL(xattn_mass_sum_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a, B);
        FS2_CHECK_LAUNCH("fs2_cross_attention_mass(sum)");
    }
    return FS2_OK;
}

}  // namespace fs2

using namespace fs2;

// workspace: delta [n_heads][Mq] (rounded up to 16 bytes), then the partial dk, dv of the row ranges
static inline long long x_delta_floats(int H, int Mq) { return ((long long)H * Mq + 3) / 4 * 4; }

extern "C" long long fs2_cross_attention_bwd_workspace(int B, int max_q, int max_k, int Mq, int Mk, int n_heads, int n_kv_heads,
                                                       int dk, int dtype) {
    (void)dtype;
    if (B <= 0 || max_q <= 0 || max_k <= 0 || Mq <= 0 || Mk <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads) return 16;
    const int n = x_dkv_split(B, max_q, max_k, n_heads, n_kv_heads);
    return (x_delta_floats(n_heads, Mq) + (n > 1 ? 2LL * n * Mk * n_kv_heads * dk : 0)) * (long long)sizeof(float);
}

extern "C" int fs2_cross_attention_bwd(const void* q, const void* k, const void* v, const void* ctx, const void* dctx,
                                       const float* lse, void* dq, void* dk_out, void* dv, const int* cu_q, const int* cu_k,
                                       void* workspace, int B, int max_q, int max_k, int Mq, int Mk, int n_heads, int n_kv_heads,
                                       int dk, int ldq, int ldk, int ldv, int ldo, int dtype, unsigned seed, unsigned stream_id,
                                       float rate, hipStream_t stream) {
    const int rc = fs2_x_check("fs2_cross_attention_bwd", q, k, cu_q, cu_k, B, max_q, max_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq,
                               ldk, dtype);
    if (rc != FS2_OK) return rc;
    const int epv = dtype == 0 ? 4 : 8;
    FS2_CHECK_ARG(rate >= 0.f && rate < 1.f, "fs2_cross_attention_bwd: dropout rate must be in [0, 1)");
    FS2_CHECK_ARG((Mq == 0 || (ctx && dctx && lse && dq)) && (Mk == 0 || (v && dk_out && dv)), "fs2_cross_attention_bwd: null argument");
    FS2_CHECK_ARG((((uintptr_t)v | (uintptr_t)ctx | (uintptr_t)dctx | (uintptr_t)dq | (uintptr_t)dk_out | (uintptr_t)dv) & 15) == 0,
                  "fs2_cross_attention_bwd: unaligned pointers");
    FS2_CHECK_ARG(ldv >= n_kv_heads * dk && ldo >= n_heads * dk && ldv % epv == 0 && ldo % epv == 0,
                  "fs2_cross_attention_bwd: bad leading dims ldv=%d ldo=%d", ldv, ldo);
    if (max_q == 0 && max_k == 0) return FS2_OK;
    FS2_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0,
                  "fs2_cross_attention_bwd: fs2_cross_attention_bwd_workspace bytes, 16-byte aligned, are needed");
    XArgs a = fs2_x_args(q, k, v, cu_q, cu_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq, ldk, ldv, ldo);
    a.ctx = (void*)ctx; a.dctx = dctx; a.lse = (float*)lse; a.dq = dq; a.dk = dk_out; a.dv = dv;
    a.drop = fs2_make_dropout(seed, stream_id, rate);
    a.delta = (float*)workspace;
    a.part = (float*)workspace + x_delta_floats(n_heads, Mq);
    a.nsplit = max_q > 0 && max_k > 0 ? x_dkv_split(B, max_q, max_k, n_heads, n_kv_heads) : 1;
#define FS2_X(TT, DKK) return launch_xattn_bwd<TT, DKK>(a, B, max_q, max_k, dk, stream)
    if (dtype == 0) {
        if (dk == 32) FS2_X(float, 32);
        if (dk == 64) FS2_X(float, 64);
        if (dk == 96) FS2_X(float, 96);
        FS2_X(float, 128);
    }
    if (dk == 32) FS2_X(bf16_t, 32);
    if (dk == 64) FS2_X(bf16_t, 64);
    if (dk == 96) FS2_X(bf16_t, 96);
    FS2_X(bf16_t, 128);
#undef FS2_X
}

extern "C" long long fs2_cross_attention_mass_workspace(int B, int max_q, int max_k, int Mk, int n_heads, int n_kv_heads, int dk,
                                                        int dtype) {
    (void)n_kv_heads; (void)dk; (void)dtype;
    if (B <= 0 || max_q <= 0 || max_k <= 0 || Mk <= 0 || n_heads <= 0) return 0;
    const int n = x_mass_split(B, max_q, max_k, n_heads);
    return n > 1 ? (long long)n * n_heads * Mk * (long long)sizeof(float) : 0;
}

extern "C" int fs2_cross_attention_mass(const void* q, const void* k, const float* lse, float* mass, const int* cu_q,
                                        const int* cu_k, void* workspace, int B, int max_q, int max_k, int Mq, int Mk, int n_heads,
                                        int n_kv_heads, int dk, int ldq, int ldk, int dtype, hipStream_t stream) {
    const int rc = fs2_x_check("fs2_cross_attention_mass", q, k, cu_q, cu_k, B, max_q, max_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq,
                               ldk, dtype);
    if (rc != FS2_OK) return rc;
    FS2_CHECK_ARG((lse || Mq == 0) && (mass || Mk == 0), "fs2_cross_attention_mass: null lse or mass");
    if (max_k == 0) return FS2_OK;
    XArgs a = fs2_x_args(q, k, nullptr, cu_q, cu_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq, ldk, 0, 0);
    a.lse = (float*)lse;
    a.mass = mass;
    a.nsplit = max_q > 0 ? x_mass_split(B, max_q, max_k, n_heads) : 1;
    a.part = (float*)workspace;
    FS2_CHECK_ARG(a.nsplit == 1 || workspace, "fs2_cross_attention_mass: this shape needs fs2_cross_attention_mass_workspace bytes");
#define FS2_X(TT, DKK) return launch_xattn_mass<TT, DKK>(a, B, max_k, stream)
    if (dtype == 0) {
        if (dk == 32) FS2_X(float, 32);
        if (dk == 64) FS2_X(float, 64);
        if (dk == 96) FS2_X(float, 96);
        FS2_X(float, 128);
    }
    if (dk == 32) FS2_X(bf16_t, 32);
    if (dk == 64) FS2_X(bf16_t, 64);
    if (dk == 96) FS2_X(bf16_t, 96);
    FS2_X(bf16_t, 128);
#undef FS2_X
}
