// Cross attention over packed ragged batches: queries [Mq] of one matrix, keys / values [Mk] of another, utterance b of the
// first against utterance b of the second (cu_q, cu_k), g = H / KV query heads to a key / value head.
//   S = q k^T / sqrt(dk);  P = softmax over the utterance's keys;  ctx = dropout(P) v;  lse = log2 sum exp2(S log2 e)
// An utterance without keys has ctx = 0 and lse = -inf.  Running maximum and sum in fp32; bf16 rounds the result alone (P goes into its
// product as two bf16 numbers).
//
// Orientation as in attention.hip: S^T = K Q^T and O^T = V^T P^T, so that a lane owns one query row and every softmax statistic
// is lane-local; the accumulator layout of P^T is used as the next operand, V is read transposed from LDS with the same map.
//   rows kernel: 4 waves x 16 QT packed rows; K / V tiles for all four in LDS: bf16 64 keys, two stages; fp32 32 keys in three bf16
//                planes, one stage, the next tile on its way in registers.
//   few kernel:  at most 16 packed rows per pair (one frame at a time): the four waves share the rows and split the KEYS,
//                each with its own 32-key tiles in wave-private LDS (fp32: K straight into registers); one merge.
// Where the pairs alone do not fill the chip, ranges of keys go to `nsplit` workgroups and a second kernel merges.
//
// Measured (floor: bytes at 5.2 TB/s, or products at 1198 TFLOP/s bf16, a sixth of that fp32, whichever is longer):
//   one frame of 256 sentences, 8 heads on 2 of 64, 160 keys, bf16: 8.1 us for 21 MB (2.6 TB/s; floor 4.1); one sentence 5.8 us, of
//     which the launch is 3.8.
//   32 x 800 frames over 120 phones, 2 heads of 128, bf16: 15.9 us for 31 MB (1.9 TB/s; floor 6.0), 18.9 with dropout.  Two key tiles leave
//     nothing to overlap: a workgroup waits for its queries and first keys, multiplies, and writes.  Over 900 keys 50.8 us, 23.6 GFLOP = 465
//     TFLOP/s (floor 20): splitting P costs 10 us of it, in vector instructions.
//   32 x 120 phones over 810 frames, 4 heads on 2 of 96, fp32: 60 us, 4.8 GFLOP = 80 TFLOP/s (floor 24), 6 of it the merge, 67 with
//     dropout.  The matrix pipe is busy a third of the time; splitting, softmax and LDS reads (31 % of their cycles bank conflicts) fill the
//     rest, and three workgroups on a CU overlap only part of it.
#include "cross_attention.h"

namespace fs2 {

// ctx rows of an utterance without keys
template <typename T, int DK>
__device__ __forceinline__ void x_zero_rows(const XArgs& a, int q0, int kvh, int r_begin, int r_end) {
    constexpr int SL = DK / 4;
    for (int e = threadIdx.x; e < (r_end - r_begin) * SL; e += blockDim.x) {
        const int r = r_begin + e / SL, q = x_query(a, r), h = kvh * a.g + r - q * a.g;
        store4<T>((T*)a.ctx + (size_t)(q0 + q) * a.ldo + h * DK + (e % SL) * 4, (f32x4){0.f, 0.f, 0.f, 0.f});
        if (a.lse && e % SL == 0) a.lse[(size_t)h * a.Mq + q0 + q] = -INFINITY;
    }
}

template <typename E, int DK, int QT, bool DROP>
__global__ __launch_bounds__(256, E::PL == 3 && DK < 128 ? 3 : 2) void xattn_rows_kernel(XArgs a) {
    typedef typename E::mem T;
    constexpr int KB = x_kb<E>(), NT = KB / 16, NC = KB / 32, NST = E::PL == 1 ? 2 : 1;
    typedef XTile<E, DK, KB, 1> TK;
    typedef XTile<E, DK, KB, 2> TV;
    typedef typename TK::frag_t frag_t;
    constexpr int KS = TK::KS, DT = TK::DT, BQ = 64 * QT, STAGE = TK::BYTES + TV::BYTES;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];     // stage s: K tile, V tile

    int b, kvh, blk, split;
    if (!x_decode(a, a.KV, b, kvh, blk, split)) return;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, a.max_q, q0, lenq);
    x_range(a.cu_k, b, a.Mk, a.max_k, k0, lenk);
    const int nrow = lenq * a.g;
    if (blk * BQ >= nrow) return;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int ntiles = (lenk + KB - 1) / KB, per = a.nsplit == 1 ? ntiles : (ntiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(t0 + per, ntiles);
    if (lenk == 0 && a.nsplit == 1) {
        x_zero_rows<T, DK>(a, q0, kvh, blk * BQ, min(nrow, blk * BQ + BQ));
        return;
    }
    if (t0 >= t1) {         // this split has no keys: (max, sum) = (-inf, 0)
        for (int r = blk * BQ + tid; r < min(nrow, blk * BQ + BQ); r += 256) {
            const int q = x_query(a, r), head = kvh * a.g + r - q * a.g;
            float* ml = a.part + (size_t)a.nsplit * a.slots * a.H * DK + (((size_t)split * a.H + head) * a.slots + b * a.max_q + q) * 2;
            ml[0] = -INFINITY;
            ml[1] = 0.f;
        }
        return;
    }
    const T* __restrict__ kb = (const T*)a.k + (size_t)k0 * a.ldk + kvh * DK;
    const T* __restrict__ vb = (const T*)a.v + (size_t)k0 * a.ldv + kvh * DK;
    XFetch<E, DK, KB, 1, 4> fk(a.ldk, wave, lane);
    XFetch<E, DK, KB, 2, 4> fv(a.ldv, wave, lane);
    auto fetch = [&](int kt, int st) __attribute__((always_inline)) {
        unsigned char* d = smem + st * STAGE;
        fk.fetch(kb + (size_t)kt * KB * a.ldk, a.ldk, lenk - kt * KB, d, wave, lane);
        fv.fetch(vb + (size_t)kt * KB * a.ldv, a.ldv, lenk - kt * KB, d + TK::BYTES, wave, lane);
    };
    fetch(t0, 0);

    // the queries, through the other stage (bf16) or ahead of the first tile (fp32): every wave has read its own before the barrier
    // behind which that memory is filled again
    frag_t qf[QT][KS];
    {
        typedef XTile<E, DK, 16 * QT, 1> TQ;
        unsigned char* own = smem + (NST == 2 ? STAGE : 0) + wave * TQ::BYTES;
        XRows<E, DK, 16 * QT> rows(a.ldq, lane);
        rows.start(a, (const T*)a.q + (size_t)q0 * a.ldq + kvh * a.g * DK, a.ldq, min(blk * BQ + wave * 16 * QT, nrow - 1), nrow, own, lane);
        rows.finish(own, lane);
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qf[t][ks] = TQ::row_frag(own, t * 16 + i, ks, g);
    }

    f32x4 o[QT][DT];
    float m_run[QT], l_part[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        m_run[t] = -INFINITY;
        l_part[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[t][dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    for (int kt = t0; kt < t1; ++kt) {
        const int st = NST == 2 ? (kt - t0) & 1 : 0;
        unsigned char* Ks = smem + st * STAGE;
        unsigned char* Vs = Ks + TK::BYTES;
        if constexpr (E::PL == 1) {
            vm_wait_barrier<0>();         // tile kt has landed; every wave is done with the other stage
        } else {
            __syncthreads();                             // every wave is done with the tile (or its queries) before
            fk.put(Ks, wave, lane);
            fv.put(Vs, wave, lane);
            __syncthreads();
            if (kt + 1 < t1) fetch(kt + 1, 0);
        }

        f32x4 s[QT][NT];
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[t][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            frag_t kf[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) kf[nt] = TK::row_frag(Ks, nt * 16 + i, ks, g);
#pragma unroll
            for (int t = 0; t < QT; ++t) x_mma<E, NT>(kf, qf[t][ks], s[t]);
        }
        // bf16: the V^T fragments of the first 32 keys are requested now and land under the softmax, those of the second 32 behind the first
        // ones' products (both at once spill at dk = 128: 32 x 800 rows over 120 keys 16.5 us against 16.2, with dropout 21.0 against 19.2).
        // The next tile's DMA is issued behind all of them: the compiler lets no transposed LDS read pass an LDS-DMA in flight (it
        // waits vmcnt(0)), so in front of them it would be waited for here.
        frag_t vf[E::PL == 1 ? NC : 1][DT];
        if constexpr (E::PL == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) vf[0][dt] = TV::col_frag(Vs, 0, dt, g, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        const int kbase = kt * KB + 4 * g;
        if (kt * KB + KB > lenk) {
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (kbase + nt * 16 + r >= lenk) s[t][nt][r] = -INFINITY;
        }
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            float m_loc = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r) m_loc = fmaxf(m_loc, s[t][nt][r]);
            m_loc = rows_max(m_loc) * a.scale_log2e;
            // the reference point moves only when a score is more than 2^8 above it (weights then stay below 2^8, which costs fp32
            // sums and bf16 weights nothing): a row's later tiles hardly ever rescale
            const bool moves = m_loc > m_run[t] + 8.0f;
            float m_use = moves ? m_loc : m_run[t];
            if (kt > t0 && !__all(!moves)) {
                const float alpha = m_run[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[t] - m_use);
                l_part[t] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[t][dt][r] *= alpha;
            }
            m_run[t] = m_use;
            m_use = m_use == -INFINITY ? 0.f : m_use;                    // nothing but -inf scores so far: no NaN
            float psum = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[t][nt][r], a.scale_log2e, -m_use));
                    s[t][nt][r] = p;
                    psum += p;
                }
            l_part[t] += psum;
            if constexpr (DROP) {      // the sum above is over the undropped probabilities
                const int row = min(blk * BQ + (wave * QT + t) * 16 + i, nrow - 1), q = x_query(a, row);
                Dropout dh = a.drop;
                dh.stream += (uint32_t)(kvh * a.g + row - q * a.g);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        s[t][nt][r] = drop_keep(dh, (uint32_t)(q0 + q), (uint32_t)(kbase + nt * 16 + r)) ? s[t][nt][r] * dh.inv_keep : 0.f;
            }
        }
        if constexpr (E::PL == 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            frag_t pf[QT];
            if constexpr (E::PL == 1) {
                if (c == NC - 1) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) vf[c][dt] = TV::col_frag(Vs, c, dt, g, i);
                    if (kt + 1 < t1) fetch(kt + 1, st ^ 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (kt * KB + KB > lenk) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) x_keep_rows(vf[c][dt], lenk - kt * KB - 32 * c, g);
                }
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    frag_t rest;
                    x_pack_weights(s[t][2 * c], s[t][2 * c + 1], pf[t], rest);
                    x_mma<E, DT>(vf[c], rest, o[t]);
                    x_mma<E, DT>(vf[c], pf[t], o[t]);
                }
            } else {
#pragma unroll
                for (int t = 0; t < QT; ++t) pf[t] = x_pack<E>(s[t][2 * c], s[t][2 * c + 1]);
#pragma unroll
                for (int dt0 = 0; dt0 < DT; dt0 += 2) {
                    frag_t v2[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) v2[u] = TV::col_frag(Vs, c, dt0 + u, g, i);
#pragma unroll
                    for (int t = 0; t < QT; ++t) x_mma<E, 2>(v2, pf[t], &o[t][dt0]);
                }
            }
        }
    }
    __syncthreads();                                     // the tiles' memory serves the waves' results now
    unsigned char* own = smem + wave * x_out_bytes<float, DK>();
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const float l = rows_sum(l_part[t]);
        const int first = blk * BQ + (wave * QT + t) * 16, r = first + i;
        const int q = x_query(a, min(r, nrow - 1)), head = kvh * a.g + min(r, nrow - 1) - q * a.g;
        if (a.nsplit == 1) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;        // no score above -inf: a zero row
            if (a.lse && g == 0 && r < nrow) a.lse[(size_t)head * a.Mq + q0 + q] = m_run[t] + __log2f(l);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[t][dt] *= inv;
            x_store_rows<T, DK>(a, (T*)a.ctx, a.ldo, q0, kvh, first, nrow, o[t], own, lane);
        } else {
            const int d = a.H * DK;
            x_store_rows<float, DK>(a, a.part + (size_t)split * a.slots * d, d, b * a.max_q, kvh, first, nrow, o[t], own, lane);
            float* ml = a.part + (size_t)a.nsplit * a.slots * d + (((size_t)split * a.H + head) * a.slots + b * a.max_q + q) * 2;
            if (g == 0 && r < nrow) {
                ml[0] = m_run[t];
                ml[1] = l;
            }
        }
    }
}

// At most 16 packed rows per (utterance, shared head).  grid (nsplit, KV, B); wave w takes the 32-key tiles t0 + w, + 4, ..
// 256 sentences x 2000 keys, 2 heads of 128, bf16: 102 us for 524 MB (5.1 TB/s, a large copy's rate); short key lists are a chain of dependent
// reads (one sentence of 120 keys: 5.1 us in the kernel; with eight waves instead of four 0.9 more).
template <typename E, int DK>
__global__ __launch_bounds__(256, 1) void xattn_few_kernel(XArgs a) {
    typedef typename E::mem T;
    typedef XTile<E, DK, 32, 1> TK;
    typedef XTile<E, DK, 32, 2> TV;
    typedef typename TK::frag_t frag_t;
    constexpr int KS = TK::KS, DT = TK::DT;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];     // wave w: V tile at w * BYTES; then the merge
    const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, a.max_q, q0, lenq);
    x_range(a.cu_k, b, a.Mk, a.max_k, k0, lenk);
    const int nrow = min(lenq * a.g, 16);
    if (nrow == 0) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15;
    if (lenk == 0 && a.nsplit == 1) {
        x_zero_rows<T, DK>(a, q0, kvh, 0, nrow);
        return;
    }
    const int rc = min(i, nrow - 1), q = x_query(a, rc), head = kvh * a.g + rc - q * a.g, qrow = q0 + q;
    const int ntiles = (lenk + 31) / 32, per = a.nsplit == 1 ? ntiles : (ntiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(t0 + per, ntiles);
    frag_t qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = x_load<E>((const T*)a.q + (size_t)qrow * a.ldq + head * DK + ks * 32 + g * 8);

    const T* __restrict__ kb = (const T*)a.k + (size_t)k0 * a.ldk + kvh * DK;
    const T* __restrict__ vb = (const T*)a.v + (size_t)k0 * a.ldv + kvh * DK;
    constexpr int KL = E::PL == 1 ? TK::BYTES : 0;          // K goes through LDS too (fp32: three planes of both do not fit)
    unsigned char* Ks = smem + wave * (TV::BYTES + KL);
    unsigned char* Vs = Ks + KL;
    XFetch<E, DK, 32, 1, 1> fk(a.ldk, 0, lane);
    XFetch<E, DK, 32, 2, 1> fv(a.ldv, 0, lane);
    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_part = 0.f;
    for (int kt = t0 + wave; kt < t1; kt += 4) {
        if constexpr (E::PL == 1) fk.fetch(kb + (size_t)kt * 32 * a.ldk, a.ldk, lenk - kt * 32, Ks, 0, lane);
        fv.fetch(vb + (size_t)kt * 32 * a.ldv, a.ldv, lenk - kt * 32, Vs, 0, lane);
        f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        if constexpr (E::PL == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // this wave's tiles have landed (no other wave reads them)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            frag_t f[2];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                if constexpr (E::PL == 1) f[nt] = TK::row_frag(Ks, nt * 16 + i, ks, g);
                else f[nt] = x_load<E>(kb + (size_t)min(kt * 32 + nt * 16 + i, lenk - 1) * a.ldk + ks * 32 + g * 8);
            }
            x_mma<E, 2>(f, qf[ks], s);
        }
        const int kbase = kt * 32 + 4 * g;
        float m_loc = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (kbase + nt * 16 + r >= lenk) s[nt][r] = -INFINITY;
                m_loc = fmaxf(m_loc, s[nt][r]);
            }
        m_loc = rows_max(m_loc) * a.scale_log2e;
        const float m_new = fmaxf(m_run, m_loc), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
        m_run = m_new;
        float psum = 0.f;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[nt][r] = __builtin_amdgcn_exp2f(fmaf(s[nt][r], a.scale_log2e, -m_use));
                psum += s[nt][r];
            }
        l_part = fmaf(l_part, alpha, psum);
        if (a.drop.thresh) {
            Dropout dh = a.drop;
            dh.stream += (uint32_t)head;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[nt][r] *= drop_mul(dh, (uint32_t)qrow, (uint32_t)(kbase + nt * 16 + r));
        }
        frag_t pf, rest;
        if constexpr (E::PL == 1) {
            x_pack_weights(s[0], s[1], pf, rest);
        } else {
            pf = x_pack<E>(s[0], s[1]);
            fv.put(Vs, 0, lane);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (int dt0 = 0; dt0 < DT; dt0 += 2) {
            frag_t v2[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                v2[u] = TV::col_frag(Vs, 0, dt0 + u, g, i);
                if constexpr (E::PL == 1)
                    if (kt * 32 + 32 > lenk) x_keep_rows(v2[u], lenk - kt * 32, g);
                o[dt0 + u] = o[dt0 + u] * alpha;
            }
            if constexpr (E::PL == 1) x_mma<E, 2>(v2, rest, &o[dt0]);
            x_mma<E, 2>(v2, pf, &o[dt0]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // read before the next tile overwrites it
    }
    // merge of the four waves: lane (g, i) of wave w holds row i, columns 16 dt + 4 g ..
    const float l = rows_sum(l_part);
    __syncthreads();
    float* mo = (float*)smem;                       // [4][16][DK]
    float* mm = mo + 4 * 16 * DK;                   // [4][16] max, then sum
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *(f32x4*)(mo + (wave * 16 + i) * DK + dt * 16 + 4 * g) = o[dt];
    if (g == 0) {
        mm[wave * 16 + i] = m_run;
        mm[64 + wave * 16 + i] = l;
    }
    __syncthreads();
    constexpr int SL = DK / 4;
    for (int e = tid; e < nrow * SL; e += 256) {
        const int r = e / SL, c = (e % SL) * 4;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, mm[w * 16 + r]);
        const float mu = mx == -INFINITY ? 0.f : mx;
        float L = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(mm[w * 16 + r] - mu);
            L = fmaf(mm[64 + w * 16 + r], f, L);
            acc += *(const f32x4*)(mo + (w * 16 + r) * DK + c) * f;
        }
        const int qq = x_query(a, r), h = kvh * a.g + r - qq * a.g;
        if (a.nsplit == 1) {
            store4<T>((T*)a.ctx + (size_t)(q0 + qq) * a.ldo + h * DK + c, acc * (L == 0.f ? 0.f : 1.0f / L));
            if (a.lse && c == 0) a.lse[(size_t)h * a.Mq + q0 + qq] = mx + __log2f(L);
        } else {
            const size_t d = (size_t)a.H * DK;
            const int slot = b * a.max_q + qq;
            *(f32x4*)(a.part + ((size_t)split * a.slots + slot) * d + h * DK + c) = acc;
            float* ml = a.part + (size_t)a.nsplit * a.slots * d + (((size_t)split * a.H + h) * a.slots + slot) * 2;
            if (c == 0) {
                ml[0] = mx;
                ml[1] = L;
            }
        }
    }
}

// Merge of the key ranges, many rows: one lane per (row, four channels), the few ranges in a loop.  A range without keys wrote no
// partial context (its sum is 0): read, not used.
template <typename T>
__global__ __launch_bounds__(256) void xattn_combine_kernel(XArgs a, int B, int dk) {
    const int d = a.H * dk, dv = d >> 2;
    const unsigned idx = blockIdx.x * 256 + threadIdx.x, slot = idx / (unsigned)dv;
    if (slot >= (unsigned)B * (unsigned)a.max_q) return;
    const int m = x_row_of(a.cu_q, a.Mq, a.max_q, slot), c = (int)(idx - slot * (unsigned)dv) * 4, h = c / dk;
    if (m < 0) return;
    const float* ml = a.part + (size_t)a.nsplit * a.slots * d + ((size_t)h * a.slots + slot) * 2;
    const size_t step = (size_t)a.H * a.slots * 2;
    float mx = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < a.nsplit; ++s) mx = fmaxf(mx, ml[s * step]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float L = 0.f;
    bool any = false;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < a.nsplit; ++s) {
        const float l = ml[s * step + 1], f = __builtin_amdgcn_exp2f(ml[s * step] - mu);
        const f32x4 o = *(const f32x4*)(a.part + ((size_t)s * a.slots + slot) * d + c);
        if (l != 0.f) {
            any = true;
            L = fmaf(l, f, L);
            acc += o * f;
        }
    }
    store4<T>((T*)a.ctx + (size_t)m * a.ldo + c, any ? acc * (1.0f / L) : acc);
    if (a.lse && c % dk == 0) a.lse[(size_t)h * a.Mq + m] = any ? mx + __log2f(L) : -INFINITY;
}

// Few rows, up to X_MAX_SPLIT ranges: one workgroup per (row, head), 1024 / dk lanes to every four channels, each takes every
// (1024 / dk)th range.  One lane for all ranges waited for 32 loads in a row (15 us of the 21 us of one frame over 65000 keys).
constexpr int X_MAX_SPLIT = 256;
template <typename T, int DK>
__global__ __launch_bounds__(256) void xattn_combine_few_kernel(XArgs a) {
    constexpr int SL = DK / 4, NL = 256 / SL;
    __shared__ float ms[X_MAX_SPLIT], ls[X_MAX_SPLIT];
    __shared__ __attribute__((aligned(16))) float red[NL][DK];
    const int h = blockIdx.x, m = x_row_of(a.cu_q, a.Mq, a.max_q, blockIdx.y), tid = threadIdx.x;
    if (m < 0) return;
    const size_t d = (size_t)a.H * DK;
    if (tid < a.nsplit) {
        const float2 t = *(const float2*)(a.part + (size_t)a.nsplit * a.slots * d + (((size_t)tid * a.H + h) * a.slots + blockIdx.y) * 2);
        ms[tid] = t.x;
        ls[tid] = t.y;
    }
    __syncthreads();
    float mx = -INFINITY;
    for (int s = tid & 63; s < a.nsplit; s += 64) mx = fmaxf(mx, ms[s]);
    mx = wave_max(mx);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float L = 0.f;
    for (int s = tid & 63; s < a.nsplit; s += 64) L += ls[s] == 0.f ? 0.f : ls[s] * __builtin_amdgcn_exp2f(ms[s] - mu);
    L = wave_sum(L);
    const int c = tid % SL * 4, lane_s = tid / SL;            // (dk = 96: 16 lanes are left over)
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = lane_s; s < a.nsplit; s += NL) {
        const f32x4 o = *(const f32x4*)(a.part + ((size_t)s * a.slots + blockIdx.y) * d + h * DK + c);
        if (ls[s] != 0.f) acc += o * __builtin_amdgcn_exp2f(ms[s] - mu);
    }
    if (lane_s < NL) *(f32x4*)(red[lane_s] + c) = acc;
    __syncthreads();
    if (tid >= SL) return;
#pragma unroll
    for (int k = 1; k < NL; ++k) acc += *(const f32x4*)(red[k] + c);
    store4<T>((T*)a.ctx + (size_t)m * a.ldo + h * DK + c, acc * (L == 0.f ? 0.f : 1.0f / L));
    if (a.lse && c == 0) a.lse[(size_t)h * a.Mq + m] = L == 0.f ? -INFINITY : mx + __log2f(L);
}

struct XPlan { bool few; int qt, nsplit; };

static XPlan x_plan(int B, int max_q, int max_k, int H, int KV, int dtype) {
    XPlan p = {};
    const int g = H / KV;
    const long rows = (long)max_q * g, pairs = (long)B * KV;
    p.few = rows <= 16;
    p.nsplit = 1;
    if (p.few) {
        const long tiles = ((long)max_k + 31) / 32;
        // the second launch costs 3 to 4 us, which a wave's fifth tile of a row pays (2 heads of 128, bf16, one sentence: 300 keys 7.7 us whole
        // and 9.4 split, 600 10.5 and 9.6, 1200 17.5 and 9.8; 32 sentences: 8.8 and 9.4, 14.4 and 12.1, 25.3 and 15.9)
        if (tiles > 16 && pairs < 256) {
            // a tile to every wave up to 32 ranges, four tiles to a wave beyond (one frame over 65000 keys, dk = 128: 24 us with 127
            // ranges, 740 without; when P was one number 127 ranges took 14.5 + 7.4 us, 253 ranges 14.4 + 13.0, 32 ranges 26.6 + 4.5)
            const long want = 512 / pairs, some = tiles / 4 < 32 ? tiles / 4 : 32, most = tiles / 16 > some ? tiles / 16 : some;
            p.nsplit = (int)(want < most ? want : most);
        }
    } else {
        // two row tiles to a wave: bf16, whose tiles cost nothing but their reads (32 x 800 rows over 120 keys: 15.9 us, one: 17.9).
        // fp32: with one, three workgroups share a CU and hide each other's LDS reads and splits, though each splits its keys for half the
        // rows (32 x 240 rows x 810 keys, dk = 96, planes still cut off: 59 us against 62 with two tiles and two workgroups)
        p.qt = rows > 64 && dtype == 1 ? 2 : 1;
        // as many workgroups as the chip holds at dk = 128 in bf16, at dk = 96 in fp32, and for every head dim: fp32 of 128 has two to a CU but takes
        // 52 us with 768 and 58 with 512 (32 x 120 rows x 810 keys, 2 heads; dk = 96 38 and 48), small bf16 heads fit more but gain nothing
        // (1024 against 512: dk = 32 18.5 and 17.5, dk = 64 22.6 and 20.4)
        const int kb = dtype == 1 ? 64 : 32, full = dtype == 1 ? 512 : 768;
        const long items = pairs * ((rows + 64 * p.qt - 1) / (64 * p.qt)), tiles = ((long)max_k + kb - 1) / kb;
        // the second launch pays from 400 keys on in bf16, 250 in fp32 (2 heads, 120 rows of one sentence: bf16 of 128 250 keys 11.6 us whole
        // and 12.5 split, 400 17.2 and 14.7, 810 32 and 16.5; fp32 of 64 250 13.4 and 12.4, 810 40 and 16)
        if (items < (dtype == 1 ? full / 2 : full) && tiles >= (dtype == 1 ? 7 : 8)) {
            const long want = full / items, most = tiles / (128 / kb);
            p.nsplit = (int)(want < most ? want : most);
        }
    }
    const int cap = p.few ? X_MAX_SPLIT : 32;
    if (p.nsplit > cap) p.nsplit = cap;
    if (p.nsplit < 1) p.nsplit = 1;
    return p;
}

template <typename E, int DK, int QT, bool DROP> static void launch_xattn_rows(const XArgs& a, dim3 grid, hipStream_t stream) {
    constexpr int KB = x_kb<E>(), stage = XTile<E, DK, KB, 1>::BYTES + XTile<E, DK, KB, 2>::BYTES;
    constexpr int rows = 4 * XTile<E, DK, 16 * QT, 1>::BYTES, out = 4 * x_out_bytes<float, DK>();
    constexpr int tiles = E::PL == 1 ? stage + (stage > rows ? stage : rows) : (stage > rows ? stage : rows), lds = tiles > out ? tiles : out;
    static unsigned long long ok = 0;
    fs2_allow_lds((const void*)xattn_rows_kernel<E, DK, QT, DROP>, lds, &ok);
    hipLaunchKernelGGL((xattn_rows_kernel<E, DK, QT, DROP>), grid, dim3(256), lds, stream, a);
}

template <typename E, int DK>
static int launch_xattn(XArgs& a, const XPlan& p, int B, int max_q, int dk, hipStream_t stream) {
    typedef typename E::mem T;
    if (p.few) {
        constexpr int merge = 4 * 16 * DK * 4 + 512, tiles = 4 * (XTile<E, DK, 32, 2>::BYTES + (E::PL == 1 ? XTile<E, DK, 32, 1>::BYTES : 0));
        constexpr int lds = merge > tiles ? merge : tiles;
        static unsigned long long ok = 0;
        fs2_allow_lds((const void*)xattn_few_kernel<E, DK>, lds, &ok);
        hipLaunchKernelGGL((xattn_few_kernel<E, DK>), dim3(a.nsplit, a.KV, B), dim3(256), lds, stream, a);
    } else {
        const int rows = max_q * a.g, nblk = (rows + 64 * p.qt - 1) / (64 * p.qt);
        const dim3 grid = fs2_x_grid(a, nblk, a.KV, B);
        if (p.qt == 2) {
            if constexpr (E::PL == 1) {
                if (a.drop.thresh) launch_xattn_rows<E, DK, 2, true>(a, grid, stream);
                else launch_xattn_rows<E, DK, 2, false>(a, grid, stream);
            }
        } else {
            if (a.drop.thresh) launch_xattn_rows<E, DK, 1, true>(a, grid, stream);
            else launch_xattn_rows<E, DK, 1, false>(a, grid, stream);
        }
    }
    FS2_CHECK_LAUNCH("fs2_cross_attention");
    if (a.nsplit > 1) {
        const long long rows = (long long)B * max_q, n = rows * (a.H * dk / 4);         // (both small where keys are split)
        if (p.few)
            hipLaunchKernelGGL((xattn_combine_few_kernel<T, DK>), dim3(a.H, (unsigned)rows), dim3(256), 0, stream, a);
        else
            hipLaunchKernelGGL(xattn_combine_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a, B, dk);
        FS2_CHECK_LAUNCH("fs2_cross_attention(merge)");
    }
    return FS2_OK;
}

}  // namespace fs2

using namespace fs2;

extern "C" long long fs2_cross_attention_workspace(int B, int max_q, int max_k, int Mq, int n_heads, int n_kv_heads, int dk,
                                                   int dtype) {
    if (B <= 0 || max_q <= 0 || max_k <= 0 || Mq <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads) return 0;
    const XPlan p = x_plan(B, max_q, max_k, n_heads, n_kv_heads, dtype);
    return p.nsplit == 1 ? 0 : (long long)p.nsplit * B * max_q * n_heads * (dk + 2) * (long long)sizeof(float);
}

extern "C" int fs2_cross_attention(const void* q, const void* k, const void* v, void* ctx, float* lse, const int* cu_q,
                                   const int* cu_k, void* workspace, int B, int max_q, int max_k, int Mq, int Mk, int n_heads,
                                   int n_kv_heads, int dk, int ldq, int ldk, int ldv, int ldo, int dtype, unsigned seed,
                                   unsigned stream_id, float rate, hipStream_t stream) {
    const int rc = fs2_x_check("fs2_cross_attention", q, k, cu_q, cu_k, B, max_q, max_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq, ldk,
                               dtype);
    if (rc != FS2_OK) return rc;
    const int epv = dtype == 0 ? 4 : 8;
    FS2_CHECK_ARG(rate >= 0.f && rate < 1.f, "fs2_cross_attention: dropout rate must be in [0, 1)");
    FS2_CHECK_ARG((v || Mk == 0) && (ctx || Mq == 0) && ((uintptr_t)v & 15) == 0 && ((uintptr_t)ctx & 15) == 0,
                  "fs2_cross_attention: null or unaligned v or ctx");
    FS2_CHECK_ARG(ldv >= n_kv_heads * dk && ldv <= (1 << 20) && ldo >= n_heads * dk && ldo <= (1 << 20) && ldv % epv == 0 && ldo % epv == 0,
                  "fs2_cross_attention: bad leading dims ldv=%d ldo=%d", ldv, ldo);
    if (max_q == 0) return FS2_OK;
    XArgs a = fs2_x_args(q, k, v, cu_q, cu_k, max_q, max_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq, ldk, ldv, ldo);
    a.ctx = ctx;
    a.lse = lse;
    a.drop = fs2_make_dropout(seed, stream_id, rate);
    const XPlan p = x_plan(B, max_q, max_k, n_heads, n_kv_heads, dtype);
    a.nsplit = p.nsplit;
    a.part = (float*)workspace;
    a.slots = p.nsplit > 1 ? B * max_q : 0;                 // (few rows where keys are split)
    FS2_CHECK_ARG(p.nsplit == 1 || (workspace && ((uintptr_t)workspace & 15) == 0),
                  "fs2_cross_attention: this shape needs fs2_cross_attention_workspace bytes, 16-byte aligned");
#define FS2_X(TT, DKK) return launch_xattn<TT, DKK>(a, p, B, max_q, dk, stream)
    if (dtype == 0) {
        if (dk == 32) FS2_X(XF32, 32);
        if (dk == 64) FS2_X(XF32, 64);
        if (dk == 96) FS2_X(XF32, 96);
        FS2_X(XF32, 128);
    }
    if (dk == 32) FS2_X(XB16, 32);
    if (dk == 64) FS2_X(XB16, 64);
    if (dk == 96) FS2_X(XB16, 96);
    FS2_X(XB16, 128);
#undef FS2_X
}
