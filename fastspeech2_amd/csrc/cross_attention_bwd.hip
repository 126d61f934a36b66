// Backward of cross attention (cross_attention.hip) and the attention mass of every key; the probabilities are recomputed tile
// by tile from q, k and the saved log-sum-exp, never stored.  With S = q k^T / sqrt(dk), P = exp2(S log2 e - lse), D the
// dropout multiplier, O = (P o D) v and upstream dO:
//   delta = sum_dv dO o O                                         xattn_delta_kernel
//         = sum_keys P o dP, which knows nothing of ctx's rounding: taken instead where a bf16 workgroup has all keys of the utterance
//           (dq up to 64, dk up to 32 of them; the fewer keys, the more that rounding weighs: 1.4 times the result's own at two)
//   dP = dO v^T o D,  dS = P o (dP - delta)                       xattn_bwd_kernel, two kinds of workgroups:
//   dq = dS k / sqrt(dk)                                            x_dq_block: one wave per 16 packed rows
//   dk = dS^T q / sqrt(dk),  dv = (P o D)^T dO                      x_dkv32_block (bf16), x_dkv_block (fp32)
//   mass[h][key] = sum_q P                                        xattn_mass_kernel
// The packed rows of a shared head are its g query heads, so the sum over the group that dk and dv need is part of the loop.
// Every output element has one writer and every sum a fixed order: no atomics, the same bits every time.
#include "cross_attention.h"

namespace fs2 {

// Measured on a training step of 32 x 800 frames over 120 phones, 2 heads of 128, bf16: delta 6.4 us for 27 MB (4.2 TB/s), the rest 39 us
// (whole step, forward included, 57 us, 70 with dropout, where the last spills 8 registers; floor 11.8); 3 x 1601 frames over 301 phones,
// 4 heads on 2 of 96, fp32: 5 + 79 + 5.5 us for 4.9 GFLOP (whole step 114 to 117, 128 with dropout, 12 registers spilled; floor 37).

template <typename T> __device__ __forceinline__ f32x4 x_load4(const T* p) {
    if constexpr (sizeof(T) == 4) return *(const f32x4*)p;
    const bf16x4 v = *(const bf16x4*)p;
    return (f32x4){(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}

// ---- dq: one workgroup per (utterance, shared head, 64 packed rows) -------------------------------------
// Two key tiles behind a wait for the rows, in each of 832 workgroups (32 x 800 rows, 2 heads): latency.  dS as two numbers is 2 of the 22
// us that these took in a launch of their own.
template <typename E, int DK, bool DROP> __device__ __forceinline__ void x_dq_block(const XArgs& a, unsigned id, unsigned char* smem) {
    typedef typename E::mem T;
    constexpr int KB = x_kb<E>(), NT = KB / 16, NC = KB / 32, NST = E::PL == 1 ? 2 : 1;
    typedef XTile<E, DK, KB, 2> TK;
    typedef XTile<E, DK, KB, 1> TV;
    typedef typename TK::frag_t frag_t;
    constexpr int KS = TK::KS, DT = TK::DT, STAGE = TK::BYTES + TV::BYTES;
    // smem: stage s: K tile (read both ways), V tile
    int b, kvh, blk, split;
    if (!x_decode_line(a, id, a.nblk_q, b, kvh, blk, split)) return;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, a.max_q, q0, lenq);
    x_range(a.cu_k, b, a.Mk, a.max_k, k0, lenk);
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
    XFetch<E, DK, KB, 2, 4> fk(a.ldk, wave, lane);
    XFetch<E, DK, KB, 1, 4> fv(a.ldv, wave, lane);
    auto fetch = [&](int kt, int st) __attribute__((always_inline)) {
        unsigned char* d = smem + st * STAGE;
        fk.fetch(kb + (size_t)kt * KB * a.ldk, a.ldk, lenk - kt * KB, d, wave, lane);
        fv.fetch(vb + (size_t)kt * KB * a.ldv, a.ldv, lenk - kt * KB, d + TK::BYTES, wave, lane);
    };
    if (lenk > 0) fetch(0, 0);

    // q and dO rows of the wave: bf16 in the other stage, both under way together; fp32 one after the other
    frag_t qf[KS], dof[KS];
    {
        typedef XTile<E, DK, 16, 1> TQ;
        unsigned char* own = smem + (NST == 2 ? STAGE : 0) + wave * TQ::BYTES;
        constexpr int NEXT = E::PL == 1 ? 4 * TQ::BYTES : 0;
        const int first = min(blk * 64 + wave * 16, nrow - 1);
        XRows<E, DK, 16> rq(a.ldq, lane), rd(a.ldo, lane);
        rq.start(a, (const T*)a.q + (size_t)q0 * a.ldq + kvh * a.g * DK, a.ldq, first, nrow, own, lane);
        rd.start(a, (const T*)a.dctx + (size_t)q0 * a.ldo + kvh * a.g * DK, a.ldo, first, nrow, own + NEXT, lane);
        rq.finish(own, lane);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = TQ::row_frag(own, i, ks, g);
        if constexpr (E::PL == 3) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            rd.finish(own, lane);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) dof[ks] = TQ::row_frag(own + NEXT, i, ks, g);
    }
    float del = 0.f, lse_q = 0.f;
    if (lenk > 0) {                    // (a batch without keys has no delta: nobody wrote it and its workspace has no room for it)
        del = a.delta[(size_t)head * a.Mq + qrow];
        lse_q = a.lse[(size_t)head * a.Mq + qrow];
    }

    f32x4 dq[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dq[dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    Dropout dh = a.drop;
    dh.stream += (uint32_t)head;
    const int ntiles = (lenk + KB - 1) / KB;
    for (int kt = 0; kt < ntiles; ++kt) {
        const int st = NST == 2 ? kt & 1 : 0;
        unsigned char* Ks = smem + st * STAGE;
        unsigned char* Vs = Ks + TK::BYTES;
        if constexpr (E::PL == 1) {
            vm_wait_barrier<0>();      // tile kt has landed; every wave is done with the other stage
        } else {
            __syncthreads();           // every wave is done with the tile (or its rows) before
            fk.put(Ks, wave, lane);
            fv.put(Vs, wave, lane);
            __syncthreads();
            if (kt + 1 < ntiles) fetch(kt + 1, 0);
        }
        f32x4 s[NT], dp[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt] = dp[nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            frag_t kf[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) kf[nt] = TK::row_frag(Ks, nt * 16 + i, ks, g);
            x_mma<E, NT>(kf, qf[ks], s);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) kf[nt] = TV::row_frag(Vs, nt * 16 + i, ks, g);
            x_mma<E, NT>(kf, dof[ks], dp);
        }
        // bf16: K^T fragments before the next tile's DMA (no transposed LDS read passes one), under the arithmetic
        frag_t kc[E::PL == 1 ? NC : 1][DT];
        if constexpr (E::PL == 1) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) kc[c][dt] = TK::col_frag(Ks, c, dt, g, i);
            __builtin_amdgcn_sched_barrier(0);
            if (kt + 1 < ntiles) fetch(kt + 1, st ^ 1);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = kt * KB + nt * 16 + 4 * g + e;
                s[nt][e] = __builtin_amdgcn_exp2f(fmaf(s[nt][e], a.scale_log2e, -lse_q));
                if constexpr (DROP) dp[nt][e] = drop_keep(dh, (uint32_t)qrow, (uint32_t)key) ? dp[nt][e] * dh.inv_keep : 0.f;
            }
        if (kt * KB + KB > lenk) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (kt * KB + nt * 16 + 4 * g + e >= lenk) s[nt][e] = dp[nt][e] = 0.f;
        }
        if constexpr (E::PL == 1)
            if (lenk <= KB) {            // all keys at hand: delta without ctx's rounding
                del = 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) del = fmaf(s[nt][e], dp[nt][e], del);
                del = rows_sum(del);
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] *= dp[nt][e] - del;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const frag_t dsf = x_pack<E>(s[2 * c], s[2 * c + 1]);
            if constexpr (E::PL == 1) {
                x_mma<E, DT>(kc[c], dsf, dq);
                x_mma<E, DT>(kc[c], x_pack_rest(s[2 * c], s[2 * c + 1], dsf), dq);
            } else {
#pragma unroll
                for (int dt0 = 0; dt0 < DT; dt0 += 2) {
                    frag_t k2[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) k2[u] = TK::col_frag(Ks, c, dt0 + u, g, i);
                    x_mma<E, 2>(k2, dsf, &dq[dt0]);
                }
            }
        }
    }
    __syncthreads();                   // the tiles' memory serves the waves' results now
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dq[dt] *= a.scale;
    x_store_rows<T, DK>(a, (T*)a.dq, a.ldq, q0, kvh, blk * 64 + wave * 16, nrow, dq, smem + wave * x_out_bytes<T, DK>(), lane);
}

// ---- dk, dv -----------------------------------------------------------------------------------------------------------
// fp32: one workgroup per (utterance, shared head, 64 keys, range of packed rows), a wave to 16 keys, its K and V operands in
// registers; row tiles of 32 in LDS for all four, split into planes once for all (a wave with a tile of its own, as in bf16, would
// split each for itself).  Bound by what a tile costs a SIMD in turn: MFMA, splits, LDS.
template <int DK, bool DROP> __device__ __forceinline__ void x_dkv_block(const XArgs& a, unsigned id, unsigned char* smem) {
    typedef XF32 E;
    typedef float T;
    typedef XTile<E, DK, 32, 2> TL;
    typedef typename TL::frag_t frag_t;
    constexpr int KS = TL::KS, DT = TL::DT;
    // smem: Q tile, dO tile (read both ways), 32 lse, 32 delta
    int b, kvh, blk, split;
    if (!x_decode_line(a, id, a.nblk, b, kvh, blk, split)) return;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, a.max_q, q0, lenq);
    x_range(a.cu_k, b, a.Mk, a.max_k, k0, lenk);
    if (blk * 64 >= lenk) return;
    const int nrow = lenq * a.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int key = blk * 64 + wave * 16 + i, kc = min(key, lenk - 1);
    const int ntiles = (nrow + 31) / 32, per = a.nsplit == 1 ? ntiles : (ntiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(t0 + per, ntiles);
    unsigned char *Qs = smem, *Ds = smem + TL::BYTES;
    float* rows_s = (float*)(smem + 2 * TL::BYTES);

    const T* __restrict__ qb = (const T*)a.q + (size_t)q0 * a.ldq + kvh * a.g * DK;
    const T* __restrict__ db = (const T*)a.dctx + (size_t)q0 * a.ldo + kvh * a.g * DK;
    XFetch<E, DK, 32, 2, 4> fq(a.ldq, wave, lane), fd(a.ldo, wave, lane);
    float stat = 0.f;
    auto fetch = [&](int qt) __attribute__((always_inline)) {
        fq.fetch_rows(a, qb, a.ldq, qt * 32, nrow, Qs, wave, lane);
        fd.fetch_rows(a, db, a.ldo, qt * 32, nrow, Ds, wave, lane);
        if (tid < 64) {
            const int r = min(qt * 32 + (tid & 31), nrow - 1), q = x_query(a, r);
            stat = (tid < 32 ? a.lse : a.delta)[(size_t)(kvh * a.g + r - q * a.g) * a.Mq + q0 + q];
        }
    };
    if (t0 < t1) fetch(t0);
    frag_t kf[KS], vf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        kf[ks] = x_load<E>((const T*)a.k + (size_t)(k0 + kc) * a.ldk + kvh * DK + ks * 32 + g * 8);
        vf[ks] = x_load<E>((const T*)a.v + (size_t)(k0 + kc) * a.ldv + kvh * DK + ks * 32 + g * 8);
    }
    f32x4 dk_[DT], dv_[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dk_[dt] = dv_[dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    for (int qt = t0; qt < t1; ++qt) {
        if (qt > t0) __syncthreads();
        fq.put(Qs, wave, lane);
        fd.put(Ds, wave, lane);
        if (tid < 64) rows_s[tid] = stat;
        __syncthreads();
        if (qt + 1 < t1) fetch(qt + 1);
        f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, dp[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            frag_t f[2];
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) f[rt] = TL::row_frag(Qs, rt * 16 + i, ks, g);
            x_mma<E, 2>(f, kf[ks], s);               // rows: packed rows qt 32 + 16 rt + 4 g + e, column: key i
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) f[rt] = TL::row_frag(Ds, rt * 16 + i, ks, g);
            x_mma<E, 2>(f, vf[ks], dp);
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const f32x4 lse4 = *(const f32x4*)(rows_s + rt * 16 + 4 * g), del4 = *(const f32x4*)(rows_s + 32 + rt * 16 + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = qt * 32 + rt * 16 + 4 * g + e;
                const bool ok = r < nrow;
                const float p = ok ? __builtin_amdgcn_exp2f(fmaf(s[rt][e], a.scale_log2e, -lse4[e])) : 0.f;
                float mul = 1.0f;
                if constexpr (DROP) {
                    const int rr = min(r, nrow - 1), q = x_query(a, rr);
                    Dropout dh = a.drop;
                    dh.stream += (uint32_t)(kvh * a.g + rr - q * a.g);
                    mul = drop_mul(dh, (uint32_t)(q0 + q), (uint32_t)kc);
                }
                dp[rt][e] = ok ? p * (dp[rt][e] * mul - del4[e]) : 0.f;
                s[rt][e] = p * mul;
            }
        }
        const frag_t pf = x_pack<E>(s[0], s[1]), dsf = x_pack<E>(dp[0], dp[1]);
#pragma unroll
        for (int dt0 = 0; dt0 < DT; dt0 += 2) {
            frag_t f[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) f[u] = TL::col_frag(Ds, 0, dt0 + u, g, i);
            x_mma<E, 2>(f, pf, &dv_[dt0]);
#pragma unroll
            for (int u = 0; u < 2; ++u) f[u] = TL::col_frag(Qs, 0, dt0 + u, g, i);
            x_mma<E, 2>(f, dsf, &dk_[dt0]);
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
    } else {                          // part[split][dk, dv][slots][KV * DK]
        const size_t w = (size_t)a.KV * DK, half = (size_t)a.slots * w;
        float* dst = a.part + (size_t)split * 2 * half + (size_t)(b * a.max_k + key) * w + kvh * DK + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            *(f32x4*)(dst + dt * 16) = dk_[dt] * a.scale;
            *(f32x4*)(dst + half + dt * 16) = dv_[dt];
        }
    }
}

// bf16: one workgroup of four waves per (utterance, shared head, 32 keys, range of packed rows).  The 32 keys stay in LDS; each wave
// streams its OWN tiles of 32 rows through a private LDS buffer (read row-wise for S and dP, transposed for dV and dK) and keeps a
// dK, dV of its own, so the loop has no barrier; the four are added through LDS at the end.  64 keys to a workgroup and one row tile
// for all four waves (the fp32 form above) leave half the chip without a workgroup at 32 x 120 phones unless the rows are split, which
// writes the gradients several times over as partial sums (27 + 5 us, before dS became two numbers; this form then 25.6).  A second
// buffer for each wave would overlap its tiles' DMA and products, but leaves one workgroup to a CU where there are slightly more
// workgroups than CUs: 41 us against 28.
template <int DK, bool DROP> __device__ __forceinline__ void x_dkv32_block(const XArgs& a, unsigned id, unsigned char* smem) {
    typedef XB16 E;
    typedef bf16_t T;
    typedef XTile<E, DK, 32, 2> TL;
    constexpr int KT = 2, KB = 16 * KT;
    typedef XTile<E, DK, KB, 1> TK;
    typedef typename TL::frag_t frag_t;
    constexpr int KS = TL::KS, DT = TL::DT, NP = TK::BYTES / 1024, NWK = NP % 4 == 0 ? 4 : (NP % 2 == 0 ? 2 : 1);
    constexpr int WAVE = 2 * TL::BYTES;                  // a wave's Q tile, dO tile: 80 KB in all at dk = 128, two workgroups per CU
    // smem: K tile, V tile, then the waves'
    int b, kvh, blk, split;
    if (!x_decode_line(a, id, a.nblk, b, kvh, blk, split)) return;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, a.max_q, q0, lenq);
    x_range(a.cu_k, b, a.Mk, a.max_k, k0, lenk);
    if (blk * KB >= lenk) return;
    const int nrow = lenq * a.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int ntiles = (nrow + 31) / 32, per = a.nsplit == 1 ? ntiles : (ntiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(t0 + per, ntiles);
    unsigned char *Ks = smem, *Vs = smem + TK::BYTES;
    unsigned char* Qs = smem + 2 * TK::BYTES + wave * WAVE;
    unsigned char* Ds = Qs + TL::BYTES;
    float stat = 0.f;                                    // lane l: lse of row l of the tile, from lane 32 on delta of row l - 32

    if (wave < NWK) {
        XFetch<E, DK, KB, 1, NWK> fk(a.ldk, wave, lane), fv(a.ldv, wave, lane);
        const size_t first = (size_t)(k0 + blk * KB);
        fk.fetch((const T*)a.k + first * a.ldk + kvh * DK, a.ldk, lenk - blk * KB, Ks, wave, lane);
        fv.fetch((const T*)a.v + first * a.ldv + kvh * DK, a.ldv, lenk - blk * KB, Vs, wave, lane);
    }
    const T* __restrict__ qb = (const T*)a.q + (size_t)q0 * a.ldq + kvh * a.g * DK;
    const T* __restrict__ db = (const T*)a.dctx + (size_t)q0 * a.ldo + kvh * a.g * DK;
    XFetch<E, DK, 32, 2, 1> fq(a.ldq, 0, lane), fd(a.ldo, 0, lane);
    auto stage = [&](int qt) __attribute__((always_inline)) {
        if (a.g == 1) {
            fq.fetch(qb + (size_t)qt * 32 * a.ldq, a.ldq, nrow - qt * 32, Qs, 0, lane);
            fd.fetch(db + (size_t)qt * 32 * a.ldo, a.ldo, nrow - qt * 32, Ds, 0, lane);
        } else {
            fq.fetch_rows(a, qb, a.ldq, qt * 32, nrow, Qs, 0, lane);
            fd.fetch_rows(a, db, a.ldo, qt * 32, nrow, Ds, 0, lane);
        }
        const int r = min(qt * 32 + (lane & 31), nrow - 1), q = x_query(a, r);
        const size_t at = (size_t)(kvh * a.g + r - q * a.g) * a.Mq + q0 + q;
        stat = (lane < 32 ? a.lse : a.delta)[at];
    };
    if (t0 + wave < t1) stage(t0 + wave);

    f32x4 dk_[DT][KT], dv_[DT][KT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) dk_[dt][kt] = dv_[dt][kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    vm_wait_barrier<0>();                    // the keys have landed, for every wave
    for (int qt = t0 + wave; qt < t1; qt += 4) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // this wave's rows have landed (no other wave reads them)
        f32x4 s[2][KT], dp[2][KT];             // [16 rows][16 keys]: lane (g, i) has rows 4 g + e, key i
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) s[rt][kt] = dp[rt][kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            frag_t rf[2], kf[KT];
#pragma unroll
            for (int u = 0; u < 2; ++u) rf[u] = TL::row_frag(Qs, u * 16 + i, ks, g);
#pragma unroll
            for (int u = 0; u < KT; ++u) kf[u] = TK::row_frag(Ks, u * 16 + i, ks, g);
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) s[rt][kt] = mma16(rf[rt].p[0], kf[kt].p[0], s[rt][kt]);
#pragma unroll
            for (int u = 0; u < 2; ++u) rf[u] = TL::row_frag(Ds, u * 16 + i, ks, g);
#pragma unroll
            for (int u = 0; u < KT; ++u) kf[u] = TK::row_frag(Vs, u * 16 + i, ks, g);
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) dp[rt][kt] = mma16(rf[rt].p[0], kf[kt].p[0], dp[rt][kt]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float lse_r = __shfl(stat, rt * 16 + 4 * g + e, 64);
                float del_r = __shfl(stat, 32 + rt * 16 + 4 * g + e, 64);
                const int r = qt * 32 + rt * 16 + 4 * g + e;
                const bool ok = r < nrow;
                Dropout dh = a.drop;
                int q = 0;
                if constexpr (DROP) {
                    const int rr = min(r, nrow - 1);
                    q = x_query(a, rr);
                    dh.stream += (uint32_t)(kvh * a.g + rr - q * a.g);
                }
                float p[KT];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    p[kt] = ok ? __builtin_amdgcn_exp2f(fmaf(s[rt][kt][e], a.scale_log2e, -lse_r)) : 0.f;
                    s[rt][kt][e] = p[kt];
                    if constexpr (DROP) {
                        const bool keep = drop_keep(dh, (uint32_t)(q0 + q), (uint32_t)min(blk * KB + kt * 16 + i, lenk - 1));
                        s[rt][kt][e] = keep ? p[kt] * dh.inv_keep : 0.f;
                        dp[rt][kt][e] = keep ? dp[rt][kt][e] * dh.inv_keep : 0.f;
                    }
                }
                if (lenk <= KB) {            // all keys at hand: delta without ctx's rounding
                    del_r = 0.f;
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) del_r = kt * 16 + i < lenk ? fmaf(p[kt], dp[rt][kt][e], del_r) : del_r;
                    del_r = row16_sum(del_r);
                }
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) dp[rt][kt][e] = ok ? p[kt] * (dp[rt][kt][e] - del_r) : 0.f;
            }
        }
        frag_t pf[KT], pr[KT], dsf[KT], dsr[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            x_pack_weights(s[0][kt], s[1][kt], pf[kt], pr[kt]);
            dsf[kt] = x_pack<E>(dp[0][kt], dp[1][kt]);
            dsr[kt] = x_pack_rest(dp[0][kt], dp[1][kt], dsf[kt]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            frag_t dot = TL::col_frag(Ds, 0, dt, g, i);
            if (qt * 32 + 32 > nrow) x_keep_rows(dot, nrow - qt * 32, g);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                dv_[dt][kt] = mma16(dot.p[0], pr[kt].p[0], dv_[dt][kt]);
                dv_[dt][kt] = mma16(dot.p[0], pf[kt].p[0], dv_[dt][kt]);
            }
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const frag_t qtr = TL::col_frag(Qs, 0, dt, g, i);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                dk_[dt][kt] = mma16(qtr.p[0], dsf[kt].p[0], dk_[dt][kt]);
                dk_[dt][kt] = mma16(qtr.p[0], dsr[kt].p[0], dk_[dt][kt]);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // read before the next tile's DMA overwrites it
        if (qt + 4 < t1) stage(qt + 4);
    }
    // add the four waves' gradients: [wave][32 keys][DK + 4] floats, dv then dk
    constexpr int LDR = DK + 4, SL = DK / 4;
    float* red = (float*)smem;
    const size_t w = (size_t)a.KV * DK, half = (size_t)a.slots * w;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
                *(f32x4*)(red + (wave * KB + kt * 16 + i) * LDR + dt * 16 + 4 * g) = which == 0 ? dv_[dt][kt] : dk_[dt][kt] * a.scale;
        __syncthreads();
        for (int e = tid; e < KB * SL; e += 256) {
            const int key = e / SL, c = (e % SL) * 4;
            if (blk * KB + key >= lenk) continue;
            f32x4 sum = *(const f32x4*)(red + key * LDR + c);
#pragma unroll
            for (int u = 1; u < 4; ++u) sum += *(const f32x4*)(red + (u * KB + key) * LDR + c);
            const size_t m = (size_t)(k0 + blk * KB + key);
            if (a.nsplit > 1)                          // part[split][dk, dv][slots][KV * DK]
                *(f32x4*)(a.part + (size_t)split * 2 * half + (which == 0 ? half : 0) + (size_t)(b * a.max_k + blk * KB + key) * w + kvh * DK +
                          c) = sum;
            else if (which == 0)
                store4<T>((T*)a.dv + m * a.ldv + kvh * DK + c, sum);
            else
                store4<T>((T*)a.dk + m * a.ldk + kvh * DK + c, sum);
        }
    }
}

// Both in one launch, the longer key workgroups first: alone, the row workgroups ended in a half-filled second round and the key
// workgroups, hardly more than CUs, left half of every CU.  32 x 800 over 120, 2 heads of 128, bf16: 37 + 6.4 us (delta, which both
// need, has become a launch) against 22 + 28; 8 x 3100 over 512: 89 + 6 against 45 + 81; 3 x 1601 over 301, fp32, dk = 96: 78 + 5
// against 46 + 47.
template <typename E, int DK, bool DROP>
__global__ __launch_bounds__(256, E::PL == 3 && DK == 128 ? 1 : 2) void xattn_bwd_kernel(XArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    if (blockIdx.x >= a.key_groups) x_dq_block<E, DK, DROP>(a, blockIdx.x - a.key_groups, smem);
    else if constexpr (E::PL == 1) x_dkv32_block<DK, DROP>(a, blockIdx.x, smem);
    else x_dkv_block<DK, DROP>(a, blockIdx.x, smem);
}

// delta: 16 lanes to a row and up to X_DELTA_HEADS of its heads, four elements at a time
constexpr int X_DELTA_HEADS = 2;
template <typename T, int DK> __global__ __launch_bounds__(256) void xattn_delta_kernel(XArgs a, int B) {
    const unsigned per = (unsigned)(a.H + X_DELTA_HEADS - 1) / X_DELTA_HEADS;
    const unsigned id = blockIdx.x * 16 + (threadIdx.x >> 4), slot = id / per;
    if (slot >= (unsigned)B * (unsigned)a.max_q) return;
    const int m = x_row_of(a.cu_q, a.Mq, a.max_q, slot), lane = threadIdx.x & 15, h0 = (int)(id - slot * per) * X_DELTA_HEADS;
    if (m < 0) return;
    float s[X_DELTA_HEADS];
#pragma unroll
    for (int u = 0; u < X_DELTA_HEADS; ++u) {                 // (the last head again where there are fewer: no branch between the loads)
        const size_t at = (size_t)m * a.ldo + min(h0 + u, a.H - 1) * DK;
        s[u] = 0.f;
#pragma unroll
        for (int c = 0; c < DK; c += 64) {
            const int e = c + lane * 4;
            if (DK % 64 == 0 || e < DK) {
                const f32x4 o = x_load4((const T*)a.ctx + at + e), d = x_load4((const T*)a.dctx + at + e);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[u] = fmaf(o[j], d[j], s[u]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < X_DELTA_HEADS; ++u) {
        s[u] = row16_sum(s[u]);
        if (lane == 0 && h0 + u < a.H) a.delta[(size_t)(h0 + u) * a.Mq + m] = s[u];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void xattn_dkv_sum_kernel(XArgs a, int B, int dk) {
    const int w = a.KV * dk;
    const unsigned wv = (unsigned)w >> 2, idx = blockIdx.x * 256 + threadIdx.x, slot = idx / (2 * wv);
    if (slot >= (unsigned)B * (unsigned)a.max_k) return;
    const int m = x_row_of(a.cu_k, a.Mk, a.max_k, slot);
    if (m < 0) return;
    const unsigned e = idx - slot * 2 * wv;
    const bool is_v = e >= wv;
    const int c = (int)(is_v ? e - wv : e) * 4;
    const size_t half = (size_t)a.slots * w;
    const float* src = a.part + (is_v ? half : 0) + (size_t)slot * w + c;
    f32x4 sum = *(const f32x4*)src;
    for (int s = 1; s < a.nsplit; ++s) sum += *(const f32x4*)(src + (size_t)s * 2 * half);
    if (is_v)
        store4<T>((T*)a.dv + (size_t)m * a.ldv + c, sum);
    else
        store4<T>((T*)a.dk + (size_t)m * a.ldk + c, sum);
}

// ---- mass: one workgroup per (utterance, head, 16 KT keys, range of queries) --------------------------------------------
// The keys are operands in the registers of every wave; the waves stream the queries, 16 at a time, through a private LDS ring of two
// tiles.  S^T = K Q^T: a lane owns one query and 4 keys of every 16, adds up its own queries' weights over the whole loop, and the 16
// queries of a row of lanes meet only at the end.  32 x 800 queries, 120 keys, 2 heads of 128, bf16: 9.4 us for 16 MB (1.7 TB/s; floor
// 3.0; 11.6 with four waves): the keys' wait and the first queries' behind it, then seven tiles to a wave, in workgroups fewer than CUs.
// 3100 queries, 512 keys, 4 heads of 64, fp32: 13.5 us with the sum over nine query ranges (floor 3.0).  64 keys to a workgroup in bf16;
// 32 in fp32, whose keys take three times the registers.
constexpr int X_MASS_WAVES = 8;

template <typename E, int DK, int KT>
__global__ __launch_bounds__(64 * X_MASS_WAVES, 2) void xattn_mass_kernel(XArgs a) {
    typedef typename E::mem T;
    constexpr int KS = DK / 32, NW = X_MASS_WAVES, KB = 16 * KT, NST = E::PL == 1 ? 2 : 1;
    typedef XTile<E, DK, 16, 1> TQ;
    typedef XTile<E, DK, KB, 1> TK;
    constexpr int PER_TILE = TQ::BYTES / 1024 + 1;            // bf16: vector-memory instructions of one tile (its DMA, its lse)
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];      // keys, then the waves' rings; at the end the sums
    int b, h, blk, split;
    if (!x_decode(a, a.H, b, h, blk, split)) return;
    int q0, lenq, k0, lenk;
    x_range(a.cu_q, b, a.Mq, a.max_q, q0, lenq);
    x_range(a.cu_k, b, a.Mk, a.max_k, k0, lenk);
    if (blk * KB >= lenk) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int kvh = x_query(a, h);                       // h / g
    const int ntiles = (lenq + 15) / 16, per = a.nsplit == 1 ? ntiles : (ntiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(t0 + per, ntiles);
    const T* __restrict__ qb = (const T*)a.q + (size_t)q0 * a.ldq + h * DK;
    const float* __restrict__ lse = a.lse + (size_t)h * a.Mq + q0;
    unsigned char* ring = smem + TK::BYTES + wave * NST * TQ::BYTES;

    constexpr int NP = TK::BYTES / 1024, NWK = E::PL == 3 || NP % NW == 0 ? NW : 4;          // waves that fetch the keys
    XFetch<E, DK, KB, 1, NWK> fk(a.ldk, wave, lane);
    if (NWK == NW || wave < NWK)
        fk.fetch((const T*)a.k + (size_t)(k0 + blk * KB) * a.ldk + kvh * DK, a.ldk, lenk - blk * KB, smem, wave, lane);
    XFetch<E, DK, 16, 1, 1> fq(a.ldq, 0, lane);
    float l_next = INFINITY;
    auto fetch = [&](int qt, int st) __attribute__((always_inline)) {
        fq.fetch(qb + (size_t)qt * 16 * a.ldq, a.ldq, lenq - qt * 16, ring + st * TQ::BYTES, 0, lane);
        l_next = lse[min(qt * 16 + i, lenq - 1)];
    };
    if (t0 + wave < t1) fetch(t0 + wave, 0);                   // under the keys' wait
    fk.put(smem, wave, lane);
    vm_wait_barrier<0>();
    XFrag<E> kf[KS][KT];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) kf[ks][kt] = TK::row_frag(smem, kt * 16 + i, ks, g);
    f32x4 acc[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) acc[kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    int st = 0;
    for (int qt = t0 + wave; qt < t1; qt += NW) {
        float l = l_next;
        const unsigned char* Qs = ring + st * TQ::BYTES;
        if constexpr (E::PL == 1) {
            if (qt + NW < t1) {
                fetch(qt + NW, st ^ 1);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER_TILE) : "memory");      // this tile has landed, the next is under way
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            st ^= 1;
        } else {
            fq.put(ring, 0, lane);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (qt + NW < t1) fetch(qt + NW, 0);
        }
        if (qt * 16 + i >= lenq || l == -INFINITY) l = INFINITY;      // no such query, or one without keys: no weight
        f32x4 s[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) x_mma<E, KT>(kf[ks], TQ::row_frag(Qs, i, ks, g), s);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[kt][e] += __builtin_amdgcn_exp2f(fmaf(s[kt][e], a.scale_log2e, -l));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // read before the tile after next overwrites it
    }
    __syncthreads();
    float (*red)[KB] = (float (*)[KB])smem;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v = row16_sum(acc[kt][e]);
            if (i == 0) red[wave][kt * 16 + 4 * g + e] = v;
        }
    __syncthreads();
    const int key = blk * KB + tid;
    if (tid < KB && key < lenk) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += red[w][tid];
        if (a.nsplit == 1) a.mass[(size_t)h * a.Mk + k0 + key] = v;
        else a.part[((size_t)split * a.H + h) * a.slots + b * a.max_k + key] = v;
    }
}

__global__ __launch_bounds__(256) void xattn_mass_sum_kernel(XArgs a, int B) {
    const unsigned idx = blockIdx.x * 256 + threadIdx.x, n = (unsigned)B * (unsigned)a.max_k, h = idx / n;
    if (h >= (unsigned)a.H) return;
    const int m = x_row_of(a.cu_k, a.Mk, a.max_k, idx - h * n);
    if (m < 0) return;
    const size_t step = (size_t)a.H * n;
    float sum = a.part[idx];
    for (int s = 1; s < a.nsplit; ++s) sum += a.part[s * step + idx];
    a.mass[(size_t)h * a.Mk + m] = sum;
}

// Row ranges of the key workgroups, chosen from the shape: one workgroup for every CU where the keys alone do not give one (the row
// workgroups fill the rest: 8 x 800 over 120, fp32, dk = 128: 47 us against 54 with two to a CU), and at least four row tiles to a
// workgroup.  The join pays from 256 rows on (one sentence of 400 frames over 120 phones, whole step without any split and with:
// bf16 27.4 and 25.1 us, of 1600 52.6 and 27.3; fp32, dk = 64: 39.6 and 28.2, 110 and 29.9).
static int x_dkv_split(int B, int max_q, int max_k, int H, int KV, int dtype) {
    const int kb = dtype == 1 ? 32 : 64;
    const long items = (long)B * KV * (((long)max_k + kb - 1) / kb), tiles = ((long)max_q * (H / KV) + 31) / 32;
    if (items >= 128 || tiles < 8) return 1;
    const long want = 256 / items, most = tiles / 4, n = want < most ? want : most;
    return (int)(n < 1 ? 1 : (n > 32 ? 32 : n));
}
constexpr int x_mass_kt(int dtype) { return dtype == 1 ? 4 : 2; }
static int x_mass_split(int B, int max_q, int max_k, int H, int dtype) {
    const int kb = 16 * x_mass_kt(dtype);
    const long items = (long)B * H * (((long)max_k + kb - 1) / kb), trips = ((long)max_q + 15) / 16 / X_MASS_WAVES;
    if (items >= 192 || trips < 8) return 1;
    const long want = 512 / items, most = trips / 2, n = want < most ? want : most;
    return (int)(n < 1 ? 1 : (n > 32 ? 32 : n));
}

template <typename E, int DK, bool DROP> static void launch_xattn_bwd_kernel(const XArgs& a, unsigned grid, hipStream_t stream) {
    constexpr int KB = x_kb<E>(), stage = XTile<E, DK, KB, 1>::BYTES + XTile<E, DK, KB, 2>::BYTES;
    constexpr int rows = (E::PL == 1 ? 8 : 4) * XTile<E, DK, 16, 1>::BYTES, out = 4 * x_out_bytes<typename E::mem, DK>();
    constexpr int tiles = E::PL == 1 ? stage + (stage > rows ? stage : rows) : (stage > rows ? stage : rows), dq = tiles > out ? tiles : out;
    constexpr int key_tiles = E::PL == 1 ? 8 * XTile<E, DK, 32, 2>::BYTES + 2 * XTile<E, DK, 32, 1>::BYTES : 2 * XTile<E, DK, 32, 2>::BYTES + 256;
    constexpr int merge = E::PL == 1 ? 4 * 32 * (DK + 4) * 4 : 0, dkv = key_tiles > merge ? key_tiles : merge, lds = dq > dkv ? dq : dkv;
    static unsigned long long ok = 0;
    fs2_allow_lds((const void*)xattn_bwd_kernel<E, DK, DROP>, lds, &ok);
    hipLaunchKernelGGL((xattn_bwd_kernel<E, DK, DROP>), dim3(grid), dim3(256), lds, stream, a);
}

template <typename E, int DK>
static int launch_xattn_bwd(XArgs& a, int B, int max_q, int max_k, int dk, hipStream_t stream) {
    typedef typename E::mem T;
    constexpr int KEYS = E::PL == 1 ? 32 : 64;
    const long long nq = ((long long)max_q * a.g + 63) / 64, nk = (max_k + KEYS - 1) / KEYS;
    fs2_x_grid(a, (int)nk, a.KV, B);
    const long long line = a.pairs >= 8 ? (a.pairs + 7) / 8 * 8 : a.pairs;
    const long long delta = (long long)B * max_q * ((a.H + X_DELTA_HEADS - 1) / X_DELTA_HEADS);
    // (2^24 workgroups of 256: a launch has fewer than 2^32 work items to a dimension)
    FS2_CHECK_ARG((delta + 15) / 16 < (1 << 24) && line * (nk * a.nsplit + nq) < (1 << 24),
                  "fs2_cross_attention_bwd: B=%d x %d heads x max_q=%d or max_k=%d in one launch", B, a.H, max_q, max_k);
    if (delta > 0 && max_k > 0) {
        hipLaunchKernelGGL((xattn_delta_kernel<T, DK>), dim3((unsigned)((delta + 15) / 16)), dim3(256), 0, stream, a, B);
        FS2_CHECK_LAUNCH("fs2_cross_attention_bwd(delta)");
    }
    a.nblk_q = (int)nq;
    a.key_groups = (unsigned)(line * nk * a.nsplit);
    const unsigned grid = a.key_groups + (unsigned)(line * nq);
    if (a.drop.thresh) launch_xattn_bwd_kernel<E, DK, true>(a, grid, stream);
    else launch_xattn_bwd_kernel<E, DK, false>(a, grid, stream);
    FS2_CHECK_LAUNCH("fs2_cross_attention_bwd");
    if (a.nsplit > 1) {
        const long long n = 2LL * B * max_k * (a.KV * dk / 4);         // (small where rows are split)
        hipLaunchKernelGGL(xattn_dkv_sum_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a, B, dk);
        FS2_CHECK_LAUNCH("fs2_cross_attention_bwd(sum)");
    }
    return FS2_OK;
}

template <typename E, int DK>
static int launch_xattn_mass(XArgs& a, int B, int max_k, hipStream_t stream) {
    constexpr int KT = x_mass_kt(E::PL == 1);
    const long long blocks = ((long long)max_k + 16 * KT - 1) / (16 * KT), line = (long long)B * a.H >= 8 ? 8 * blocks : blocks;
    FS2_CHECK_ARG(line * 64 * X_MASS_WAVES < (1ll << 32), "fs2_cross_attention_mass: B=%d x %d heads x max_k=%d in one launch", B, a.H, max_k);
    constexpr int lds = XTile<E, DK, 16 * KT, 1>::BYTES + X_MASS_WAVES * (E::PL == 1 ? 2 : 1) * XTile<E, DK, 16, 1>::BYTES;
    static unsigned long long ok = 0;
    fs2_allow_lds((const void*)xattn_mass_kernel<E, DK, KT>, lds, &ok);
    const dim3 grid = fs2_x_grid(a, (max_k + 16 * KT - 1) / (16 * KT), a.H, B);
    hipLaunchKernelGGL((xattn_mass_kernel<E, DK, KT>), grid, dim3(64 * X_MASS_WAVES), lds, stream, a);
    FS2_CHECK_LAUNCH("fs2_cross_attention_mass");
    if (a.nsplit > 1) {
        const long long n = (long long)B * max_k * a.H;
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
    if (B <= 0 || max_q <= 0 || max_k <= 0 || Mq <= 0 || Mk <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads) return 16;
    const int n = x_dkv_split(B, max_q, max_k, n_heads, n_kv_heads, dtype);
    return (x_delta_floats(n_heads, Mq) + (n > 1 ? 2LL * n * B * max_k * n_kv_heads * dk : 0)) * (long long)sizeof(float);
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
    FS2_CHECK_ARG(ldv >= n_kv_heads * dk && ldv <= (1 << 20) && ldo >= n_heads * dk && ldo <= (1 << 20) && ldv % epv == 0 && ldo % epv == 0,
                  "fs2_cross_attention_bwd: bad leading dims ldv=%d ldo=%d", ldv, ldo);
    if (max_q == 0 && max_k == 0) return FS2_OK;
    FS2_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0,
                  "fs2_cross_attention_bwd: fs2_cross_attention_bwd_workspace bytes, 16-byte aligned, are needed");
    XArgs a = fs2_x_args(q, k, v, cu_q, cu_k, max_q, max_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq, ldk, ldv, ldo);
    a.ctx = (void*)ctx; a.dctx = dctx; a.lse = (float*)lse; a.dq = dq; a.dk = dk_out; a.dv = dv;
    a.drop = fs2_make_dropout(seed, stream_id, rate);
    a.delta = (float*)workspace;
    a.part = (float*)workspace + x_delta_floats(n_heads, Mq);
    a.nsplit = max_q > 0 && max_k > 0 ? x_dkv_split(B, max_q, max_k, n_heads, n_kv_heads, dtype) : 1;
    a.slots = a.nsplit > 1 ? B * max_k : 0;                 // (few keys where rows are split)
#define FS2_X(TT, DKK) return launch_xattn_bwd<TT, DKK>(a, B, max_q, max_k, dk, stream)
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

extern "C" long long fs2_cross_attention_mass_workspace(int B, int max_q, int max_k, int Mk, int n_heads, int n_kv_heads, int dk,
                                                        int dtype) {
    (void)n_kv_heads; (void)dk;
    if (B <= 0 || max_q <= 0 || max_k <= 0 || Mk <= 0 || n_heads <= 0) return 0;
    const int n = x_mass_split(B, max_q, max_k, n_heads, dtype);
    return n > 1 ? (long long)n * n_heads * B * max_k * (long long)sizeof(float) : 0;
}

extern "C" int fs2_cross_attention_mass(const void* q, const void* k, const float* lse, float* mass, const int* cu_q,
                                        const int* cu_k, void* workspace, int B, int max_q, int max_k, int Mq, int Mk, int n_heads,
                                        int n_kv_heads, int dk, int ldq, int ldk, int dtype, hipStream_t stream) {
    const int rc = fs2_x_check("fs2_cross_attention_mass", q, k, cu_q, cu_k, B, max_q, max_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq,
                               ldk, dtype);
    if (rc != FS2_OK) return rc;
    FS2_CHECK_ARG((lse || Mq == 0) && (mass || Mk == 0), "fs2_cross_attention_mass: null lse or mass");
    if (max_k == 0) return FS2_OK;
    XArgs a = fs2_x_args(q, k, nullptr, cu_q, cu_k, max_q, max_k, Mq, Mk, n_heads, n_kv_heads, dk, ldq, ldk, 0, 0);
    a.lse = (float*)lse;
    a.mass = mass;
    a.nsplit = max_q > 0 ? x_mass_split(B, max_q, max_k, n_heads, dtype) : 1;
    a.slots = a.nsplit > 1 ? B * max_k : 0;
    a.part = (float*)workspace;
    FS2_CHECK_ARG(a.nsplit == 1 || workspace, "fs2_cross_attention_mass: this shape needs fs2_cross_attention_mass_workspace bytes");
#define FS2_X(TT, DKK) return launch_xattn_mass<TT, DKK>(a, B, max_k, stream)
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
