// Shared parts of the cross-attention kernels (cross_attention.hip, cross_attention_bwd.hip): queries of one packed ragged
// matrix against the keys / values of another (frames to phones, phones to frames, one frame at a time), with `g` query
// heads to every key / value head.
//
// Row packing.  The g query heads that share a key / value head meet the same keys, so a work item is a (utterance, SHARED
// head) pair and its query side the g * Lq rows r = q * g + j (query q, head kvh * g + j): K and V are staged once for the
// whole group, and the gradients of shared K / V sum over the group inside the accumulators.
#pragma once
#include "common.h"

namespace fs2 {

struct XArgs {
    const void* q;       // [Mq, ldq] T, head h at columns h * dk
    const void* k;       // [Mk, ldk] T, shared head at columns kvh * dk
    const void* v;       // [Mk, ldv] T
    void* ctx;           // [Mq, ldo] T
    float* lse;          // [H][Mq] log2-domain log-sum-exp (or null)
    const int* cu_q;     // [B + 1]
    const int* cu_k;     // [B + 1]
    int Mq, Mk, max_q, max_k, ldq, ldk, ldv, ldo, H, KV;
    int g;               // H / KV
    unsigned magic;      // floor(2^32 / g) + 1 (g > 1): r / g = umulhi(r, magic) for r < 2^24, g <= 128
    float scale_log2e;   // log2(e) / sqrt(dk)
    float scale;         // 1 / sqrt(dk)
    int nblk, pairs;     // blocks of a pair, (utterance, head) pairs: see x_decode
    int nblk_q;          // backward: row blocks of a pair, and the workgroups in front of the row blocks'
    unsigned key_groups;
    unsigned kv_magic;   // 1 / heads-per-utterance of the pair index
    Dropout drop;        // dropout of the probabilities: site drop.stream + head, row = packed query row, col = key index
    int nsplit;          // ranges of the summed axis over workgroups (1: none), partial results to `part`
    float* part;         // by slot, b * longest + row of the utterance: the rows at work and no others of the matrix
    int slots;           // B * longest (of the queries, or of the keys in the backward and the mass)
    // backward
    const void* dctx;    // [Mq, ldo] T
    float* delta;        // [H][Mq]
    void *dq, *dk, *dv;  // as q, k, v
    float* mass;         // [H][Mk]
};

typedef __attribute__((address_space(3))) void x_lds_void;
typedef const __attribute__((address_space(1))) void x_gbl_void;

// whether a probability stays.  Selecting the scaled value by it (and not multiplying by drop_mul) keeps the registers of 16 multipliers out of
// the loop: 32 x 800 rows over 120 keys, dk = 128, bf16, took 26 us with them and 21 so (18.9 since the V fragments are read in two steps)
__device__ __forceinline__ bool drop_keep(const Dropout& d, uint32_t row, uint32_t col) { return drop_hash(d.seed, d.stream, row, col) >= d.thresh; }

// rows [r0, r0 + len) of utterance b.  The offsets come from device memory: whatever they hold, no access leaves [0, M), and
// an utterance ends after `longest` rows, which the grids and the 32-bit row arithmetic count on
__device__ __forceinline__ void x_range(const int* cu, int b, int M, int longest, int& r0, int& len) {
    const int c0 = min(max(cu[b], 0), M), c1 = min(max(cu[b + 1], c0), M);
    r0 = c0;
    len = min(c1 - c0, longest);
}
// row `slot % longest` of utterance `slot / longest`, -1 if it has none: the rows that the launches behind a split work on
__device__ __forceinline__ int x_row_of(const int* cu, int M, int longest, unsigned slot) {
    const unsigned b = slot / (unsigned)longest;
    int r0, len;
    x_range(cu, (int)b, M, longest, r0, len);
    const int i = (int)(slot - b * (unsigned)longest);
    return i < len ? r0 + i : -1;
}
// packed row -> query index inside the utterance; head in group = r - q * g
__device__ __forceinline__ int x_query(const XArgs& a, int r) { return a.g == 1 ? r : (int)__umulhi((unsigned)r, a.magic); }

// Workgroup order.  Ids are dealt round-robin to the 8 XCDs, each with its own L2; the blocks of one (utterance, head) pair read
// the same keys (or queries), so they go to one XCD: grid (8 nblk, pairs / 8, nsplit), pair 8 y + x % 8, block x / 8.  Fewer than 8
// pairs would leave XCDs idle: grid (nblk, pairs, nsplit), dealt as they come.  Without a division but the pair's.
__device__ __forceinline__ bool x_decode(const XArgs& a, int heads, int& b, int& h, int& blk, int& split) {
    split = blockIdx.z;
    int pair;
    if (a.pairs >= 8) {
        blk = blockIdx.x >> 3;
        pair = blockIdx.y * 8 + (blockIdx.x & 7);
    } else {
        blk = blockIdx.x;
        pair = blockIdx.y;
    }
    if (pair >= a.pairs) return false;
    b = heads == 1 ? pair : (int)__umulhi((unsigned)pair, a.kv_magic);       // exact for pair * heads < 2^32: pair < 2^19, heads <= 4096
    h = pair - b * heads;
    return true;
}

// the same order from the id in a one-dimensional grid of `nblk` blocks to a pair
__device__ __forceinline__ bool x_decode_line(const XArgs& a, unsigned id, unsigned nblk, int& b, int& h, int& blk, int& split) {
    const unsigned ny = a.pairs >= 8 ? (unsigned)(a.pairs + 7) >> 3 : (unsigned)a.pairs, t = a.pairs >= 8 ? id >> 3 : id;
    const unsigned u = t / nblk;
    blk = (int)(t - u * nblk);
    split = (int)(u / ny);
    const int y = (int)u - split * (int)ny, pair = a.pairs >= 8 ? y * 8 + (int)(id & 7) : y;
    if (pair >= a.pairs) return false;
    b = a.KV == 1 ? pair : (int)__umulhi((unsigned)pair, a.kv_magic);
    h = pair - b * a.KV;
    return true;
}

// ---- operands ---------------------------------------------------------------------------------------------------------
// Both types run on the bf16 matrix pipe (v_mfma_f32_16x16x32_bf16, fp32 accumulation).
//   XB16: bf16 operands as they are.
//   XF32: an fp32 value is the exact sum of three bf16 numbers, x0 = x to the nearest, x1 = x - x0 to the nearest, x2 = the rest (|x1| <=
//         2^-8 |x|, |x2| <= 2^-17 |x|, of either sign).  A product of two is x0 y0 + (x0 y1 + x1 y0) + (x0 y2 + x1 y1 + x2 y0) up to
//         (2^-24 + 2^-34) |x y|, six MFMAs of 16 cycles where the fp32 MFMA form of the same tile (eight 16x16x4, 32 cycles each) takes
//         256.  (Planes cut off instead of rounded leave up to 2^-21 |x y|, always towards zero.)
struct XB16 { typedef bf16_t mem; static constexpr int PL = 1; };
struct XF32 { typedef float mem; static constexpr int PL = 3; };
template <typename E> struct XFrag { bf16x8 p[E::PL]; };

template <typename E, int N> __device__ __forceinline__ void x_mma(const XFrag<E> (&a)[N], const XFrag<E>& b, f32x4* c) {
    if constexpr (E::PL == 1) {
#pragma unroll
        for (int n = 0; n < N; ++n) c[n] = mma16(a[n].p[0], b.p[0], c[n]);
    } else {
        constexpr int ia[6] = {2, 1, 0, 1, 0, 0}, ib[6] = {0, 1, 2, 0, 1, 0};        // small terms first
#pragma unroll
        for (int t = 0; t < 6; ++t)
#pragma unroll
            for (int n = 0; n < N; ++n) c[n] = mma16(a[n].p[ia[t]], b.p[ib[t]], c[n]);
    }
}

// the three planes of two values, packed in pairs.  Between bf16's largest number and fp32's the first plane stays at the former instead of
// rounding to infinity (CLAMP: values from memory; weights and their gradients are not that large).  An infinity becomes a NaN: infinity
// - infinity is in its rest.  32 x 120 rows over 810 keys, dk = 96: 60.0 us, 58.5 without the clamp, 56.2 with planes cut off.
__device__ __forceinline__ uint32_t x_round2(float a, float b) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    return __builtin_bit_cast(uint32_t, (bf16x2){(bf16_t)a, (bf16_t)b});
}
template <bool CLAMP> __device__ __forceinline__ void x_split2(float a, float b, uint32_t& w0, uint32_t& w1, uint32_t& w2) {
    constexpr float most = 3.3895313892515355e38f;
    w0 = CLAMP ? x_round2(__builtin_amdgcn_fmed3f(a, -most, most), __builtin_amdgcn_fmed3f(b, -most, most)) : x_round2(a, b);
    const float ra = a - __builtin_bit_cast(float, w0 << 16), rb = b - __builtin_bit_cast(float, w0 & 0xffff0000u);
    w1 = x_round2(ra, rb);
    w2 = x_round2(ra - __builtin_bit_cast(float, w1 << 16), rb - __builtin_bit_cast(float, w1 & 0xffff0000u));
}
struct XRaw { float v[8]; };          // eight consecutive fp32 values on their way to a fragment
template <bool CLAMP> __device__ __forceinline__ XFrag<XF32> x_split8(const XRaw& x) {
    uint4 w[3];
    x_split2<CLAMP>(x.v[0], x.v[1], w[0].x, w[1].x, w[2].x);
    x_split2<CLAMP>(x.v[2], x.v[3], w[0].y, w[1].y, w[2].y);
    x_split2<CLAMP>(x.v[4], x.v[5], w[0].z, w[1].z, w[2].z);
    x_split2<CLAMP>(x.v[6], x.v[7], w[0].w, w[1].w, w[2].w);
    XFrag<XF32> f;
#pragma unroll
    for (int pl = 0; pl < 3; ++pl) f.p[pl] = __builtin_bit_cast(bf16x8, w[pl]);
    return f;
}
__device__ __forceinline__ XRaw x_raw(const float* p) {
    XRaw r;
    *(f32x4*)&r.v[0] = *(const f32x4*)p;
    *(f32x4*)&r.v[4] = *(const f32x4*)(p + 4);
    return r;
}
// eight consecutive elements of memory as an operand
template <typename E> __device__ __forceinline__ XFrag<E> x_load(const typename E::mem* p) {
    if constexpr (E::PL == 1) {
        XFrag<E> f;
        f.p[0] = *(const bf16x8*)p;
        return f;
    } else {
        return x_split8<true>(x_raw(p));
    }
}
// element j of an operand
template <typename E> __device__ __forceinline__ float x_value(const XFrag<E>& f, int j) {
    float v = to_f32(f.p[E::PL - 1][j]);
#pragma unroll
    for (int pl = E::PL - 2; pl >= 0; --pl) v += to_f32(f.p[pl][j]);
    return v;
}
// accumulator pair -> operand (k-slot (g, jj) <-> row 16 (jj / 4) + 4 g + jj % 4 of the 32)
template <typename E> __device__ __forceinline__ XFrag<E> x_pack(const f32x4& lo, const f32x4& hi) {
    if constexpr (E::PL == 1) {
        XFrag<E> f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            f.p[0][r] = (bf16_t)lo[r];
            f.p[0][4 + r] = (bf16_t)hi[r];
        }
        return f;
    } else {
        XRaw x;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x.v[r] = lo[r];
            x.v[4 + r] = hi[r];
        }
        return x_split8<false>(x);
    }
}

// bf16: a value goes into a product as two numbers, or the sum over keys (or rows) carries its rounding: with P as one number ctx and
// dv were 1.2 .. 1.4 times as far off as rounding the result alone, with dS as one dq and dk 1.4 .. 1.55 times.
// What x_pack<XB16> rounded away, as another operand (dS).
__device__ __forceinline__ XFrag<XB16> x_pack_rest(const f32x4& lo, const f32x4& hi, const XFrag<XB16>& f) {
    XFrag<XB16> r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        r.p[0][e] = (bf16_t)(lo[e] - (float)f.p[0][e]);
        r.p[0][4 + e] = (bf16_t)(hi[e] - (float)f.p[0][4 + e]);
    }
    return r;
}
// Weights >= 0 (P) as f + r, both > 0 where the weight is: f is the weight cut off, r what is left, below 2^-7 of it, and 2^-23 of it more so
// that it is never zero, rounded to half a step: together off by 2^-15.  A remainder of either sign, or of zero, would make NaN of an
// infinite value's weight times infinity.
__device__ __forceinline__ void x_pack_weights(const f32x4& lo, const f32x4& hi, XFrag<XB16>& f, XFrag<XB16>& r) {
    uint4 w;
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const float a = e < 4 ? lo[e] : hi[e - 4], b = e < 4 ? lo[e + 1] : hi[e - 3];
        const uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
        ((uint32_t*)&w)[e >> 1] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
        rest[e] = fmaf(a, 1.0f + 0x1p-23f, -__builtin_bit_cast(float, ua & 0xffff0000u));
        rest[e + 1] = fmaf(b, 1.0f + 0x1p-23f, -__builtin_bit_cast(float, ub & 0xffff0000u));
    }
    f.p[0] = __builtin_bit_cast(bf16x8, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) r.p[0][e] = (bf16_t)rest[e];
}

// A transposed fragment (XTile::col_frag, c = 0) of a tile with `left` rows: those behind them, copies of the last one, become zero.  Their
// weights are zero, but zero times an infinite element is NaN.
__device__ __forceinline__ void x_keep_rows(XFrag<XB16>& f, int left, int g) {
    uint4 w = __builtin_bit_cast(uint4, f.p[0]);
    auto mask = [](int n) { return n >= 2 ? 0xffffffffu : (n == 1 ? 0xffffu : 0u); };
    const int n = left - 4 * g;
    w.x &= mask(n);
    w.y &= mask(n - 2);
    w.z &= mask(n - 16);
    w.w &= mask(n - 18);
    f.p[0] = __builtin_bit_cast(bf16x8, w);
}

// ---- tiles of ROWS rows x DK in LDS ---------------------------------------------------------------------------------
// Fragment reads take one 16-byte slot of 16 rows, transposed reads 32 bytes of 8 rows at a time; both should meet all 64 banks once.
//   XB16 (filled by LDS-DMA, lane-linear): unpadded rows whose slots are rotated by WAY * (row >> RSH); rows narrower than 256 bytes
//         share a rotation where several of them make up one pass over the banks.
//   XF32 (three planes, written by ds_write): rows padded to an odd number of slots (WAY 1, read row-wise) or to 2 more than the
//         slots (WAY 2, read transposed, or both ways).  dk = 96 rotated like XB16 spent 54 % of its LDS cycles on conflicts.
template <typename E, int DK, int ROWS, int WAY> struct XTile {
    typedef typename E::mem T;
    typedef XFrag<E> frag_t;
    static constexpr int NS = DK / 8;                                                   // slots of a row
    static constexpr int ROWB = E::PL == 1 ? DK * 2 : (WAY == 1 ? (NS | 1) : NS + 2) * 16;
    static constexpr int PLANE = ROWS * ROWB;
    static constexpr int BYTES = E::PL * PLANE;
    static constexpr int KS = DK / 32;
    static constexpr int DT = DK / 16;
    static constexpr int RSH = DK == 64 ? 1 : (DK == 32 ? 2 : 0);

    // byte of logical slot `slot` of row `row`
    static __device__ __forceinline__ int at(int row, int slot) {
        if constexpr (E::PL == 1) return row * ROWB + ((slot + WAY * (row >> RSH)) % NS) * 16;
        return row * ROWB + slot * 16;
    }
    // row `row`, elements 32 ks + 8 g .. + 7
    static __device__ __forceinline__ frag_t row_frag(const unsigned char* img, int row, int ks, int g) {
        frag_t f;
        const unsigned char* p = img + at(row, ks * 4 + g);
#pragma unroll
        for (int pl = 0; pl < E::PL; ++pl) f.p[pl] = *(const bf16x8*)(p + pl * PLANE);
        return f;
    }
    // column 16 dt + i, rows 32 c + {4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3}: the slot map of an accumulator used as operand.
    // Transposed 4 x 16 block reads: lane 4 q + p of a 16-lane group supplies row q, columns 4 p .. 4 p + 3
    static __device__ __forceinline__ frag_t col_frag(const unsigned char* img, int c, int dt, int g, int i) {
        frag_t f;
        const int row0 = 32 * c + 4 * g + (i >> 2), slot = dt * 2 + ((i & 3) >> 1), sub = (i & 1) * 8;
        const unsigned char *p0 = img + at(row0, slot) + sub, *p1 = img + at(row0 + 16, slot) + sub;
#pragma unroll
        for (int pl = 0; pl < E::PL; ++pl) {
            const bf16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(p0 + pl * PLANE));
            const bf16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(p1 + pl * PLANE));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                f.p[pl][r] = lo4[r];
                f.p[pl][4 + r] = hi4[r];
            }
        }
        return f;
    }
};

// Keys of a tile: bf16 64, two stages filled by LDS-DMA; fp32 32, one stage in three planes, the next tile loaded ahead into registers
// and split on the way into LDS (64 would leave room for one workgroup on a CU, and for too few registers).
template <typename E> constexpr int x_kb() { return E::PL == 3 ? 32 : 64; }

// ---- memory -> tile, by NW waves ---------------------------------------------------------------------------------------
// fetch() starts the rows [0, left) at `tile` (clamped to the last of them), put() finishes.  Sources are 32-bit byte offsets from the
// tile's first row, clamped by min() (of offsets in one column: the offset of the smaller row).
//   XB16: fetch is LDS-DMA (16 bytes a lane, lane-linear on the LDS side: the rotation goes into the source), put nothing; the caller
//         waits vmcnt(0).  Power-of-two rows: the swizzle repeats every (NS << RSH) / WAY rows, a wave needs one period's offsets.
//   XF32: fetch loads into registers (32 bytes a lane and 16-byte slot), put splits them and writes the three planes.
// Packed rows of the g > 1 query heads of a shared head (`rows`): the address is worked out row by row.
template <typename E, int DK, int ROWS, int WAY, int NW> struct XFetch;

template <int DK, int ROWS, int WAY, int NW> struct XFetch<XB16, DK, ROWS, WAY, NW> {
    typedef XTile<XB16, DK, ROWS, WAY> TL;
    static constexpr int PIECES = TL::BYTES / 1024, PP = PIECES / NW, NS = TL::NS, ROWB = TL::ROWB;
    static_assert(PIECES % NW == 0, "the same number of pieces for every wave");
    static constexpr bool POW2 = (NS & (NS - 1)) == 0;
    static constexpr int STEP = NW * 1024 / ROWB, PERIOD = (NS << TL::RSH) / WAY;          // rows between a wave's pieces
    static constexpr int N = !POW2 ? PP : (PERIOD <= STEP ? 1 : (PERIOD / STEP < PP ? PERIOD / STEP : PP));
    unsigned off[N], col[N];
    __device__ __forceinline__ XFetch(int ld, int wave, int lane) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int o = (wave + NW * n) * 1024 + lane * 16, row = o / ROWB, slot = (o % ROWB) >> 4;
            col[n] = (unsigned)((slot + WAY * NS - (WAY * (row >> TL::RSH)) % NS) % NS) * 16u;       // physical slot `slot` holds this one
            off[n] = (unsigned)row * (unsigned)ld * 2u + col[n];
        }
    }
    __device__ __forceinline__ void fetch(const bf16_t* __restrict__ tile, int ld, int left, unsigned char* dst, int wave, int) {
        const unsigned ldb = (unsigned)ld * 2u, last = (unsigned)(min(left, ROWS) - 1) * ldb;
#pragma unroll
        for (int pp = 0; pp < PP; ++pp) {
            const unsigned so = min(off[pp % N] + (unsigned)(pp / N * N * STEP) * ldb, last + col[pp % N]);
            __builtin_amdgcn_global_load_lds((x_gbl_void*)((const unsigned char*)tile + so), (x_lds_void*)(dst + (wave + NW * pp) * 1024),
                                             16, 0, 0);
        }
    }
    __device__ __forceinline__ void fetch_rows(const XArgs& a, const bf16_t* __restrict__ base, int ld, int first, int nrow,
                                               unsigned char* dst, int wave, int lane) {
#pragma unroll 1
        for (int pp = 0; pp < PP; ++pp) {
            const int p = wave + NW * pp, o = p * 1024 + lane * 16, row = o / ROWB, slot = (o % ROWB) >> 4;
            const int r = min(first + row, nrow - 1), q = x_query(a, r);
            const int s = (slot + WAY * NS - (WAY * (row >> TL::RSH)) % NS) % NS;
            __builtin_amdgcn_global_load_lds((x_gbl_void*)(base + (size_t)q * ld + (r - q * a.g) * DK + s * 8), (x_lds_void*)(dst + p * 1024),
                                             16, 0, 0);
        }
    }
    __device__ __forceinline__ void put(unsigned char*, int, int) {}
};

template <int DK, int ROWS, int WAY, int NW> struct XFetch<XF32, DK, ROWS, WAY, NW> {
    typedef XTile<XF32, DK, ROWS, WAY> TL;
    static constexpr int CPR = DK / 4, CHUNKS = ROWS * CPR;                     // 16-byte chunks of a row, of the tile
    static constexpr int N = (CHUNKS + 64 * NW - 1) / (64 * NW);                // of a lane (the last of them may be missing)
    static __device__ __forceinline__ bool has(int id) { return CHUNKS % (64 * NW) == 0 || id < CHUNKS; }
    f32x4 r[N];
    unsigned off[N];
    __device__ __forceinline__ XFetch(int ld, int wave, int lane) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int id = n * 64 * NW + wave * 64 + lane, row = id / CPR, c = id - row * CPR;
            off[n] = (unsigned)row * (unsigned)ld * 4u + (unsigned)c * 16u;
        }
    }
    __device__ __forceinline__ void fetch(const float* __restrict__ tile, int ld, int left, unsigned char*, int wave, int lane) {
        if (left >= ROWS) {
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (has(n * 64 * NW + wave * 64 + lane)) r[n] = *(const f32x4*)((const unsigned char*)tile + off[n]);
            return;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int id = n * 64 * NW + wave * 64 + lane, row = id / CPR, c = id - row * CPR;
            if (has(id))
                r[n] = *(const f32x4*)((const unsigned char*)tile + (unsigned)min(row, left - 1) * (unsigned)ld * 4u + (unsigned)c * 16u);
        }
    }
    __device__ __forceinline__ void fetch_rows(const XArgs& a, const float* __restrict__ base, int ld, int first, int nrow, unsigned char*,
                                               int wave, int lane) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int id = n * 64 * NW + wave * 64 + lane, row = id / CPR, c = id - row * CPR;
            const int rr = min(first + row, nrow - 1), q = x_query(a, rr);
            if (has(id)) r[n] = *(const f32x4*)(base + (size_t)q * ld + (rr - q * a.g) * DK + c * 4);
        }
    }
    __device__ __forceinline__ void put(unsigned char* dst, int wave, int lane) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int id = n * 64 * NW + wave * 64 + lane, row = id / CPR, c = id - row * CPR;
            if (!has(id)) continue;
            uint2 w[3];
            x_split2<true>(r[n][0], r[n][1], w[0].x, w[1].x, w[2].x);
            x_split2<true>(r[n][2], r[n][3], w[0].y, w[1].y, w[2].y);
            unsigned char* at = dst + TL::at(row, c >> 1) + (c & 1) * 8;
#pragma unroll
            for (int pl = 0; pl < 3; ++pl) *(uint2*)(at + pl * TL::PLANE) = w[pl];
        }
    }
};

// A wave's own packed rows [first, first + ROWS) of the heads at `base` as operands, through its own LDS (XTile<E, DK, ROWS, 1>::BYTES):
// a fragment load straight from memory has 16 rows in consecutive lanes, one cache access per lane instead of one per line (64
// against 8 at dk = 128; the attention mass of 32 x 800 queries spent 9 us of cache accesses that way).  start(), then finish().
template <typename E, int DK, int ROWS> struct XRows {
    typedef XTile<E, DK, ROWS, 1> TL;
    XFetch<E, DK, ROWS, 1, 1> f;
    __device__ __forceinline__ XRows(int ld, int lane) : f(ld, 0, lane) {}
    __device__ __forceinline__ void start(const XArgs& a, const typename E::mem* __restrict__ base, int ld, int first, int nrow,
                                          unsigned char* lds, int lane) {
        if (a.g == 1)
            f.fetch(base + (size_t)first * ld, ld, nrow - first, lds, 0, lane);
        else
            f.fetch_rows(a, base, ld, first, nrow, lds, 0, lane);
    }
    // XB16: what start() began has landed (vmcnt(0) waits for everything the wave has under way)
    __device__ __forceinline__ void finish(unsigned char* lds, int lane) {
        f.put(lds, 0, lane);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
};

// Rows of results back to memory: accumulators of 16 packed rows (lane (g, i): row i, columns 16 dt + 4 g ..) through the wave's own
// LDS (16 x (DK * 4 + 16) bytes at most), then 16 bytes a lane along the rows.
template <typename T, int DK> constexpr int x_out_bytes() { return 16 * (DK * (int)sizeof(T) + 16); }
template <typename T, int DK>
__device__ __forceinline__ void x_store_rows(const XArgs& a, T* __restrict__ dst, int ld, int q0, int kvh, int first, int nrow,
                                             const f32x4 (&v)[DK / 16], unsigned char* lds, int lane) {
    constexpr int PITCH = DK * (int)sizeof(T) + 16, CPR = DK * (int)sizeof(T) / 16, N = 16 * CPR / 64;
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int dt = 0; dt < DK / 16; ++dt) store4<T>((T*)(lds + i * PITCH) + dt * 16 + 4 * g, v[dt]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int id = n * 64 + lane, row = id / CPR, c = id - row * CPR, r = first + row;
        if (r < nrow) {
            const int q = x_query(a, r);
            *(vec16*)((unsigned char*)(dst + (size_t)(q0 + q) * ld + (kvh * a.g + r - q * a.g) * DK) + c * 16) =
                *(const vec16*)(lds + row * PITCH + c * 16);
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // read before the next rows overwrite it
}

}  // namespace fs2

// ---- host side: the checks every entry point of the family shares ------------------------------------------------
static inline int fs2_x_check(const char* who, const void* q, const void* k, const int* cu_q, const int* cu_k, int B, int max_q,
                              int max_k, int Mq, int Mk, int H, int KV, int dk, int ldq, int ldk, int dtype) {
    FS2_CHECK_ARG(cu_q && cu_k && B > 0 && Mq >= 0 && Mk >= 0 && max_q >= 0 && max_k >= 0, "%s: bad args", who);
    FS2_CHECK_ARG((q || Mq == 0) && (k || Mk == 0), "%s: null q or k", who);
    FS2_CHECK_ARG(dtype == 0 || dtype == 1, "%s: dtype=%d (0 fp32, 1 bf16)", who, dtype);
    FS2_CHECK_ARG(dk == 32 || dk == 64 || dk == 96 || dk == 128, "%s: head dim %d unsupported (32/64/96/128)", who, dk);
    FS2_CHECK_ARG(H > 0 && KV > 0 && H % KV == 0 && H / KV <= 128 && H <= 4096, "%s: %d heads over %d key heads", who, H, KV);
    FS2_CHECK_ARG(B <= 65535 && max_q <= Mq && max_k <= Mk, "%s: B=%d (<= 65535), max_q=%d > Mq=%d or max_k=%d > Mk=%d", who, B,
                  max_q, Mq, max_k, Mk);
    FS2_CHECK_ARG((long long)max_q * (H / KV) <= (1 << 24), "%s: max_q=%d with %d heads to a key head", who, max_q, H / KV);
    FS2_CHECK_ARG(max_k <= (1 << 30), "%s: max_k=%d beyond 2^30", who, max_k);
    const long long longest = (long long)max_q * (H / KV) > max_k ? (long long)max_q * (H / KV) : max_k;
    FS2_CHECK_ARG((long long)B * H <= (1 << 19) && (long long)B * H * ((longest + 31) / 32) < (1ll << 30),
                  "%s: B=%d x %d heads x %lld rows in one launch", who, B, H, longest);
    const int epv = dtype == 0 ? 4 : 8;
    FS2_CHECK_ARG(ldq <= (1 << 20) && ldk <= (1 << 20), "%s: leading dims ldq=%d, ldk=%d beyond 2^20", who, ldq, ldk);
    FS2_CHECK_ARG(ldq >= H * dk && ldk >= KV * dk && ldq % epv == 0 && ldk % epv == 0, "%s: bad leading dims ldq=%d ldk=%d", who, ldq,
                  ldk);
    FS2_CHECK_ARG(((uintptr_t)q & 15) == 0 && ((uintptr_t)k & 15) == 0, "%s: unaligned q or k", who);
    return FS2_OK;
}

// grid of x_decode
static inline dim3 fs2_x_grid(fs2::XArgs& a, int nblk, int heads, int B) {
    a.nblk = nblk;
    a.pairs = B * heads;
    a.kv_magic = heads > 1 ? (unsigned)((1ull << 32) / heads + 1) : 0u;
    return a.pairs >= 8 ? dim3(8 * nblk, (a.pairs + 7) / 8, a.nsplit) : dim3(nblk, a.pairs, a.nsplit);
}

static inline fs2::XArgs fs2_x_args(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, int max_q, int max_k,
                                    int Mq, int Mk, int H, int KV, int dk, int ldq, int ldk, int ldv, int ldo) {
    fs2::XArgs a = {};
    a.q = q; a.k = k; a.v = v; a.cu_q = cu_q; a.cu_k = cu_k;
    a.Mq = Mq; a.Mk = Mk; a.max_q = max_q; a.max_k = max_k; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo;
    a.H = H; a.KV = KV; a.g = H / KV;
    a.magic = a.g > 1 ? (unsigned)((1ull << 32) / a.g + 1) : 0u;
    a.scale = 1.0f / sqrtf((float)dk);
    a.scale_log2e = 1.4426950408889634f * a.scale;
    a.nsplit = 1;
    return a;
}
