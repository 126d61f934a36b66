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
    int Mq, Mk, ldq, ldk, ldv, ldo, H, KV;
    int g;               // H / KV
    unsigned magic;      // floor(2^32 / g) + 1 (g > 1): r / g = umulhi(r, magic) for r < 2^24, g <= 128
    float scale_log2e;   // log2(e) / sqrt(dk)
    float scale;         // 1 / sqrt(dk)
    PairOrder order;     // workgroup order over (utterance, shared head) pairs
    Dropout drop;        // dropout of the probabilities: site drop.stream + head, row = packed query row, col = key index
    int nsplit;          // ranges of the summed axis over workgroups (1: none), partial results to `part`
    float* part;
    // backward
    const void* dctx;    // [Mq, ldo] T
    float* delta;        // [H][Mq]
    void *dq, *dk, *dv;  // as q, k, v
    float* mass;         // [H][Mk]
};

typedef __attribute__((address_space(3))) void x_lds_void;
typedef const __attribute__((address_space(1))) void x_gbl_void;

// rows [r0, r0 + len) of utterance b.  The offsets come from device memory: whatever they hold, no access leaves [0, M)
__device__ __forceinline__ void x_range(const int* cu, int b, int M, int& r0, int& len) {
    const int c0 = min(max(cu[b], 0), M), c1 = min(max(cu[b + 1], c0), M);
    r0 = c0;
    len = c1 - c0;
}
// packed row -> query index inside the utterance; head in group = r - q * g
__device__ __forceinline__ int x_query(const XArgs& a, int r) { return a.g == 1 ? r : (int)__umulhi((unsigned)r, a.magic); }

// Tiles of ROWS rows x DK in LDS: unpadded rows whose 16-byte slots are rotated by ROT * (row >> RSH), so that fragment reads
// of 16 rows (ROT = 1) and transposed reads of 4 rows x 64 bytes (ROT = 2) spread over the banks; rows narrower than 256
// bytes share a rotation where several of them make up one pass over the banks.  Filled by LDS-DMA (lane-linear on the LDS
// side): the rotation goes into the source address.
template <typename T, int DK, int ROWS = 64> struct XTile {
    static constexpr int ROWB = DK * (int)sizeof(T);
    static constexpr int NS = ROWB / 16;
    static constexpr int BYTES = ROWS * ROWB;
    static constexpr int PIECES = BYTES / 1024;
    static constexpr int EPS = 16 / (int)sizeof(T);
    static constexpr int KS = DK / 32;
    static constexpr int DT = DK / 16;
    static constexpr int RSH = ROWB == 128 ? 1 : (ROWB == 64 ? 2 : 0);
    typedef typename Frag<T>::type frag_t;

    template <int ROT> static __device__ __forceinline__ int rot(int row) { return (ROT * (row >> RSH)) % NS; }

    // rows [first, first + ROWS) of a plain matrix, clamped to its last row (`len` > 0)
    template <int ROT, int NW>
    static __device__ __forceinline__ void stage(const T* __restrict__ base, int ld, int first, int len, unsigned char* dst,
                                                 int wave, int lane) {
        static_assert(PIECES % NW == 0, "the same number of pieces for every wave");
#pragma unroll
        for (int pp = 0; pp < PIECES / NW; ++pp) {
            const int p = wave + NW * pp;
            const int off = p * 1024 + lane * 16, row = off / ROWB, slot = (off % ROWB) >> 4;
            const int r = min(first + row, len - 1);
            const int s = (slot + NS - rot<ROT>(row)) % NS;      // physical slot `slot` holds logical slot s
            __builtin_amdgcn_global_load_lds((x_gbl_void*)(base + (size_t)r * ld + s * EPS), (x_lds_void*)(dst + p * 1024), 16, 0, 0);
        }
    }
    // packed rows [first, first + ROWS) of the g heads that share a key head: `base` at the group's first head
    template <int ROT, int NW>
    static __device__ __forceinline__ void stage_rows(const XArgs& a, const T* __restrict__ base, int ld, int first, int nrow,
                                                      unsigned char* dst, int wave, int lane) {
        static_assert(PIECES % NW == 0, "the same number of pieces for every wave");
#pragma unroll
        for (int pp = 0; pp < PIECES / NW; ++pp) {
            const int p = wave + NW * pp;
            const int off = p * 1024 + lane * 16, row = off / ROWB, slot = (off % ROWB) >> 4;
            const int r = min(first + row, nrow - 1);
            const int q = x_query(a, r);
            const int s = (slot + NS - rot<ROT>(row)) % NS;
            __builtin_amdgcn_global_load_lds((x_gbl_void*)(base + (size_t)q * ld + (r - q * a.g) * DK + s * EPS),
                                             (x_lds_void*)(dst + p * 1024), 16, 0, 0);
        }
    }
    // row `row`, elements 32 ks + 8 g .. + 7
    template <int ROT> static __device__ __forceinline__ frag_t row_frag(const unsigned char* img, int row, int ks, int g) {
        const unsigned char* rowp = img + row * ROWB;
        if constexpr (sizeof(T) == 2) {
            return *(const frag_t*)(rowp + (((ks * 4 + g) + rot<ROT>(row)) % NS) * 16);
        } else {
            const f32x4 v0 = *(const f32x4*)(rowp + (((ks * 8 + 2 * g) + rot<ROT>(row)) % NS) * 16);
            const f32x4 v1 = *(const f32x4*)(rowp + (((ks * 8 + 2 * g + 1) + rot<ROT>(row)) % NS) * 16);
            return (frag_t){v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        }
    }
    // column 16 dt + i, rows 32 c + {4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3}: the slot map of an accumulator used as operand
    template <int ROT> static __device__ __forceinline__ frag_t col_frag(const unsigned char* img, int c, int dt, int g, int i) {
        frag_t f;
        if constexpr (sizeof(T) == 2) {
            // transposed 4 x 16 block read: lane 4 q + p of a 16-lane group supplies row q, columns 4 p .. 4 p + 3
            const int row0 = 32 * c + 4 * g + (i >> 2), row1 = row0 + 16;
            const int slot = dt * 2 + ((i & 3) >> 1), sub = (i & 1) * 8;
            const unsigned char* p0 = img + row0 * ROWB + ((slot + rot<ROT>(row0)) % NS) * 16 + sub;
            const unsigned char* p1 = img + row1 * ROWB + ((slot + rot<ROT>(row1)) % NS) * 16 + sub;
            const bf16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)p0);
            const bf16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)p1);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                f[r] = lo4[r];
                f[4 + r] = hi4[r];
            }
        } else {
#pragma unroll
            for (int jj = 0; jj < 8; ++jj) {
                const int row = 32 * c + 16 * (jj >> 2) + 4 * g + (jj & 3), col = dt * 16 + i;
                f[jj] = *(const T*)(img + row * ROWB + (((col >> 2) + rot<ROT>(row)) % NS) * 16 + (col & 3) * 4);
            }
        }
        return f;
    }
};

// accumulator pair -> operand fragment (k-slot (g, jj) <-> row 16 (jj / 4) + 4 g + jj % 4 of the 32)
template <typename T> __device__ __forceinline__ typename Frag<T>::type x_pack(const f32x4& lo, const f32x4& hi) {
    typename Frag<T>::type f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        f[r] = from_f32<T>(lo[r]);
        f[4 + r] = from_f32<T>(hi[r]);
    }
    return f;
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
    const long long longest = (long long)max_q * (H / KV) > max_k ? (long long)max_q * (H / KV) : max_k;
    FS2_CHECK_ARG((long long)B * H * ((longest + 63) / 64) < (1ll << 30), "%s: B=%d x %d heads x %lld rows in one launch", who, B, H,
                  longest);
    const int epv = dtype == 0 ? 4 : 8;
    FS2_CHECK_ARG(ldq >= H * dk && ldk >= KV * dk && ldq % epv == 0 && ldk % epv == 0, "%s: bad leading dims ldq=%d ldk=%d", who, ldq,
                  ldk);
    FS2_CHECK_ARG(((uintptr_t)q & 15) == 0 && ((uintptr_t)k & 15) == 0, "%s: unaligned q or k", who);
    return FS2_OK;
}

static inline fs2::XArgs fs2_x_args(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, int Mq, int Mk, int H,
                                    int KV, int dk, int ldq, int ldk, int ldv, int ldo) {
    fs2::XArgs a = {};
    a.q = q; a.k = k; a.v = v; a.cu_q = cu_q; a.cu_k = cu_k;
    a.Mq = Mq; a.Mk = Mk; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo;
    a.H = H; a.KV = KV; a.g = H / KV;
    a.magic = a.g > 1 ? (unsigned)((1ull << 32) / a.g + 1) : 0u;
    a.scale = 1.0f / sqrtf((float)dk);
    a.scale_log2e = 1.4426950408889634f * a.scale;
    a.nsplit = 1;
    return a;
}
