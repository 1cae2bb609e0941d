// Shared pieces of the attention over token sequences (band_attn_fwd.hip, band_attn_step.hip, band_attn_bwd.hip).
//
//   query row i of sequence b stands at p = k_len - q_len + i; key j < k_len is visible when j <= p + right and
//   (j >= p - left or j < sinks);  x_j = log2(e) * (scale * q.k_j + bias[clip(j - p)]);  out = sum 2^(x_j - lse) v_j
//
// All products run on 32x32 MFMA tiles with the softmax rows on the lane axis of the accumulators, so that the
// probabilities of a tile are, as they stand in the registers, the second operand of the product behind them.
#pragma once
#include <cfloat>

#include "attn_common.hpp"

namespace dsw {

constexpr int BAND_TILE = 64;    // keys (forward, dQ) or query rows (dK, dV) staged at a time
constexpr int BAND_ROWS = 128;   // query rows (forward, dQ) or keys (dK, dV) of a workgroup: 4 waves x 32
constexpr int BAND_MARGIN = 96;  // a tile of 64 x 32 spans 95 distances: entries past the clip distance in the LDS bias
constexpr int BAND_MAX_DISTANCE = 512;
constexpr int BAND_FAR = 1 << 29;  // "unlimited": beyond every length, and sums of two stay inside 32 bits

struct BandTensor {
    const void *p;
    dsw_strides s;
};
// How a call's tensors are accessed, a template argument of the kernels (a branch per access cost more than the access):
// 0  16-byte pieces: D and all strides multiples of 16 bytes, rows 16-byte aligned; bf16 tiles go to LDS without registers
// 1  4-byte pieces: everything a multiple of 4 bytes, and 8 <= D (heads of 30); bf16 tiles go to LDS without registers
// 2  single elements (D < 8, odd sizes in bf16, or rows so far apart that a tile spans 2 GiB)

struct BandArgs {
    BandTensor q, k, v, out, dout, dq, dk, dv;
    int B, Lq, Lk, Hq, Hkv, G, D;
    int left, right, sinks;
    float c, scale;  // scale * log2(e), scale
    const int *q_lens, *k_lens;
    const float *table;  // [n_buckets][Hq] or null
    const int *buckets;  // [2 M + 1]
    int n_buckets, M;
    float *lse;          // [B][Hq][Lq], base 2; +inf for rows without a visible key (2^(x - inf) = 0 in the backward)
    float *top;          // with a bias table: [B][Hq][Lq], taken out of lse (see band_keep)
    float *lse_rest;     // fp32 calls without a bias table: [B][Hq][Lq] or null, what the rounding of lse left behind
    float *out32;        // [B][Lq][Hq][D] or null
    bf16_t *rest;        // [B][Lq][Hq][D] or null: out before its rounding, less out
    float *delta;        // [B][Hq][Lq]
    float *partial;      // step kernel: see there; dQ kernel: bias gradients by distance
    int nsplit, nrb, staged;  // step kernel; staged: floats of the bias by head and distance in LDS, or 0
    float *shares;       // dK, dV kernel: sums of the blocks that several workgroups share
    int sink_blocks, sink_chunks, chunks;
};

// ---- element types ------------------------------------------------------------------------------------------
// A fragment is the 8 elements a lane hands to one 32x32x16 product: row (or column) lane % 32, k = 8 * (lane / 32)...
template <typename T> struct band_t;
template <> struct band_t<bf16_t> {
    typedef uint4 frag;
    template <int DP> static constexpr int elems(int rows) { return rows * DP; }
    static constexpr int nbuf(int) { return 2; }
};
template <> struct band_t<float> {
    struct frag { float4 lo, hi; };
    template <int DP> static constexpr int elems(int rows) { return rows * (DP + 4); }
    static constexpr int nbuf(int dp) { return dp == 128 ? 1 : 2; }
};

__device__ __forceinline__ f32x16 band_mma(const uint4 &a, const uint4 &b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 band_mma(const band_t<float>::frag &a, const band_t<float>::frag &b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo.x, b.lo.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo.y, b.lo.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo.z, b.lo.z, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo.w, b.lo.w, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi.x, b.hi.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi.y, b.hi.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi.z, b.hi.z, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi.w, b.hi.w, c, 0, 0, 0);
    return c;
}

// l + the sum of a fragment's elements, as they enter the product behind it
typedef __bf16 band_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float band_sum(const uint4 &f, float l) {
    const band_bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
    l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(band_bf16x2, f.x), one, l, false);
    l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(band_bf16x2, f.y), one, l, false);
    l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(band_bf16x2, f.z), one, l, false);
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(band_bf16x2, f.w), one, l, false);
}
__device__ __forceinline__ float band_sum(const band_t<float>::frag &f, float l) {
    return l + (((f.lo.x + f.lo.y) + (f.lo.z + f.lo.w)) + ((f.hi.x + f.hi.y) + (f.hi.z + f.hi.w)));
}

__device__ __forceinline__ f32x16 band_zero() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

// registers 8c .. 8c+7 of a 32x32 result as a fragment (bf16: rounded to nearest even)
__device__ __forceinline__ void band_pack(const f32x16 &s, int c, uint4 &f) {
    f = make_uint4(pack_bf16(s[8 * c], s[8 * c + 1]), pack_bf16(s[8 * c + 2], s[8 * c + 3]),
                   pack_bf16(s[8 * c + 4], s[8 * c + 5]), pack_bf16(s[8 * c + 6], s[8 * c + 7]));
}
__device__ __forceinline__ void band_pack(const f32x16 &s, int c, band_t<float>::frag &f) {
    f.lo = make_float4(s[8 * c], s[8 * c + 1], s[8 * c + 2], s[8 * c + 3]);
    f.hi = make_float4(s[8 * c + 4], s[8 * c + 5], s[8 * c + 6], s[8 * c + 7]);
}
// what the rounding of v to a fragment left behind: subtracted from v, and rounded in its turn; with two such rests a
// fragment carries the 24 bits of fp32
__device__ __forceinline__ uint32_t band_rest2(float &a, float &b, uint32_t rounded) {
    a -= __uint_as_float(rounded << 16);
    b -= __uint_as_float(rounded & 0xffff0000u);
    return pack_bf16(a, b);
}
__device__ __forceinline__ void band_rest(float *v, const uint4 &f, uint4 &rest) {
    rest = make_uint4(band_rest2(v[0], v[1], f.x), band_rest2(v[2], v[3], f.y), band_rest2(v[4], v[5], f.z), band_rest2(v[6], v[7], f.w));
}

// ---- global memory: 8 consecutive elements of a row, zero past D -------------------------------------------------
struct __attribute__((packed, aligned(4))) band_u16x8 { uint32_t x, y, z, w; };
struct __attribute__((packed, aligned(4))) band_f32x4 { float x, y, z, w; };   // (unaligned vector accesses are legal)

template <int MODE> __device__ __forceinline__ uint4 band_load8(const bf16_t *row, int col, int D) {
    if constexpr (MODE == 0) return col < D ? *reinterpret_cast<const uint4 *>(row + col) : make_uint4(0u, 0u, 0u, 0u);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (MODE == 1) {
            w[i] = col + 2 * i < D ? *reinterpret_cast<const uint32_t *>(row + col + 2 * i) : 0u;
        } else {
            const uint32_t lo = col + 2 * i < D ? row[col + 2 * i] : 0u, hi = col + 2 * i + 1 < D ? row[col + 2 * i + 1] : 0u;
            w[i] = lo | (hi << 16);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int MODE> __device__ __forceinline__ band_t<float>::frag band_load8(const float *row, int col, int D) {
    band_t<float>::frag f;
    if constexpr (MODE == 0) {
        f.lo = col < D ? *reinterpret_cast<const float4 *>(row + col) : f4zero();
        f.hi = col + 4 < D ? *reinterpret_cast<const float4 *>(row + col + 4) : f4zero();
        return f;
    }
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < D ? row[col + i] : 0.f;
    f.lo = make_float4(v[0], v[1], v[2], v[3]);
    f.hi = make_float4(v[4], v[5], v[6], v[7]);
    return f;
}
// the piece at p, all 8 elements inside the row
__device__ __forceinline__ uint4 band_piece(const bf16_t *p) {
    const band_u16x8 t = *reinterpret_cast<const band_u16x8 *>(p);
    return make_uint4(t.x, t.y, t.z, t.w);
}
__device__ __forceinline__ band_t<float>::frag band_piece(const float *p) {
    const band_f32x4 a = *reinterpret_cast<const band_f32x4 *>(p), b = *reinterpret_cast<const band_f32x4 *>(p + 4);
    band_t<float>::frag f;
    f.lo = make_float4(a.x, a.y, a.z, a.w);
    f.hi = make_float4(b.x, b.y, b.z, b.w);
    return f;
}
__device__ __forceinline__ void band_clear(uint4 &f) { f = make_uint4(0u, 0u, 0u, 0u); }
__device__ __forceinline__ void band_clear(band_t<float>::frag &f) { f.lo = f4zero(), f.hi = f4zero(); }

template <int MODE> __device__ __forceinline__ void band_store8(bf16_t *row, int col, const float *v, int D) {
    const uint4 u = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    if constexpr (MODE == 0) {
        if (col < D) *reinterpret_cast<uint4 *>(row + col) = u;
    } else if constexpr (MODE == 1) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + 2 * i < D) *reinterpret_cast<uint32_t *>(row + col + 2 * i) = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < D) row[col + i] = f32_to_bf16(v[i]);
    }
}
template <int MODE> __device__ __forceinline__ void band_store8(float *row, int col, const float *v, int D) {
    if constexpr (MODE == 0) {
        if (col < D) *reinterpret_cast<float4 *>(row + col) = make_float4(v[0], v[1], v[2], v[3]);
        if (col + 4 < D) *reinterpret_cast<float4 *>(row + col + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < D) row[col + i] = v[i];
    }
}

template <typename T> __device__ __forceinline__ const T *band_row(const BandTensor &t, int b, long long l, int h) {
    return static_cast<const T *>(t.p) + b * t.s.b + l * t.s.l + h * t.s.h;
}

// Transposed result tiles (accumulator rows = head-dim columns, lane = row of the tensor): 8 consecutive columns per
// lane by an exchange of the two lane halves, then one store per 16 columns.  All lanes must call it (the exchange);
// `on` says whether this lane's row is written.
template <typename T, int DP, int MODE>
__device__ __forceinline__ void band_store_row(T *row, const f32x16 *acc, float mul, int D, int hh, bool on) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[db][8 * p + i] * mul),
                                                                __float_as_uint(acc[db][8 * p + 4 + i] * mul), false, false);
                v[i] = __uint_as_float(r[0]);
                v[4 + i] = __uint_as_float(r[1]);
            }
            if (on) band_store8<MODE>(row, 32 * db + 16 * p + 8 * hh, v, D);
        }
}

// what the rounding of such a tile's rows left behind, rounded in its turn
template <int DP, int MODE>
__device__ __forceinline__ void band_store_rest(bf16_t *row, const f32x16 *acc, float mul, int D, int hh, bool on) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
        f32x16 left;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float v = acc[db][r] * mul;
            left[r] = v - bf16_to_f32(f32_to_bf16(v));
        }
        band_store_row<bf16_t, 32, MODE>(row + 32 * db, &left, 1.f, D - 32 * db, hh, on);
    }
}

// ---- LDS images of [rows][DP] tiles --------------------------------------------------------------------------------
// bf16: 16-byte slots XORed with a pattern of the row, such that 16 rows' reads of one slot and the transposing reads of
// 4 rows x 32 columns fall on distinct banks; fp32: rows padded by 16 bytes.
template <int DP> __device__ __forceinline__ int band_flip(int row) {
    if constexpr (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return slot_flip<DP>(row);
}
template <typename T, int DP> __device__ __forceinline__ int band_at(int row, int col) {
    if constexpr (sizeof(T) == 2) return row * DP + (((col >> 3) ^ band_flip<DP>(row)) << 3) + (col & 7);
    else return row * (DP + 4) + col;
}
template <int DP> __device__ __forceinline__ void band_put(bf16_t *m, int row, int slot, const uint4 &f) {
    *reinterpret_cast<uint4 *>(m + band_at<bf16_t, DP>(row, 8 * slot)) = f;
}
template <int DP> __device__ __forceinline__ void band_put(float *m, int row, int slot, const band_t<float>::frag &f) {
    float *p = m + band_at<float, DP>(row, 8 * slot);
    *reinterpret_cast<float4 *>(p) = f.lo;
    *reinterpret_cast<float4 *>(p + 4) = f.hi;
}
// rows of the image as the first operand: row row0 + lane % 32, columns 16 c + 8 (lane / 32) ..
template <int DP> __device__ __forceinline__ uint4 band_rows(const bf16_t *m, int row, int c, int hh) {
    return *reinterpret_cast<const uint4 *>(m + band_at<bf16_t, DP>(row, 16 * c + 8 * hh));
}
template <int DP> __device__ __forceinline__ band_t<float>::frag band_rows(const float *m, int row, int c, int hh) {
    const float *p = m + band_at<float, DP>(row, 16 * c + 8 * hh);
    band_t<float>::frag f;
    f.lo = *reinterpret_cast<const float4 *>(p);
    f.hi = *reinterpret_cast<const float4 *>(p + 4);
    return f;
}
// columns of the image as the first operand: column 32 db + lane % 32; element e is row row0 + (e & 3) + 8 (e >> 2) +
// 4 (lane / 32), the rows that registers 8c .. 8c+7 of a 32x32 result hold for row0 = 16 c
template <int DP> __device__ __forceinline__ uint4 band_cols(const bf16_t *m, int row0, int db, int lane) {
    const int row = row0 + 4 * (lane >> 5) + ((lane >> 2) & 3), col = 32 * db + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const uint2 a = lds_read_tr16(m + band_at<bf16_t, DP>(row, col)), b = lds_read_tr16(m + band_at<bf16_t, DP>(row + 8, col));
    return make_uint4(a.x, a.y, b.x, b.y);
}
template <int DP> __device__ __forceinline__ band_t<float>::frag band_cols(const float *m, int row0, int db, int lane) {
    const float *p = m + band_at<float, DP>(row0 + 4 * (lane >> 5), 32 * db + (lane & 31));
    constexpr int S = DP + 4;
    band_t<float>::frag f;
    f.lo = make_float4(p[0], p[S], p[2 * S], p[3 * S]);
    f.hi = make_float4(p[8 * S], p[9 * S], p[10 * S], p[11 * S]);
    return f;
}

// ---- staging of 64-row tiles by the whole workgroup (256 threads) ------------------------------------------------
// Tiles of one slice (a head of one sequence, rows `ld` apart) and their LDS images.  Rows behind the last one read as copies of
// it: what they hold is masked, and nothing past the sequence is touched.  DIRECT (bf16, modes 0 and 1): fetch()
// starts the copy straight into the image, band_landed() waits for it; the columns past D repeat the row's last piece
// (the queries are zero in those columns of K, and those columns of V add to columns of the result that are not stored).
// The copies are written in assembly because the compiler, which cannot tell the images apart, would wait for them in front
// of the first LDS read of any image; m0, which carries their destination, is used by nothing else in these kernels.
// Otherwise fetch() loads registers and put() writes the image; in mode 1 the last piece of a row is the one that ends
// with it, and clear() has to have zeroed the columns past D once.
// What lanes exchange through LDS: neither the barrier nor a wave's in-order LDS accesses are by themselves something that the
// compiler keeps loads and stores on their side of.
__device__ __forceinline__ void band_fence() { asm volatile("" ::: "memory"); }
__device__ __forceinline__ void band_barrier() {
    band_fence();
    lds_barrier();
    band_fence();
}
__device__ __forceinline__ void band_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t band_lds_address(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}
template <typename T, int DP, int MODE> struct BandStage {
    static constexpr int N = DP / 32, SLOTS = DP / 8, STEP = 256 / SLOTS;  // pieces per thread, per row; rows between a thread's pieces
    static constexpr bool DIRECT = MODE <= 1 && sizeof(T) == 2, DWORDS = DIRECT && MODE == 1;
    static constexpr int COPIES = DWORDS ? 4 * N : N, BYTES = DWORDS ? 256 : 1024;  // copy instructions per wave and tile, bytes of each
    long long ld;  // bytes
    uint32_t ld32;
    typename band_t<T>::frag f[DIRECT ? 1 : N];
    static constexpr bool KEPT = DIRECT && COPIES <= 4;  // (more would cost more registers than their computation takes time)
    uint32_t off[KEPT ? COPIES : 1];  // this lane's bytes of each copy, from the tile's first row

    // row and byte within the row of what copy i of this lane fetches: the place in the image follows from the lane, the
    // logical piece there from the image's pattern
    static __device__ __forceinline__ void source(int i, int D, int &r, int &byte) {
        const int lane = threadIdx.x & 63, n = (threadIdx.x >> 6) * COPIES + i;
        if constexpr (DWORDS) {
            const int at = n * 64 + lane, w = at % (DP / 2);
            r = at / (DP / 2);
            byte = 2 * min((((w >> 2) ^ band_flip<DP>(r)) << 3) + 2 * (w & 3), D - 2);
        } else {
            r = n * (64 / SLOTS) + lane / SLOTS;
            byte = 16 * min((lane % SLOTS) ^ band_flip<DP>(r), D / 8 - 1);
        }
    }
    __device__ __forceinline__ void init(long long row, int D) {
        ld = row * (long long)sizeof(T);
        ld32 = (uint32_t)ld;
        if constexpr (KEPT) {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                int r, byte;
                source(i, D, r, byte);
                off[i] = (uint32_t)r * ld32 + byte;
            }
        }
    }
    // the 64 rows at `tile`, of which rows 0 .. last exist
    __device__ __forceinline__ void fetch(const char *tile, int last, int D, T *image) {
        if constexpr (DIRECT) {
            const uint32_t to = __builtin_amdgcn_readfirstlane(band_lds_address(image) + (threadIdx.x >> 6) * (COPIES * BYTES));
            const uint64_t at = reinterpret_cast<uint64_t>(tile);  // (the same in all lanes, which the compiler does not always see)
            // (readfirstlane returns an int: without the casts a low half with its top bit set would fill the high half)
            const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32));
            const uint64_t rows = ((uint64_t)hi << 32) | lo;
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                uint32_t from = off[KEPT ? i : 0];
                if (!KEPT || last < BAND_TILE - 1) {
                    int r, byte;
                    source(i, D, r, byte);
                    from = (uint32_t)min(r, last) * ld32 + byte;
                }
                if constexpr (DWORDS)
                    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to + i * BYTES), "v"(from), "s"(rows) : "memory");
                else
                    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to + i * BYTES), "v"(from), "s"(rows) : "memory");
            }
        } else {
            const int r0 = threadIdx.x / SLOTS, col = 8 * (threadIdx.x % SLOTS);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = min(r0 + i * STEP, last);
                if constexpr (MODE == 2) {
                    f[i] = band_load8<2>(reinterpret_cast<const T *>(tile + (long long)r * ld), col, D);
                } else {
                    const T *p = reinterpret_cast<const T *>(tile + (uint32_t)r * ld32);
                    if constexpr (MODE == 1) f[i] = band_piece(p + min(col, D - 8));
                    else f[i] = band_load8<0>(p, col, D);
                }
            }
        }
    }
    __device__ __forceinline__ void put(T *image, int D) const {
        if constexpr (!DIRECT) {
            const int r0 = threadIdx.x / SLOTS, slot = threadIdx.x % SLOTS;
            if (MODE != 1 || 8 * slot + 8 <= D) {
#pragma unroll
                for (int i = 0; i < N; ++i) band_put<DP>(image, r0 + i * STEP, slot, f[i]);
            } else if (8 * slot < D) {
                // the piece that ends with the row lies across two of the image's: one element at a time (those of the
                // piece before it come a second time, with the values it wrote)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    T e[8];
                    *reinterpret_cast<typename band_t<T>::frag *>(e) = f[i];
#pragma unroll
                    for (int k = 0; k < 8; ++k) image[band_at<T, DP>(r0 + i * STEP, D - 8 + k)] = e[k];
                }
            }
        }
    }
    // zeros in the columns past D of `rows` rows of images, by the whole workgroup; a barrier is the caller's
    static __device__ __forceinline__ void clear(T *image, int rows, int D) {
        if constexpr (MODE == 1 && !DIRECT)
            for (int e = threadIdx.x; e < rows * (DP - D); e += 256) image[band_at<T, DP>(e / (DP - D), D + e % (DP - D))] = (T)0;
    }
};

// ---- lengths, tiles -----------------------------------------------------------------------------------------------------
struct BandSeq {
    int kn, qn, off;  // keys, query rows, position of row 0
};
__device__ __forceinline__ BandSeq band_seq(const BandArgs &a, int b) {
    BandSeq s;
    s.kn = a.k_lens ? min(max(a.k_lens[b], 0), a.Lk) : a.Lk;
    s.qn = a.q_lens ? min(max(a.q_lens[b], 0), a.Lq) : a.Lq;
    s.off = s.kn - s.qn;
    return s;
}
// Tiles of `size` keys that rows at positions p_lo..p_hi need: the sinks' tiles, then the window's without a gap.
struct BandTiles {
    int n_sink, first, count;
    __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : first + i - n_sink; }
};
template <int SIZE> __device__ __forceinline__ BandTiles band_tiles(const BandArgs &a, int kn, int p_lo, int p_hi) {
    BandTiles t;
    const int j_hi = min(kn - 1, p_hi + a.right);
    t.n_sink = t.first = t.count = 0;
    if (j_hi < 0 || p_hi < p_lo) return t;
    t.first = max(0, p_lo - a.left) / SIZE;
    const int last = j_hi / SIZE;
    if (last < t.first) return t;
    t.n_sink = min((a.sinks + SIZE - 1) / SIZE, t.first);
    t.count = t.n_sink + last - t.first + 1;
    return t;
}

// the walk over them: first key and its rows' address in a slice, without a multiplication per tile
struct BandWalk {
    const char *base, *p;
    long long step, jump;
    __device__ __forceinline__ void init(const void *slice, long long ld_bytes, int size, const BandTiles &t) {
        base = static_cast<const char *>(slice);
        step = ld_bytes * size;
        jump = step * t.first;
        p = t.n_sink ? base : base + jump;
    }
    __device__ __forceinline__ void next(int i, const BandTiles &t) { p = i == t.n_sink ? base + jump : p + step; }  // to tile i
};

// the bias of one head by distance, times log2(e), in LDS: entry e is distance sign * (e - M - BAND_MARGIN), clipped
__device__ __forceinline__ float band_bias_at(const BandArgs &a, int head, int rel) {
    const int m = min(max(rel, -a.M), a.M) + a.M;
    const int bucket = min(max(a.buckets[m], 0), a.n_buckets - 1);
    const float v = a.table[(size_t)bucket * a.Hq + head];
    // (finite entries stay finite: the type's lowest value masks like any other large negative one)
    return __builtin_isinf(v) ? v : v != v ? v : fminf(fmaxf(v * LOG2E, -FLT_MAX), FLT_MAX);
}
// A finite bias, however low, only ever weighs a key against others.  So that a row of which nothing else is left still gets
// the softmax of its scores, a reference (the row's maximum, or near it) that is far from zero is taken from the bias before
// the score comes to it, in the backward too, which for the same reason finds it apart from log2(l).  A moderate one
// is taken from the sum, as rounded: the exponent of a row's only key is then zero, and its result the key's value.
__device__ __forceinline__ bool band_remote(float top) { return __any(fabsf(top) > 1024.f); }
// log2(e) * logit - top
__device__ __forceinline__ float band_exponent(float s, float c, float bias, float top, bool remote) {
    return remote ? __builtin_fmaf(s, c, bias - top) : __builtin_fmaf(s, c, bias) - top;
}
// What is left of a score beside a reference that swallowed it (beyond 2^31 its rounding alone is a hundred) may overflow, or
// leave nothing of any key.  Rows whose denominator comes out of the middle of fp32's range are done again by band_careful.
// (The reference's own key gives 2^0 else, so that nothing is below and only what climbs above; rows without a key: m = -inf.)
__device__ __forceinline__ bool band_strayed(float m, float l) { return m != -INFINITY && !(l >= 0x1p-64f && l <= 0x1p100f); }
// what a row leaves for its backward: top + log2(l), or with a bias the two apart; l is the sum of 2^(exponent - lift)
__device__ __forceinline__ void band_keep(const BandArgs &a, size_t at, bool off, float top, float lift, float l) {
    const float log_l = off ? INFINITY : __builtin_amdgcn_logf(l) + lift;
    if (a.top) a.top[at] = off ? 0.f : top;
    const float sum = top + log_l, part = sum - top;
    a.lse[at] = a.top || off ? log_l : sum;
    if (a.lse_rest) a.lse_rest[at] = off ? 0.f : (top - (sum - part)) + (log_l - part);
}
// Without a bias an exponent of the backward is one multiply-add, scale * s - lse: the product is not rounded, as the reference
// was, and lse is rounded once more, which puts probabilities off by 2^-25 of the logits' size.  For fp32 calls, whose matrix
// instructions leave the time, the product is rounded first and what the rounding of lse left is taken off as well: a row's
// only key then has the probability 1, whatever its score.  (For bf16 the size has to pass 2^16 before it is seen, and the
// same costs dk and dv 15 %.)
template <typename T> constexpr bool band_whole(bool bias) { return !bias && sizeof(T) == 4; }
__device__ __forceinline__ void band_stage_bias(const BandArgs &a, int head, int sign, float *dst, int threads) {
    const int n = 2 * (a.M + BAND_MARGIN) + 1;
    for (int e = threadIdx.x; e < n; e += threads) dst[e] = band_bias_at(a, head, sign * (e - a.M - BAND_MARGIN));
}
// Which keys of a tile a row sees: key base + off is visible when off <= hi and (off >= lo or off < first).  Decided with
// selects on scalars throughout: branches that write single elements of the 16-wide accumulators were seen to be
// compiled wrongly (an element's store was lost).
struct BandMask {
    int hi, lo, first;
    __device__ __forceinline__ bool sees(int off) const { return (off <= hi) & ((off >= lo) | (off < first)); }
};
// one row at position p against keys from `base` on
__device__ __forceinline__ BandMask band_row_mask(const BandArgs &a, int p, int kn, int base) {
    return {min(kn - 1, p + a.right) - base, p - a.left - base, a.sinks - base};
}

// A 64-key or 32-key tile against the 32 rows of a wave, decided by a handful of scalars made once per wave
template <int SIZE> struct BandEdges {
    int none_hi, none_lo, hi_ok, lo_ok, sinks;
    __device__ __forceinline__ void init(const BandArgs &a, int kn, int w_lo, int w_hi, bool on) {
        none_hi = on ? min(kn - 1, w_hi + a.right) : -1;   // j0 beyond: no key of the tile is seen
        none_lo = w_lo - a.left - (SIZE - 1);              // j0 before, and no sink: likewise
        hi_ok = min(kn - SIZE, w_lo + a.right - (SIZE - 1));  // j0 up to here: no row's right end cuts the tile
        lo_ok = w_hi - a.left;                             // j0 from here: no row's left end does
        sinks = a.sinks;
    }
    __device__ __forceinline__ bool none(int j0) const { return j0 > none_hi || (j0 < none_lo && j0 >= sinks); }
    __device__ __forceinline__ bool cut_hi(int j0) const { return j0 > hi_ok; }
    __device__ __forceinline__ bool cut_lo(int j0) const { return j0 < lo_ok && j0 + SIZE > sinks; }
};

// The query rows of a workgroup (forward, dQ).  Made twice, before the loop and after it, from the arguments: what only
// the end needs does not have to be kept in scalar registers through the loop, which were spilled for it.
// Which piece of work a workgroup takes, of `per` pieces for each (sequence, key head): hardware deals workgroups to the
// eight XCDs in turn, and those of one key head belong on one of them, whose L2 then holds the keys once.  Key heads are dealt
// in turn as well, so that sequences of unequal lengths, or empty ones, spread over all XCDs (a run of neighbours for
// each XCD: dq 65 us for 41, dk and dv 63 for 52, three sequences of 0, 680 and 1021 tokens, fp32, 6 heads of 32); what is left
// of them after whole rounds of eight is cut into eight runs.
__device__ __forceinline__ int band_piece_of(int block, int blocks, int per) {
    const int whole = blocks / per / 8 * 8 * per;
    if (block >= whole) return whole + xcd_remap(block - whole, blocks - whole);
    const int at = block >> 3, round = at / per;
    return (round * 8 + (block & 7)) * per + (at - round * per);
}

struct BandPlace {
    int b, h, hk, i_lo, i0, i;
    BandSeq sq;
    BandTiles tiles;
    // `rows` of a workgroup: 128, or 64 where two waves share 32
    __device__ __forceinline__ BandPlace(const BandArgs &a, int block, int blocks, int rows = BAND_ROWS) {
        const int nqb = (a.Lq + rows - 1) / rows;
        const int idx = band_piece_of(block, blocks, nqb * a.G);
        const int g = idx % a.G, rest = idx / a.G;
        const int qb = nqb - 1 - rest % nqb, bh = rest / nqb;  // (the last rows of a causal call have the most to do: first)
        hk = bh % a.Hkv, b = bh / a.Hkv, h = hk * a.G + g;
        i_lo = qb * rows;
        i0 = i_lo + 32 * (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & (rows / 32 - 1));
        i = i0 + (threadIdx.x & 31);
        sq = band_seq(a, b);
        tiles = band_tiles<BAND_TILE>(a, sq.kn, sq.off + i_lo, sq.off + min(i_lo + rows, sq.qn) - 1);
    }
};

// Non-finite values in keys or values that a row does not see must not reach it: a probability of zero times an
// infinity is not zero.  The tiles' products cannot tell, so a wave that ends with a non-finite result (seen nowhere
// else) does its tiles again key by key, touching only what each row sees.  So does one whose sums strayed (see there): with a
// bias the reference has a second part here, `lift`, the largest exponent that is left beside m.  Lane = row as in the kernels;
// m, l and acc as they leave them (l of one lane half).
template <typename T, int DP, bool BIAS, int SIZE>
__device__ __forceinline__ void band_careful(const BandArgs &a, const T *qrow, const T *kbase, const T *vbase, int head, int p,
                                             bool on, int kn, const BandTiles &tiles, int t_begin, int t_end, int t_step, int hh,
                                             float &m, float &lift, float &l, f32x16 *acc) {
    m = -INFINITY;
    lift = l = 0.f;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) acc[db] = band_zero();
    for (int t = t_begin; t < t_end; t += t_step)
        for (int j = tiles.at(t) * SIZE; j < min(tiles.at(t) * SIZE + SIZE, kn); ++j) {
            const bool vis = on & band_row_mask(a, p, kn, j).sees(0);
            if (!__any(vis)) continue;
            const T *kr = kbase + (long long)j * a.k.s.l, *vr = vbase + (long long)j * a.v.s.l;
            float s = 0.f;
            if (vis)
                for (int d = hh; d < a.D; d += 2) s = __builtin_fmaf(io<T>::ld(qrow + d), io<T>::ld(kr + d), s);
            s += __shfl_xor(s, 32, 64);
            const float bias = BIAS && vis ? band_bias_at(a, head, j - p) : 0.f, x = __builtin_fmaf(s, a.c, bias);
            const bool counts = vis && x != -INFINITY;
            // (not a number: the row has a reference all the same, so that its sums count, and show it)
            const float mn = vis ? fmaxf(m, x != x ? 0.f : x) : m, left = band_exponent(s, a.c, bias, mn, BIAS && band_remote(vis ? mn : 0.f));
            // (what the sums so far are worth beside mn, as an exponent; nothing at first)
            const float before = m == -INFINITY ? -INFINITY : mn == m ? lift : lift + (m - mn);
            const float ln = BIAS && counts ? fmaxf(before, left) : BIAS && m != -INFINITY ? before : 0.f;
            const float alpha = before == ln ? 1.f : __builtin_amdgcn_exp2f(before - ln);
            const float e = counts ? __builtin_amdgcn_exp2f(left - ln) : 0.f;
            m = mn;
            lift = ln;
            l = l * alpha + (hh == 0 ? e : 0.f);
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = 32 * db + rho(r) + 4 * hh;
                    const bool take = vis & (d < a.D);
                    const float v = take ? io<T>::ld(vr + d) : 0.f, sum = __builtin_fmaf(e, v, acc[db][r] * alpha);
                    acc[db][r] = take ? sum : acc[db][r];
                }
        }
}

// floats of a row's share in the split forward: D sums, the reference, the denominator, with a bias the lift
__host__ __device__ __forceinline__ int band_share_floats(const BandArgs &a) { return a.D + (a.table ? 3 : 2); }

// Allows a kernel the LDS of its launch: always as much as any of these launches takes, so that calls of different sizes from
// several threads leave each other's limit alone.
constexpr size_t BAND_LDS = 128 * 1024;
template <typename K> int band_allow_lds(const char *who, K kern, size_t lds) {
    if (lds <= 65536) return DSW_OK;
    if (lds > BAND_LDS) return fail(DSW_EUNSUPPORTED, "%s: %zu bytes of LDS", who, lds);
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)BAND_LDS);
    return e == hipSuccess ? DSW_OK : fail(DSW_ELAUNCH, "%s: %zu bytes of LDS: %s", who, lds, hipGetErrorString(e));
}
int band_make_args(const char *who, const dsw_band_desc *d, BandArgs &a);
// fills t and raises `mode` to what the tensor needs
int band_tensor(const char *who, const char *name, const void *p, const dsw_strides *s, int dtype, int D, bool null_ok, BandTensor &t, int &mode);
// likewise a.rest, where the description has it
int band_rest_tensor(const char *who, const dsw_band_desc *d, BandArgs &a, int &mode);
// (T, DP, MODE) for a call
#define DSW_BAND_DISPATCH(dtype, D, mode, T, DP, MODE, ...)                                                           \
    DSW_DISPATCH_DTYPE(dtype, T, {                                                                                      \
        if ((mode) == 2) { constexpr int MODE = 2; DSW_BAND_WIDTHS(D, DP, __VA_ARGS__) }                                \
        else if ((mode) == 1) { constexpr int MODE = 1; DSW_BAND_WIDTHS(D, DP, __VA_ARGS__) }                           \
        else { constexpr int MODE = 0; DSW_BAND_WIDTHS(D, DP, __VA_ARGS__) }                                            \
    })
#define DSW_BAND_WIDTHS(D, DP, ...)                               \
    if ((D) <= 32) { constexpr int DP = 32; __VA_ARGS__; }        \
    else if ((D) <= 64) { constexpr int DP = 64; __VA_ARGS__; }   \
    else { constexpr int DP = 128; __VA_ARGS__; }
// how the dK, dV kernel shares its key blocks out (band_attn_bwd.hip)
struct BandChunks {
    int sink_blocks, sink_chunks, chunks;
    long long shares;  // workgroups that write a share
};
// launches the kernel for few query rows (band_attn_step.hip) and the one that joins its splits
int band_launch_step(BandArgs &a, int dtype, int mode, hipStream_t st);
// whether a call goes there, and how many row blocks and splits it has
bool band_step_plan(const dsw_band_desc &d, int &nrb, int &nsplit);

}  // namespace dsw
