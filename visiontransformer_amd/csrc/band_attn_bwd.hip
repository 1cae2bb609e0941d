// Attention over token sequences, backward (see band_attn.hpp for the mathematics and the register layouts).
//
//   delta_i = dout_i . out_i        P = 2^(x - lse)        dS = P (dout v^T - delta)
//   dq = scale dS k     dk = scale dS^T q     dv = P^T dout     dtable[b, head] = sum of dS over the pairs of bucket b
//
// Two kernels that each own what they write, so that no sum depends on the order in which workgroups run: one over
// row blocks (dq, delta, and the bias gradient by distance), then one over key blocks (dk, dv; the query heads that
// share a key head are walked one after the other and meet in the accumulators).  Both recompute the scores.  Layouts as in
// the forward: the 16 registers of a tile's P and dS are the second operand of the products that follow.
//
// Rounding, for bf16 tensors: P and dS enter their products in bf16 (2^-8 each, as the matrix instructions take them); P is
// divided by the sum of the rounded probabilities of the forward, which may put a row off by as much as one of them; dS itself,
// delta and all sums are fp32.  dq, dk and dv are 2.3e-3 to 2.4e-3 (rms) from 64 bits, of which their own rounding is 1.7e-3.
//
// Neither pipe is full: products (four and three per tile) and the exponentials between them take turns at two waves a SIMD,
// which the accumulators' registers allow.  2 x 4096 tokens, 16 heads on 4 of 64, window 1024, bf16: dk and dv 98 us, 610 TFLOP/s of the
// visible pairs' products, matrix pipe 32 % and vector pipe 43 % busy, and 8 us for their join; dq 74 us, 610 TFLOP/s, 33 and
// 49 %.  With a table's gradient, 2 x 2048 tokens, 8 heads of 64, all visible: dq 70 us (17 and 31 %), dk and dv 61 (27 and 42 %).
#include "band_attn.hpp"

namespace dsw {

// ---- dk, dv: 128 keys of a workgroup, 32 per wave -----------------------------------------------------------------
// A key block's work is its row tiles times the query heads that share the keys.  Blocks of sinks are seen by every row
// behind them, the others by a window's; and where there are few blocks, one workgroup each does not fill the chip.  So a
// block is cut into `chunks` (`sink_chunks`) runs of that work; more than one leave fp32 sums in `shares`, which
// band_attn_join_dkv_kernel adds in their order.
template <typename T, int DP, int MODE, bool BIAS>
__global__ __launch_bounds__(256, (DP == 128 || sizeof(T) == 4 ? 1 : 2)) void band_attn_dkv_kernel(const BandArgs a) {
    constexpr int NB = band_t<T>::nbuf(DP), ELEMS = band_t<T>::template elems<DP>(BAND_TILE), C = DP / 16;
    constexpr bool AHEAD = DP < 128 && (sizeof(T) == 2 || DP == 32);  // registers for LDS reads well ahead of the products that need them
    constexpr bool WHOLE = band_whole<T>(BIAS);
    constexpr int STATS = BIAS ? 4 : WHOLE ? 3 : 2;
    using Stage = BandStage<T, DP, MODE>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T *const lds = reinterpret_cast<T *>(smem);                        // [NB][Q | dO]
    float *const stats = reinterpret_cast<float *>(lds + NB * 2 * ELEMS);  // [NB][-lse - top | delta | top | -lse][64], WHOLE: [-lse | delta | -lse_rest]
    float *const bias = stats + NB * STATS * BAND_TILE;

    const int nkb = (a.Lk + BAND_ROWS - 1) / BAND_ROWS, units = a.sink_blocks * a.sink_chunks + (nkb - a.sink_blocks) * a.chunks;
    const int idx = band_piece_of(blockIdx.x, gridDim.x, units);
    const int bh = idx / units, unit = idx - bh * units, hk = bh % a.Hkv, b = bh / a.Hkv;
    const bool of_sinks = unit < a.sink_blocks * a.sink_chunks;
    const int nc = of_sinks ? a.sink_chunks : a.chunks, left_over = unit - (of_sinks ? 0 : a.sink_blocks * a.sink_chunks);
    const int kb = (of_sinks ? 0 : a.sink_blocks) + left_over / nc, chunk = left_over % nc;
    const int lane = threadIdx.x & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const BandSeq sq = band_seq(a, b);
    const int k_lo = kb * BAND_ROWS, k_hi = min(k_lo + BAND_ROWS, sq.kn) - 1;
    const int j_lo = k_lo + 32 * wave, j_hi = j_lo + 31, j = j_lo + l31;
    const bool key_on = j < sq.kn;

    // query rows that see a key of this block
    const int first = max(0, k_lo - a.right - sq.off) / BAND_TILE;
    const int last_row = k_lo < a.sinks ? sq.qn - 1 : min(sq.qn - 1, k_hi + a.left - sq.off);
    const int n_tiles = k_lo < sq.kn && last_row >= 0 ? max(0, last_row / BAND_TILE - first + 1) : 0;
    // this chunk's steps: the tiles of the first head, of the second, ...
    const int share = (n_tiles * a.G + nc - 1) / nc, begin = min(chunk * share, n_tiles * a.G), end = min(begin + share, n_tiles * a.G);

    typename band_t<T>::frag kf[C], vf[C];
    const T *const krow = band_row<T>(a.k, b, j, hk), *const vrow = band_row<T>(a.v, b, j, hk);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (key_on) {
            kf[c] = band_load8<MODE>(krow, 16 * c + 8 * hh, a.D);
            vf[c] = band_load8<MODE>(vrow, 16 * c + 8 * hh, a.D);
        } else {
            band_clear(kf[c]);
            band_clear(vf[c]);
        }
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) dk[db] = dv[db] = band_zero();

    Stage qs, gs;
    float st = 0.f;
    if (MODE == 1 && !Stage::DIRECT && a.D < DP) {
        Stage::clear(lds, NB * 2 * BAND_TILE, a.D);
        __syncthreads();
    }
    qs.init(a.q.s.l, a.D);
    gs.init(a.dout.s.l, a.D);
    auto fetch = [&](int tile, int h, T *image) {
        const int i0 = tile * BAND_TILE;
        if (threadIdx.x < STATS * BAND_TILE) {
            const int i = i0 + (threadIdx.x & (BAND_TILE - 1));
            const int stat = threadIdx.x / BAND_TILE;
            const size_t at = ((size_t)b * a.Hq + h) * a.Lq + min(i, sq.qn - 1);
            if (WHOLE && stat == 2) {
                st = a.lse_rest ? -a.lse_rest[at] : 0.f;
            } else {
                st = (stat == 1 ? a.delta : stat == 2 ? a.top : a.lse)[at];
                if (BIAS && stat == 0) st += a.top[at];
                if (stat == 0 || stat == 3) st = i < sq.qn ? -st : -INFINITY;
            }
        }
        qs.fetch(reinterpret_cast<const char *>(band_row<T>(a.q, b, i0, h)), sq.qn - 1 - i0, a.D, image);
        gs.fetch(reinterpret_cast<const char *>(band_row<T>(a.dout, b, i0, h)), sq.qn - 1 - i0, a.D, image + ELEMS);
    };
    int g = n_tiles ? begin / n_tiles : 0, tile = first + begin - g * n_tiles;
    if (begin < end) fetch(tile, hk * a.G + g, lds);
    bool new_head = true;
    for (int step = begin; step < end; ++step) {
        T *const Q = lds + (NB == 2 ? ((step - begin) & 1) : 0) * 2 * ELEMS, *const G = Q + ELEMS;
        float *const S = stats + (NB == 2 ? ((step - begin) & 1) : 0) * STATS * BAND_TILE;
        if constexpr (NB == 1) band_barrier();
        if constexpr (BIAS) {
            if (new_head) {
                band_barrier();  // the last head's readers are done
                band_stage_bias(a, hk * a.G + g, -1, bias, 256);
            }
        }
        if constexpr (Stage::DIRECT) {
            band_landed();
        } else {
            qs.put(Q, a.D);
            gs.put(G, a.D);
        }
        if (threadIdx.x < STATS * BAND_TILE) S[threadIdx.x] = st;
        if constexpr (Stage::DIRECT) band_barrier();
        const int i0 = tile * BAND_TILE;
        new_head = tile + 1 == first + n_tiles;
        tile = new_head ? first : tile + 1;
        g += new_head;
        if (step + 1 < end) fetch(tile, hk * a.G + g, lds + (NB == 2 ? ((step + 1 - begin) & 1) : 0) * 2 * ELEMS);
        if constexpr (!Stage::DIRECT) band_barrier();
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
            const int r0 = i0 + 32 * u, p_lo = sq.off + r0, p_hi = sq.off + min(r0 + 31, sq.qn - 1);
            if (r0 >= sq.qn || j_lo >= sq.kn || j_lo > p_hi + a.right || (j_hi < p_lo - a.left && j_lo >= a.sinks)) continue;
            const bool full = j_hi < sq.kn && j_hi <= p_lo + a.right && (j_lo >= p_hi - a.left || j_hi < a.sinks);
            f32x16 s = band_zero(), dp = band_zero();
            float nl[16], del[16];
            {
                typename band_t<T>::frag qf[C], gf[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    qf[c] = band_rows<DP>(Q, 32 * u + l31, c, hh);
                    gf[c] = band_rows<DP>(G, 32 * u + l31, c, hh);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    *reinterpret_cast<float4 *>(nl + 4 * k) = *reinterpret_cast<const float4 *>(S + 32 * u + 8 * k + 4 * hh);
                    *reinterpret_cast<float4 *>(del + 4 * k) = *reinterpret_cast<const float4 *>(S + BAND_TILE + 32 * u + 8 * k + 4 * hh);
                }
                if (sizeof(T) == 2 || DP == 32) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    s = band_mma(qf[c], kf[c], s);
                    dp = band_mma(gf[c], vf[c], dp);
                }
            }
            typename band_t<T>::frag gc[2][DP / 32], qc[2][DP / 32];
            auto columns_ahead = [&]() {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) {
                        gc[k][db] = band_cols<DP>(G, 32 * u + 16 * k, db, lane);
                        qc[k][db] = band_cols<DP>(Q, 32 * u + 16 * k, db, lane);
                    }
            };
            if (AHEAD && !BIAS) columns_ahead();
            float cs = a.c;
            if constexpr (WHOLE) {
                cs = 1.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = s[r] * a.c + nl[r];
                    nl[r] = S[2 * BAND_TILE + 32 * u + 4 * hh + rho(r)];
                }
            }
            if constexpr (BIAS) {
                const bool near = j_lo - p_hi < a.M && j_hi - p_lo > -a.M;
                if (band_remote(S[2 * BAND_TILE + 32 * u + l31])) {
                    // top and lse apart, and one row after the other: this is rare, and must not cost registers
                    cs = 1.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int row = 32 * u + 4 * hh + rho(r), e = near ? p_lo + 4 * hh + rho(r) - j + a.M + BAND_MARGIN : j_lo > p_hi ? 0 : 2 * (a.M + BAND_MARGIN);
                        s[r] = band_exponent(s[r], a.c, bias[e], S[2 * BAND_TILE + row], true);
                        nl[r] = S[3 * BAND_TILE + row];
                        band_fence();
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else if (near) {
                    const float *br = bias + (p_lo + 4 * hh - j + a.M + BAND_MARGIN);
#pragma unroll
                    for (int r = 0; r < 16; ++r) nl[r] += br[rho(r)];
                } else {
                    const float bu = bias[j_lo > p_hi ? 0 : 2 * (a.M + BAND_MARGIN)];
#pragma unroll
                    for (int r = 0; r < 16; ++r) nl[r] += bu;
                }
            }
            if (AHEAD && BIAS) columns_ahead();  // (behind the bias, which has no registers to spare)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], cs, nl[r]));
            if (!full) {
                // the mask from the key's side: position p sees key j when p >= j - right and (p <= j + left or j < sinks)
                const int p_min = key_on ? j - a.right - p_lo - 4 * hh : BAND_FAR, p_max = j < a.sinks ? BAND_FAR : j + a.left - p_lo - 4 * hh;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = (int)(rho(r) >= p_min) & (int)(rho(r) <= p_max) ? s[r] : 0.f;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = s[r] * (dp[r] - del[r]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                typename band_t<T>::frag pf, sf;
                band_pack(s, k, pf);
                band_pack(dp, k, sf);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    if (!AHEAD) {
                        gc[k][db] = band_cols<DP>(G, 32 * u + 16 * k, db, lane);
                        qc[k][db] = band_cols<DP>(Q, 32 * u + 16 * k, db, lane);
                    }
                    dv[db] = band_mma(gc[k][db], pf, dv[db]);
                    dk[db] = band_mma(qc[k][db], sf, dk[db]);
                }
            }
        }
    }
    // (keys behind the sequence: their P and dS are zero, and so are these rows)
    if (nc == 1) {
        const bool store = j < a.Lk;
        band_store_row<T, DP, MODE>(const_cast<T *>(band_row<T>(a.dk, b, j, hk)), dk, a.scale, a.D, hh, store);
        band_store_row<T, DP, MODE>(const_cast<T *>(band_row<T>(a.dv, b, j, hk)), dv, 1.f, a.D, hh, store);
    } else {
        const int per = a.chunks > 1 ? units : a.sink_blocks * a.sink_chunks;  // shares of one (sequence, key head)
        float *const at = a.shares + (((size_t)bh * per + unit) * 2 * BAND_ROWS + 32 * wave + l31) * a.D;
        // (fp32 rows of D: 16-byte pieces fit where D is a multiple of 4, as in mode 0)
        band_store_row<float, DP, MODE>(at, dk, 1.f, a.D, hh, true);
        band_store_row<float, DP, MODE>(at + (size_t)BAND_ROWS * a.D, dv, 1.f, a.D, hh, true);
    }
}

// V elements of a row of dk or dv per thread (4 where every row is a whole number of them): the sum of the block's shares, in
// their order.  2 * 128 * D elements per block, D / V workgroups.
template <typename T, int V> __global__ __launch_bounds__(256) void band_attn_join_dkv_kernel(const BandArgs a) {
    const int nkb = (a.Lk + BAND_ROWS - 1) / BAND_ROWS, n_sink = a.sink_blocks * a.sink_chunks;
    const int blocks = a.chunks > 1 ? nkb : a.sink_blocks, per = a.chunks > 1 ? n_sink + (nkb - a.sink_blocks) * a.chunks : n_sink;
    const int wgs = a.D / V, block = blockIdx.x / wgs, bh = block / blocks, kb = block - bh * blocks, hk = bh % a.Hkv, b = bh / a.Hkv;
    const int nc = kb < a.sink_blocks ? a.sink_chunks : a.chunks;
    const int unit = kb < a.sink_blocks ? kb * a.sink_chunks : n_sink + (kb - a.sink_blocks) * a.chunks;
    const int size = BAND_ROWS * a.D, e = ((blockIdx.x - block * wgs) * 256 + threadIdx.x) * V;
    const int which = e >= size, row = (e - which * size) / a.D, d = e - which * size - row * a.D, j = kb * BAND_ROWS + row;
    if (j >= a.Lk) return;
    const float *src = a.shares + ((size_t)bh * per + unit) * 2 * size + e;
    const BandTensor &t = which ? a.dv : a.dk;
    T *dst = const_cast<T *>(band_row<T>(t, b, j, hk)) + d;
    const float mul = which ? 1.f : a.scale;
    if constexpr (V == 4) {
        float4 v = f4zero();
#pragma unroll 4
        for (int c = 0; c < nc; ++c) v = v + *reinterpret_cast<const float4 *>(src + (size_t)c * 2 * size);
        io<T>::st4(dst, v * mul);
    } else {
        float v = 0.f;
        for (int c = 0; c < nc; ++c) v += src[(size_t)c * 2 * size];
        io<T>::st(dst, v * mul);
    }
}

// Two workgroups a CU are wanted (one for wide heads, whose registers allow no more); a run of the work is at least 8
// steps long, so that its share does not cost more than it brings.  In fp32, whose products take 16 times as long, runs of 2
// steps pay, and so does a finer cut (4 a CU: 63 us for 68 for 3 x 1021 tokens, 6 heads of 32).  A block of
// sinks, which every row sees, is cut into runs as long as the others' ones, or, where that would make more shares than balance
// needs, a quarter of what each resident workgroup has to do in all, a thousand or two of them (4 x 32768 tokens, 16 heads of
// 128, window 256: without that the workspace was 520 MiB with 4 sinks and 16 GiB with 4096, for 8 MiB with none).
static BandChunks band_chunks(const BandArgs &a, int dtype) {
    BandChunks c = {0, 1, 1, 0};
    const long long nkb = (a.Lk + BAND_ROWS - 1) / BAND_ROWS, heads = (long long)a.B * a.Hkv, tiles = (a.Lq + BAND_TILE - 1) / BAND_TILE;
    if (nkb == 0 || heads == 0 || tiles == 0 || a.G == 0) return c;  // (nothing, or zeros, to write)
    const long long window = (long long)a.left + a.right + BAND_ROWS, reach = window >= a.Lq ? tiles : window / BAND_TILE + 2;
    const long long normal = (reach < tiles ? reach : tiles) * a.G;  // steps of a block in the middle
    const long long want = dtype == DSW_F32 ? 1024 : a.D > 64 ? 256 : 512, n = (want + heads * nkb - 1) / (heads * nkb), most = normal / (dtype == DSW_F32 ? 2 : 8);
    c.chunks = (int)(n < most ? n : most);
    if (c.chunks < 1) c.chunks = 1;
    if (c.chunks > 64) c.chunks = 64;
    const long long sink_blocks = a.sinks > 0 && normal < tiles * a.G ? (a.sinks + BAND_ROWS - 1) / BAND_ROWS : 0;
    c.sink_blocks = (int)(sink_blocks < nkb ? sink_blocks : nkb);
    const long long run = (normal + c.chunks - 1) / c.chunks, all = heads * (c.sink_blocks * tiles * a.G + (nkb - c.sink_blocks) * normal);
    const long long resident = dtype == DSW_F32 || a.D > 64 ? 256 : 512, part = all / (4 * resident);
    const long long len = run > part ? run : part, k = (tiles * a.G + len - 1) / len;
    c.sink_chunks = c.sink_blocks ? (int)(k < 1024 ? k : 1024) : 1;
    c.shares = heads * ((c.sink_chunks > 1 ? (long long)c.sink_blocks * c.sink_chunks : 0));
    if (c.chunks > 1) c.shares = heads * ((long long)c.sink_blocks * c.sink_chunks + (nkb - c.sink_blocks) * c.chunks);
    return c;
}

// ---- dq: 32 rows per wave; delta, which the other kernel reads; bias gradient by distance ---------------------------
// Four waves of 32 rows each where that fills the chip.  SPLIT, for short calls: 64 rows, and two waves on each 32 that take
// the first and the second half of every key tile and add their sums at the end.
template <typename T, int DP, int MODE, bool BIAS, bool DTABLE, bool SPLIT>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DP == 128 ? 1 : 2)) void band_attn_dq_kernel(const BandArgs a) {
    constexpr int NB = band_t<T>::nbuf(DP), ELEMS = band_t<T>::template elems<DP>(BAND_TILE), C = DP / 16;
    constexpr bool AHEAD = DP < 128 && (sizeof(T) == 2 || DP == 32);  // registers for LDS reads well ahead of the products that need them
    constexpr int ROWS = SPLIT ? BAND_ROWS / 2 : BAND_ROWS;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T *const lds = reinterpret_cast<T *>(smem);  // [NB][K | V]
    float *const bias = reinterpret_cast<float *>(lds + NB * 2 * ELEMS);
    const int BL = 2 * (a.M + BAND_MARGIN) + 1;
    // (a table's gradient only) dS of a tile by distance, [4 waves][32 rows][64], and what each wave summed, [4][BL]
    float *const slant = bias + ((BL + 3) & ~3), *const sums = slant + 4 * 32 * 64;

    const int lane = threadIdx.x & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const BandPlace at(a, blockIdx.x, gridDim.x, ROWS);
    const BandSeq &sq = at.sq;
    const BandTiles &tiles = at.tiles;
    const int b = at.b, h = at.h, i = at.i;
    const bool row_on = i < sq.qn;
    const int p = sq.off + i, w_lo = sq.off + at.i0, w_hi = sq.off + min(at.i0 + 31, sq.qn - 1);
    BandEdges<32> edges;
    edges.init(a, sq.kn, w_lo, w_hi, at.i0 < sq.qn);
    const int key_hi = min(sq.kn - 1, p + a.right), key_lo = p - a.left;
    const float scale = a.c;
    const int D = a.D, M = a.M;

    if constexpr (BIAS) band_stage_bias(a, h, 1, bias, 256);
    if constexpr (DTABLE) {
        for (int e = threadIdx.x; e < 4 * (32 * 64 + BL); e += 256) slant[e] = 0.f;  // (before the first tile's barrier)
    }
    typename band_t<T>::frag qf[C], gf[C];
    const T *const qrow = band_row<T>(a.q, b, i, h), *const grow = band_row<T>(a.dout, b, i, h);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (row_on) {
            qf[c] = band_load8<MODE>(qrow, 16 * c + 8 * hh, D);
            gf[c] = band_load8<MODE>(grow, 16 * c + 8 * hh, D);
        } else {
            band_clear(qf[c]);
            band_clear(gf[c]);
        }
    }
    const size_t stat = ((size_t)b * a.Hq + h) * a.Lq + i;
    const float nl = row_on ? -a.lse[stat] : -INFINITY, top = BIAS && row_on ? a.top[stat] : 0.f;
    const bool remote = BIAS && band_remote(top);
    constexpr bool WHOLE = band_whole<T>(BIAS);
    const float low = WHOLE && row_on && a.lse_rest ? -a.lse_rest[stat] : 0.f;
    // delta = dout . out, from the result before its rounding where that was kept (whole, in three parts of 8 bits, or as what the
    // rounding left behind: with the rounded result alone dq and dk of a row of one dominant key were mostly its error).  It is the
    // diagonal of a product formed like dout v^T below: for a row that sees a single key, whose result is that key's value,
    // the two are then the same number and dS is exactly zero.
    float del = 0.f;
    {
        f32x16 d = band_zero();
        const T *const orow = band_row<T>(a.out, b, i, h);
        const float *const o32 = a.out32 ? a.out32 + (((size_t)b * a.Lq + i) * a.Hq + h) * D : nullptr;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = 16 * c + 8 * hh;
            if constexpr (DTABLE && sizeof(T) == 2) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = row_on && col + e < D ? o32[col + e] : 0.f;
                uint4 part = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])), next;
                d = band_mma(part, gf[c], d);
                band_rest(v, part, next);
                d = band_mma(next, gf[c], d);
                band_rest(v, next, part);
                d = band_mma(part, gf[c], d);
            } else {
                typename band_t<T>::frag of;
                band_clear(of);
                if (row_on) of = band_load8<MODE>(orow, col, D);
                d = band_mma(of, gf[c], d);
                if constexpr (sizeof(T) == 2) {
                    if (a.rest) {
                        band_clear(of);
                        if (row_on) of = band_load8<MODE>(a.rest + (((size_t)b * a.Lq + i) * a.Hq + h) * D, col, D);
                        d = band_mma(of, gf[c], d);
                    }
                }
            }
        }
        float mine = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) mine = rho(r) + 4 * hh == l31 ? d[r] : mine;
        del = mine + __shfl_xor(mine, 32, 64);  // (in one of the two halves, zero in the other)
    }
    if (row_on && hh == 0 && wave < ROWS / 32) a.delta[stat] = del;
    f32x16 dq[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) dq[db] = band_zero();
    float far_lo = 0.f, far_hi = 0.f;

    using Stage = BandStage<T, DP, MODE>;
    Stage ks, vs;
    ks.init(a.k.s.l, D);
    vs.init(a.v.s.l, D);
    if (MODE == 1 && !Stage::DIRECT && D < DP) {
        Stage::clear(lds, NB * 2 * BAND_TILE, D);
        __syncthreads();
    }
    BandWalk kw, vw;
    kw.init(band_row<T>(a.k, b, 0, at.hk), ks.ld, BAND_TILE, tiles);
    vw.init(band_row<T>(a.v, b, 0, at.hk), vs.ld, BAND_TILE, tiles);
    int jt = tiles.n_sink ? 0 : tiles.first * BAND_TILE;
    if (tiles.count) {
        ks.fetch(kw.p, sq.kn - 1 - jt, D, lds);
        vs.fetch(vw.p, sq.kn - 1 - jt, D, lds + ELEMS);
    }
    for (int it = 0; it < tiles.count; ++it) {
        T *const K = lds + (NB == 2 ? (it & 1) : 0) * 2 * ELEMS, *const V = K + ELEMS;
        if constexpr (Stage::DIRECT) {
            band_landed();
            band_barrier();
        } else {
            if constexpr (NB == 1) band_barrier();
            ks.put(K, D);
            vs.put(V, D);
        }
        const int tile = jt;
        jt = it + 1 == tiles.n_sink ? tiles.first * BAND_TILE : jt + BAND_TILE;
        if (it + 1 < tiles.count) {
            T *const K1 = lds + (NB == 2 ? ((it + 1) & 1) : 0) * 2 * ELEMS;
            kw.next(it + 1, tiles);
            vw.next(it + 1, tiles);
            ks.fetch(kw.p, sq.kn - 1 - jt, D, K1);
            vs.fetch(vw.p, sq.kn - 1 - jt, D, K1 + ELEMS);
        }
        if constexpr (!Stage::DIRECT) band_barrier();
#pragma unroll 1
        for (int u = SPLIT ? wave >> 1 : 0; u < (SPLIT ? (wave >> 1) + 1 : 2); ++u) {
            const int j0 = tile + 32 * u;
            if (edges.none(j0)) continue;
            f32x16 s = band_zero(), dp = band_zero();
            {
                typename band_t<T>::frag kf[C], vf[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    kf[c] = band_rows<DP>(K, 32 * u + l31, c, hh);
                    vf[c] = band_rows<DP>(V, 32 * u + l31, c, hh);
                }
                if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    s = band_mma(kf[c], qf[c], s);
                    dp = band_mma(vf[c], gf[c], dp);
                }
            }
            typename band_t<T>::frag kc[2][DP / 32];
            if (AHEAD) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) kc[k][db] = band_cols<DP>(K, 32 * u + 16 * k, db, lane);
            }
            float cs = scale, shift = nl;
            bool near = false;
            const int e0 = j0 + 4 * hh - p + M + BAND_MARGIN;
            if constexpr (BIAS) {
                near = j0 + 31 - w_lo > -M && j0 - w_hi < M;
                if (near) {
                    cs = 1.f;
                    if (remote) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] = band_exponent(s[r], scale, bias[e0 + rho(r)], top, true);
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] = band_exponent(s[r], scale, bias[e0 + rho(r)], top, false);
                    }
                } else if (remote) {
                    const float left = bias[j0 > w_hi ? BL - 1 : 0] - top;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], scale, left);
                    cs = 1.f;
                } else {
                    shift += bias[j0 > w_hi ? BL - 1 : 0] - top;
                }
            } else if constexpr (WHOLE) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = s[r] * scale + nl;
                cs = 1.f, shift = low;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], cs, shift));
            if (edges.cut_hi(j0)) {
                const int hi = key_hi - j0 - 4 * hh;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = rho(r) <= hi ? s[r] : 0.f;
            }
            if (edges.cut_lo(j0)) {
                const int lo = key_lo - j0 - 4 * hh, first = edges.sinks - j0 - 4 * hh;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = (int)(rho(r) >= lo) | (int)(rho(r) < first) ? s[r] : 0.f;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= dp[r] - del;
            if constexpr (DTABLE) {
                // A row's 32 values go one column further left than the row's above, so that the 63 distances of the tile are
                // columns (the rest of the 64 x 32 stays zero), and a lane sums one: in order, where the atomic additions
                // of LDS, in no order, took 140 cycles for each of the 16 registers.
                if (near) {
                    float *const mine = slant + wave * 32 * 64;
                    band_fence();
#pragma unroll
                    for (int r = 0; r < 16; ++r) mine[l31 * 63 + 31 + 4 * hh + rho(r)] = s[r];
                    band_fence();  // (a wave's LDS accesses complete in order)
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < 32; ++k) part[k & 3] += mine[64 * k + lane];
                    float *const at_distance = sums + wave * BL + (j0 - w_lo + lane - 31 + M + BAND_MARGIN);
                    *at_distance += (part[0] + part[1]) + (part[2] + part[3]);
                    band_fence();
                } else {
                    float t = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) t += s[r];
                    if (j0 > w_hi) far_hi += t;
                    else far_lo += t;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                typename band_t<T>::frag sf;
                band_pack(s, k, sf);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    if (!AHEAD) kc[k][db] = band_cols<DP>(K, 32 * u + 16 * k, db, lane);
                    dq[db] = band_mma(kc[k][db], sf, dq[db]);
                }
            }
        }
    }
    if constexpr (SPLIT) {
        __syncthreads();
        float *const meet = reinterpret_cast<float *>(smem) + (wave & 1) * 32 * DP + lane;  // [2][registers][lane]
        if (wave >= 2) {
#pragma unroll
            for (int k = 0; k < DP / 2; ++k) meet[64 * k] = dq[k >> 4][k & 15];
        }
        __syncthreads();
        if (wave < 2) {
#pragma unroll
            for (int k = 0; k < DP / 2; ++k) dq[k >> 4][k & 15] += meet[64 * k];
        }
    }
    band_store_row<T, DP, MODE>(const_cast<T *>(band_row<T>(a.dq, b, i, h)), dq, a.scale, a.D, hh, i < a.Lq && (!SPLIT || wave < 2));

    if constexpr (DTABLE) {
        // clipped distances meet in the two end entries, then the four waves' sums are added
        far_lo = wave_sum(far_lo);
        far_hi = wave_sum(far_hi);
        __syncthreads();
        if (threadIdx.x < 8) {
            float *const t = sums + (threadIdx.x >> 1) * BL;
            const int e = threadIdx.x & 1 ? BL - 1 - BAND_MARGIN : BAND_MARGIN, dir = threadIdx.x & 1 ? 1 : -1;
            float v = t[e];
            for (int k = 1; k <= BAND_MARGIN; ++k) v += t[e + dir * k];
            t[e] = v;
        }
        __syncthreads();
        if (lane == 0) {
            sums[wave * BL + BAND_MARGIN] += far_lo;
            sums[wave * BL + BL - 1 - BAND_MARGIN] += far_hi;
        }
        __syncthreads();
        const int n = 2 * a.M + 1;
        const int nqb = (a.Lq + ROWS - 1) / ROWS;
        float *const dst = a.partial + ((size_t)h * a.B * nqb + (size_t)b * nqb + at.i_lo / ROWS) * n;
        for (int e = threadIdx.x; e < n; e += 256) {
            const float *const t = sums + BAND_MARGIN + e;
            dst[e] = (t[0] + t[BL]) + (t[2 * BL] + t[3 * BL]);
        }
    }
}

// d_table[bucket][head] = the sum of the head's `rows` row blocks over the distances of the bucket: the distances listed in
// their order, then all pairs of a block and a listed distance over 256 threads, so that buckets of one distance and of
// hundreds keep them all busy.  (Sums by distance first and by bucket in a second launch took the same time, and one more launch.)
__global__ __launch_bounds__(256) void band_attn_table_kernel(const float *__restrict__ partial, const int *__restrict__ buckets, int rows, int n,
                                                              int n_buckets, int heads, float *__restrict__ d_table) {
    __shared__ int list[2 * BAND_MAX_DISTANCE + 1], length;
    __shared__ float red[4];
    const int bucket = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63;
    if (threadIdx.x < 64) {
        int at = 0;
        for (int e0 = 0; e0 < n; e0 += 64) {
            const bool in = e0 + lane < n && min(max(buckets[e0 + lane], 0), n_buckets - 1) == bucket;
            const unsigned long long all = __ballot(in);
            if (in) list[at + __popcll(all & ((1ull << lane) - 1))] = e0 + lane;
            at += __popcll(all);
        }
        if (lane == 0) length = at;
    }
    __syncthreads();
    const float *const src = partial + (size_t)h * rows * n;
    const unsigned cnt = length, pairs = cnt * (unsigned)rows;  // (the caller sees to it that n * rows fits)
    float v = 0.f;
#pragma unroll 4
    for (unsigned k = threadIdx.x; k < pairs; k += 256) {
        const unsigned r = k / cnt;
        v += src[(size_t)r * n + list[k - r * cnt]];
    }
    v = wave_sum(v);
    if (lane == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) d_table[(size_t)bucket * heads + h] = (red[0] + red[1]) + (red[2] + red[3]);
}

// rows of a dq workgroup: 64 while 128 would leave SIMDs without a wave
static int band_dq_rows(const BandArgs &a) {
    return (long long)a.B * a.Hq * ((a.Lq + BAND_ROWS - 1) / BAND_ROWS) < 256 ? BAND_ROWS / 2 : BAND_ROWS;
}

template <typename T, int DP, int MODE, bool BIAS, bool DTABLE> static int launch_bwd(const BandArgs &a, hipStream_t st) {
    const size_t images = (size_t)band_t<T>::nbuf(DP) * 2 * band_t<T>::template elems<DP>(BAND_TILE) * sizeof(T);
    const size_t bl = BIAS ? (2 * (a.M + BAND_MARGIN) + 1) * sizeof(float) : 0;
    if (a.Lq && a.Hq) {
        const size_t lds = images + (DTABLE ? ((bl + 15) & ~(size_t)15) + 4 * (32 * 64 * sizeof(float) + bl) : bl);
        const bool split = band_dq_rows(a) < BAND_ROWS;
        auto kern = split ? band_attn_dq_kernel<T, DP, MODE, BIAS, DTABLE, true> : band_attn_dq_kernel<T, DP, MODE, BIAS, DTABLE, false>;
        if (int rc = band_allow_lds("dsw_band_attn_bwd", kern, lds)) return rc;
        kern<<<dim3((unsigned)((long long)a.B * a.Hq * ((a.Lq + band_dq_rows(a) - 1) / band_dq_rows(a)))), 256, lds, st>>>(a);
        if (int rc = check_launch("dsw_band_attn_bwd (dq)")) return rc;
    }
    if (a.Lk) {
        const size_t lds = images + (size_t)band_t<T>::nbuf(DP) * (BIAS ? 4 : band_whole<T>(BIAS) ? 3 : 2) * BAND_TILE * sizeof(float) + bl;
        auto kern = band_attn_dkv_kernel<T, DP, MODE, BIAS>;
        if (int rc = band_allow_lds("dsw_band_attn_bwd", kern, lds)) return rc;
        const long long nkb = (a.Lk + BAND_ROWS - 1) / BAND_ROWS, heads = (long long)a.B * a.Hkv;
        kern<<<dim3((unsigned)(heads * (a.sink_blocks * a.sink_chunks + (nkb - a.sink_blocks) * a.chunks))), 256, lds, st>>>(a);
        if (int rc = check_launch("dsw_band_attn_bwd (dk, dv)")) return rc;
        const long long joined = heads * (a.chunks > 1 ? nkb : a.sink_chunks > 1 ? a.sink_blocks : 0);
        if (joined) {
            if (joined * a.D >= (1LL << 31)) return fail(DSW_EUNSUPPORTED, "dsw_band_attn_bwd: %lld shared key blocks", joined);
            if (MODE == 0) band_attn_join_dkv_kernel<T, 4><<<dim3((unsigned)(joined * (a.D / 4))), 256, 0, st>>>(a);
            else band_attn_join_dkv_kernel<T, 1><<<dim3((unsigned)(joined * a.D)), 256, 0, st>>>(a);
            if (int rc = check_launch("dsw_band_attn_bwd (join)")) return rc;
        }
    }
    return DSW_OK;
}

static size_t round16(size_t n) { return (n + 3) & ~(size_t)3; }

}  // namespace dsw

using namespace dsw;

extern "C" size_t dsw_band_attn_bwd_workspace(const dsw_band_desc *d) {
    BandArgs a;
    if (band_make_args("dsw_band_attn_bwd_workspace", d, a)) return 0;
    size_t n = round16((size_t)a.B * a.Hq * a.Lq);
    n += (size_t)band_chunks(a, d->dtype).shares * 2 * BAND_ROWS * a.D;
    if (a.table) n += (size_t)a.Hq * ((size_t)a.B * ((a.Lq + band_dq_rows(a) - 1) / band_dq_rows(a))) * (2 * a.M + 1);
    return n * sizeof(float);
}

extern "C" int dsw_band_attn_bwd(const dsw_band_desc *d, const void *q, const dsw_strides *sq, const void *k, const dsw_strides *sk,
                                 const void *v, const dsw_strides *sv, const void *out, const dsw_strides *so, const float *out32,
                                 const void *dout, const dsw_strides *sdo, const float *lse, void *dq, const dsw_strides *sdq, void *dk,
                                 const dsw_strides *sdk, void *dv, const dsw_strides *sdv, float *d_table, void *workspace,
                                 size_t workspace_bytes, void *stream) {
    const char *who = "dsw_band_attn_bwd";
    BandArgs a;
    int rc = band_make_args(who, d, a);
    if (rc) return rc;
    if (a.B == 0 || a.Hkv == 0) return DSW_OK;
    const bool no_rows = a.Lq == 0 || a.Hq == 0, no_keys = a.Lk == 0;  // (no query heads: dk and dv are zeros all the same)
    int mode = 0;
    if ((rc = band_tensor(who, "q", q, sq, d->dtype, a.D, no_rows, a.q, mode)) || (rc = band_tensor(who, "k", k, sk, d->dtype, a.D, no_keys, a.k, mode)) ||
        (rc = band_tensor(who, "v", v, sv, d->dtype, a.D, no_keys, a.v, mode)) || (rc = band_tensor(who, "out", out, so, d->dtype, a.D, no_rows, a.out, mode)) ||
        (rc = band_tensor(who, "dout", dout, sdo, d->dtype, a.D, no_rows, a.dout, mode)) || (rc = band_tensor(who, "dq", dq, sdq, d->dtype, a.D, no_rows, a.dq, mode)) ||
        (rc = band_tensor(who, "dk", dk, sdk, d->dtype, a.D, no_keys, a.dk, mode)) || (rc = band_tensor(who, "dv", dv, sdv, d->dtype, a.D, no_keys, a.dv, mode)))
        return rc;
    if (!no_rows && (rc = band_rest_tensor(who, d, a, mode))) return rc;
    DSW_REQUIRE(no_rows || lse, "%s: null lse", who);
    DSW_REQUIRE(d_table == nullptr || a.table, "%s: a gradient for a table that is not there", who);
    DSW_REQUIRE(d_table == nullptr || no_rows || d->dtype == DSW_F32 || out32, "%s: the table's gradient needs the forward's out32", who);
    const int n = 2 * a.M + 1;
    const long long rows = (long long)a.B * ((a.Lq + band_dq_rows(a) - 1) / band_dq_rows(a));
    if (d_table && (rows * n >= (1LL << 31) || a.Hq > 65535))
        return fail(DSW_EUNSUPPORTED, "%s: a table's gradient over %lld row blocks of %d heads", who, rows, a.Hq);
    const size_t need = dsw_band_attn_bwd_workspace(d);
    DSW_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), "%s: workspace of %zu bytes, %zu are needed", who, workspace_bytes, need);
    a.lse = const_cast<float *>(lse);
    a.lse_rest = a.table || d->dtype != DSW_F32 ? nullptr : d->lse_rest;
    a.top = a.table && lse ? a.lse + (size_t)a.B * a.Hq * a.Lq : nullptr;
    a.out32 = const_cast<float *>(out32);
    a.delta = static_cast<float *>(workspace);
    const BandChunks chunks = band_chunks(a, d->dtype);
    a.sink_blocks = chunks.sink_blocks, a.sink_chunks = chunks.sink_chunks, a.chunks = chunks.chunks;
    a.shares = a.delta + round16((size_t)a.B * a.Hq * a.Lq);
    a.partial = a.shares + (size_t)chunks.shares * 2 * BAND_ROWS * a.D;
    hipStream_t st = as_stream(stream);
    DSW_BAND_DISPATCH(d->dtype, a.D, mode, T, DP, MODE, {
        rc = d_table ? launch_bwd<T, DP, MODE, true, true>(a, st)
             : a.table ? launch_bwd<T, DP, MODE, true, false>(a, st) : launch_bwd<T, DP, MODE, false, false>(a, st);
    });
    if (rc || d_table == nullptr || a.Hq == 0) return rc;
    band_attn_table_kernel<<<dim3(a.n_buckets, a.Hq), 256, 0, st>>>(a.partial, a.buckets, (int)rows, n, a.n_buckets, a.Hq, d_table);
    return check_launch("dsw_band_attn_bwd (table)");
}
