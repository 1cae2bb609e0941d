// Attention over token sequences, forward (see band_attn.hpp for the mathematics and the register layouts).
//
// One workgroup takes 128 query rows of one head, 32 per wave, and walks the key tiles of 64 that its rows can see: the
// sinks' tiles, then the window's.  A tile's K and V rows go through LDS (read by all four waves), in bf16 straight from
// memory, the next tile's while this one is worked on.  S^T = K Q^T puts a row's scores into the registers of two lanes,
// and its probabilities are the second operand of the product with V as they stand.  The reference of a row is the
// maximum over the first tile in which it sees a key, not a running one (no maximum, no exchange, no rescaling in the loop):
// fp32 and bf16 reach 2^127 beyond it; sums that pass 2^60 move the reference up, and a workgroup that overflowed all
// the same goes over its tiles again with the running maximum.  Tiles that every row sees whole carry no mask.
//
// Rounding, for bf16 tensors: the probabilities enter the product with V in bf16, one rounding of 2^-8 each, because the matrix
// instructions take 16-bit operands (a second part would be a second product); they are divided by the sum of the rounded
// ones, so that their weights sum to one.  Results are 2.1e-3 to 2.3e-3 (rms) from 64 bits, of which their own rounding is 1.7e-3.
// Where a table wants its gradient (EXACT) the probabilities enter in three parts of 8 bits: 1.66e-3, as the rounding alone.
// Scores, exponents, sums and the log-sum-exp are fp32; the latter is that of the rounded probabilities.
//
// Neither pipe is full: the matrix instructions and the vector instructions around them (per score: an exponential of 4 plain
// instructions' time, a multiply-add, half a conversion, half an addition) take turns in the two or three waves of a SIMD.  Without
// bias, bf16: 16384 tokens, 8 heads of 128, window 4096: 264 to 294 us by card and clock, 820 to 910 TFLOP/s of the visible
// scores' products (a large matrix product reaches 1194), matrix pipe 50 % and vector pipe 44 % busy while an engine has waves,
// and a fifth of the launch in which engines have run out of them; 4 maps of 4096 tokens, 6 heads of 30, window 1025: 39 us,
// matrix 14 %, vector 48 %, of which 16 us remain with a window of one key (launch, first loads, stores).  Tried without gain: tiles two ahead, two tiles between barriers, the next
// tile's products under this one's exponentials by hand, 4 waves a SIMD (registers spill).
#include "band_attn.hpp"

namespace dsw {

template <typename T, int DP, int MODE, bool BIAS, bool EXACT>
__global__ __launch_bounds__(256, (DP == 128 ? (sizeof(T) == 4 ? 1 : 2) : sizeof(T) == 4 || EXACT ? 2 : 3)) void band_attn_fwd_kernel(const BandArgs a_) {
    constexpr int NB = band_t<T>::nbuf(DP), ELEMS = band_t<T>::template elems<DP>(BAND_TILE), C = DP / 16;
    constexpr bool KEEP = sizeof(T) == 4 || EXACT;  // (probabilities that are not rounded to bf16: see band_exponent)
    using Stage = BandStage<T, DP, MODE>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T *const lds = reinterpret_cast<T *>(smem);  // [NB][K | V]
    float *const bias = reinterpret_cast<float *>(lds + NB * 2 * ELEMS);
    const int lane = threadIdx.x & 63, l31 = lane & 31, hh = lane >> 5;

    f32x16 o[DP / 32];
    float m, l;
    bool safe = false, spoiled;
    {
        const BandArgs &a = a_;
        const BandPlace at(a, blockIdx.x, gridDim.x);
        const BandSeq &sq = at.sq;
        const BandTiles &tiles = at.tiles;
        const bool row_on = at.i < sq.qn;
        const int p = sq.off + at.i, w_lo = sq.off + at.i0, w_hi = sq.off + min(at.i0 + 31, sq.qn - 1);
        BandEdges<BAND_TILE> edges;
        edges.init(a, sq.kn, w_lo, w_hi, at.i0 < sq.qn);
        const int key_hi = min(sq.kn - 1, p + a.right), key_lo = p - a.left;
        const float scale = a.c;
        const int D = a.D, M = a.M;
        if constexpr (BIAS) band_stage_bias(a, at.h, 1, bias, 256);

        typename band_t<T>::frag qf[C];
        const T *const qrow = band_row<T>(a.q, at.b, at.i, at.h);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (row_on) qf[c] = band_load8<MODE>(qrow, 16 * c + 8 * hh, D);
            else band_clear(qf[c]);
        }
        Stage ks, vs;
        ks.init(a.k.s.l, D);
        vs.init(a.v.s.l, D);
        if (MODE == 1 && !Stage::DIRECT && D < DP) {
            Stage::clear(lds, NB * 2 * BAND_TILE, D);
            __syncthreads();
        }
        const T *const kbase = band_row<T>(a.k, at.b, 0, at.hk), *const vbase = band_row<T>(a.v, at.b, 0, at.hk);
        for (;;) {
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) o[db] = band_zero();
            bool fresh = true;  // some row has no reference yet
            BandWalk kw, vw;
            kw.init(kbase, ks.ld, BAND_TILE, tiles);
            vw.init(vbase, vs.ld, BAND_TILE, tiles);
            int j0 = tiles.n_sink ? 0 : tiles.first * BAND_TILE;
            if (tiles.count) {
                ks.fetch(kw.p, sq.kn - 1 - j0, D, lds);
                vs.fetch(vw.p, sq.kn - 1 - j0, D, lds + ELEMS);
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
                const int j1 = it + 1 == tiles.n_sink ? tiles.first * BAND_TILE : j0 + BAND_TILE;
                if (it + 1 < tiles.count) {
                    T *const K1 = lds + (NB == 2 ? ((it + 1) & 1) : 0) * 2 * ELEMS;
                    kw.next(it + 1, tiles);
                    vw.next(it + 1, tiles);
                    ks.fetch(kw.p, sq.kn - 1 - j1, D, K1);
                    vs.fetch(vw.p, sq.kn - 1 - j1, D, K1 + ELEMS);
                }
                if constexpr (!Stage::DIRECT) band_barrier();
                const int j = j0;
                j0 = j1;
                if (edges.none(j)) continue;

                // LDS reads are issued well ahead of the products that need them (left alone, each comes right in front of its product)
                f32x16 s[2];
                {
                    typename band_t<T>::frag kf[2][C];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int c = 0; c < C; ++c) kf[u][c] = band_rows<DP>(K, 32 * u + l31, c, hh);
                        if (DP == 128 || u == 1) __builtin_amdgcn_sched_barrier(0);
                        if (DP == 128) {
                            s[u] = band_zero();
#pragma unroll
                            for (int c = 0; c < C; ++c) s[u] = band_mma(kf[u][c], qf[c], s[u]);
                        }
                    }
                    if (DP < 128) {
                        s[0] = s[1] = band_zero();
#pragma unroll
                        for (int c = 0; c < C; ++c)
#pragma unroll
                            for (int u = 0; u < 2; ++u) s[u] = band_mma(kf[u][c], qf[c], s[u]);
                    }
                }
                if (edges.cut_hi(j)) {
                    const int hi = key_hi - j - 4 * hh;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[u][r] = 32 * u + rho(r) <= hi ? s[u][r] : -INFINITY;
                }
                if (edges.cut_lo(j)) {
                    const int lo = key_lo - j - 4 * hh, first = edges.sinks - j - 4 * hh;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            s[u][r] = (int)(32 * u + rho(r) >= lo) | (int)(32 * u + rho(r) < first) ? s[u][r] : -INFINITY;
                }
                // the logits are scale * s + bu, or, where distances of the tile are not clipped, scale * s + br[..]
                float bu = 0.f;
                const float *const br = bias + (j + 4 * hh - p + M + BAND_MARGIN);
                bool near = false;
                if constexpr (BIAS) {
                    near = j + BAND_TILE - 1 - w_lo > -M && j - w_hi < M;
                    if (!near) bu = bias[j > w_hi ? 2 * (M + BAND_MARGIN) : 0];
                }
                if (fresh || safe) {
                    float x = s[0][0];
                    if (near) {
                        x = -INFINITY;
#pragma unroll
                        for (int r = 0; r < 32; ++r) x = fmaxf(x, __builtin_fmaf(s[r >> 4][r & 15], scale, br[32 * (r >> 4) + rho(r & 15)]));
                    } else {
#pragma unroll
                        for (int r = 1; r < 32; ++r) x = fmaxf(x, s[r >> 4][r & 15]);
                        x = __builtin_fmaf(x, scale, bu);
                    }
                    x = max_across_halves(x);
                    const float mn = m == -INFINITY || safe ? fmaxf(m, x) : m;
                    const float alpha = mn == m || m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    l *= alpha;
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
                    fresh = __any((int)row_on & (int)(m == -INFINITY));
                }
                const float mr = m == -INFINITY ? 0.f : m;
                if constexpr (BIAS || KEEP) {
                    if (near && !band_remote(mr)) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[u][r] = band_exponent(s[u][r], scale, br[32 * u + rho(r)], mr, false);
                    } else if (near) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[u][r] = band_exponent(s[u][r], scale, br[32 * u + rho(r)], mr, true);
                    } else if (!BIAS) {  // (with a bias a row's only key is its own position's: near)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[u][r] = band_exponent(s[u][r], scale, bu, mr, false);
                    } else {
                        const float shift = bu - mr;
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[u][r] = __builtin_fmaf(s[u][r], scale, shift);
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    typename band_t<T>::frag vf[2][DP / 32];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int db = 0; db < DP / 32; ++db) vf[k][db] = band_cols<DP>(V, 32 * u + 16 * k, db, lane);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[u][r] = __builtin_amdgcn_exp2f(BIAS || KEEP ? s[u][r] : __builtin_fmaf(s[u][r], scale, -mr));
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        typename band_t<T>::frag pf;
                        band_pack(s[u], k, pf);
                        l = band_sum(pf, l);
#pragma unroll
                        for (int db = 0; db < DP / 32; ++db) o[db] = band_mma(vf[k][db], pf, o[db]);
                        if constexpr (EXACT) {  // the probabilities' other 16 bits
                            uint4 rf;
                            float rest[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) rest[e] = s[u][8 * k + e];
                            band_rest(rest, pf, rf);
                            l = band_sum(rf, l);
#pragma unroll
                            for (int db = 0; db < DP / 32; ++db) o[db] = band_mma(vf[k][db], rf, o[db]);
                            uint4 rf2;
                            band_rest(rest, rf, rf2);
                            l = band_sum(rf2, l);
#pragma unroll
                            for (int db = 0; db < DP / 32; ++db) o[db] = band_mma(vf[k][db], rf2, o[db]);
                        }
                    }
                }
                if (__any(l > 0x1p60f)) {
                    // far above the reference: move it up, by what the sum comes to (a large reference takes no step of 60
                    // exactly, the largest ones none at all)
                    const float up = l > 0x1p60f ? 60.f : 0.f, to = m + fmaxf(up, __shfl_xor(up, 32, 64));
                    const float down = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
                    m = to;
                    l *= down;
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[db][r] *= down;
                }
            }
            float bad = l * 0.f;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) bad = __builtin_fmaf(o[db][r], 0.f, bad);
            spoiled = __any((int)row_on & ((int)(bad != 0.f) | (int)band_strayed(m, l + __shfl_xor(l, 32, 64))));
            // a second time with the maximum over all keys so far as the reference, if anything overflowed or strayed
            if (safe || !__syncthreads_or(spoiled)) break;
            safe = true;
        }
    }

    auto again = __builtin_amdgcn_kernarg_segment_ptr();
    int block = blockIdx.x;
    asm volatile("" : "+s"(again), "+s"(block));  // (the same values, but for all the compiler knows others)
    const BandArgs &a = *(const BandArgs *)again;
    const BandPlace at(a, block, gridDim.x);
    const bool row_on = at.i < at.sq.qn;
    float lift = 0.f;
    if (spoiled && safe)
        band_careful<T, DP, BIAS, BAND_TILE>(a, band_row<T>(a.q, at.b, at.i, at.h), band_row<T>(a.k, at.b, 0, at.hk), band_row<T>(a.v, at.b, 0, at.hk),
                                             at.h, at.sq.off + at.i, row_on, at.sq.kn, at.tiles, 0, at.tiles.count, 1, hh, m, lift, l, o);
    l += __shfl_xor(l, 32, 64);
    const float inv = !row_on || l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)  // rows behind the sequence: zeros, whatever the tiles held
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] = row_on ? o[db][r] : 0.f;
    const bool store = at.i < a.Lq;
    band_store_row<T, DP, MODE>(const_cast<T *>(band_row<T>(a.out, at.b, at.i, at.h)), o, inv, a.D, hh, store);
    if constexpr (EXACT)  // (in mode 0 D is a multiple of 8)
        band_store_row<float, DP, MODE>(a.out32 + (((size_t)at.b * a.Lq + at.i) * a.Hq + at.h) * a.D, o, inv, a.D, hh, store);
    if constexpr (sizeof(T) == 2) {
        if (a.rest) band_store_rest<DP, MODE>(a.rest + (((size_t)at.b * a.Lq + at.i) * a.Hq + at.h) * a.D, o, inv, a.D, hh, store);
    }
    if (a.lse && store && hh == 0)
        band_keep(a, ((size_t)at.b * a.Hq + at.h) * a.Lq + at.i, !row_on || l == 0.f, m, lift, l);
}

template <typename T, int DP, int MODE, bool BIAS, bool EXACT> static int launch_fwd(const BandArgs &a, hipStream_t st) {
    const size_t lds = (size_t)band_t<T>::nbuf(DP) * 2 * band_t<T>::template elems<DP>(BAND_TILE) * sizeof(T) +
                       (BIAS ? (2 * (a.M + BAND_MARGIN) + 1) * sizeof(float) : 0);
    auto kern = band_attn_fwd_kernel<T, DP, MODE, BIAS, EXACT>;
    if (int rc = band_allow_lds("dsw_band_attn_fwd", kern, lds)) return rc;
    const long long grid = (long long)a.B * a.Hq * ((a.Lq + BAND_ROWS - 1) / BAND_ROWS);
    kern<<<dim3((unsigned)grid), 256, lds, st>>>(a);
    return check_launch("dsw_band_attn_fwd");
}

int band_tensor(const char *who, const char *name, const void *p, const dsw_strides *s, int dtype, int D, bool null_ok, BandTensor &t, int &mode) {
    DSW_REQUIRE((p && s) || null_ok, "%s: null %s", who, name);
    t.p = p;
    t.s = s ? *s : dsw_strides{0, 0, 0};
    DSW_REQUIRE(t.s.b >= 0 && t.s.l >= 0 && t.s.h >= 0, "%s: negative stride of %s", who, name);
    const int size = dtype == DSW_F32 ? 4 : 2;
    auto fits = [&](int bytes) {
        const int n = bytes / size;
        return D % n == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0 && t.s.b % n == 0 && t.s.l % n == 0 && t.s.h % n == 0;
    };
    const int m = D < 8 || !fits(4) || t.s.l * size * BAND_TILE >= (1LL << 31) ? 2 : fits(16) ? 0 : 1;
    mode = m > mode ? m : mode;
    return DSW_OK;
}

int band_rest_tensor(const char *who, const dsw_band_desc *d, BandArgs &a, int &mode) {
    if (d->out_rest == nullptr) return DSW_OK;
    DSW_REQUIRE(d->dtype == DSW_BF16, "%s: out_rest goes with bf16 tensors", who);
    BandTensor t;
    const dsw_strides s = {(long long)a.Lq * a.Hq * a.D, (long long)a.Hq * a.D, a.D};
    a.rest = static_cast<bf16_t *>(d->out_rest);
    return band_tensor(who, "out_rest", d->out_rest, &s, d->dtype, a.D, false, t, mode);
}

int band_make_args(const char *who, const dsw_band_desc *d, BandArgs &a) {
    DSW_REQUIRE(d, "%s: null description", who);
    if (d->dtype != DSW_F32 && d->dtype != DSW_BF16) return fail(DSW_EUNSUPPORTED, "%s: dtype code %d", who, d->dtype);
    DSW_REQUIRE(d->B >= 0 && d->Lq >= 0 && d->Lk >= 0 && d->Hq >= 0 && d->Hkv >= 0, "%s: negative size", who);
    if (d->D < 1 || d->D > 128) return fail(DSW_EUNSUPPORTED, "%s: head dim %d outside 1..128", who, d->D);
    if (d->Lq > BAND_FAR || d->Lk > BAND_FAR) return fail(DSW_EUNSUPPORTED, "%s: sequences of %d and %d tokens", who, d->Lq, d->Lk);
    DSW_REQUIRE(d->Hq == 0 || (d->Hkv > 0 && d->Hq % d->Hkv == 0), "%s: %d query heads over %d key heads", who, d->Hq, d->Hkv);
    DSW_REQUIRE(d->left >= -1 && d->right >= -1 && d->sinks >= 0, "%s: window (%d, %d) with %d sinks", who, d->left, d->right, d->sinks);
    DSW_REQUIRE(d->scale > 0.f && d->scale < INFINITY, "%s: scale %g is not a positive number", who, (double)d->scale);
    const long long blocks = (long long)d->B * (d->Hq > d->Hkv ? d->Hq : d->Hkv) * (((d->Lq > d->Lk ? d->Lq : d->Lk) + 31) / 32);
    if (blocks >= (1LL << 31)) return fail(DSW_EUNSUPPORTED, "%s: %lld row blocks", who, blocks);
    a = BandArgs{};
    a.B = d->B, a.Lq = d->Lq, a.Lk = d->Lk, a.Hq = d->Hq, a.Hkv = d->Hkv, a.D = d->D;
    a.G = d->Hkv ? d->Hq / d->Hkv : 0;
    a.left = d->left < 0 || d->left > BAND_FAR ? BAND_FAR : d->left;
    a.right = d->right < 0 || d->right > BAND_FAR ? BAND_FAR : d->right;
    a.sinks = d->sinks > BAND_FAR ? BAND_FAR : d->sinks;
    a.scale = d->scale, a.c = d->scale * LOG2E;
    a.q_lens = d->q_lens, a.k_lens = d->k_lens;
    a.table = d->bias_table, a.buckets = d->bias_buckets;
    if (d->bias_table) {
        DSW_REQUIRE(d->bias_buckets && d->n_buckets >= 1, "%s: a bias table without its bucket map", who);
        if (d->max_distance < 1 || d->max_distance > BAND_MAX_DISTANCE)
            return fail(DSW_EUNSUPPORTED, "%s: bias distances up to %d (1..%d are built)", who, d->max_distance, BAND_MAX_DISTANCE);
        a.n_buckets = d->n_buckets, a.M = d->max_distance;
    }
    return DSW_OK;
}

}  // namespace dsw

using namespace dsw;

extern "C" size_t dsw_band_attn_fwd_workspace(const dsw_band_desc *d) {
    int nrb = 0, nsplit = 0;
    BandArgs a;
    if (band_make_args("dsw_band_attn_fwd_workspace", d, a) || !band_step_plan(*d, nrb, nsplit) || nsplit < 2) return 0;
    return (size_t)d->B * d->Hkv * nrb * nsplit * 32 * band_share_floats(a) * sizeof(float);
}

extern "C" int dsw_band_attn_fwd(const dsw_band_desc *d, const void *q, const dsw_strides *sq, const void *k, const dsw_strides *sk,
                                 const void *v, const dsw_strides *sv, void *out, const dsw_strides *so, float *lse, float *out32,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "dsw_band_attn_fwd";
    BandArgs a;
    int rc = band_make_args(who, d, a);
    if (rc) return rc;
    if (a.B == 0 || a.Lq == 0 || a.Hq == 0) return DSW_OK;
    const bool no_keys = a.Lk == 0;
    int mode = 0;
    if ((rc = band_tensor(who, "q", q, sq, d->dtype, a.D, false, a.q, mode)) || (rc = band_tensor(who, "k", k, sk, d->dtype, a.D, no_keys, a.k, mode)) ||
        (rc = band_tensor(who, "v", v, sv, d->dtype, a.D, no_keys, a.v, mode)) || (rc = band_tensor(who, "out", out, so, d->dtype, a.D, false, a.out, mode)))
        return rc;
    DSW_REQUIRE(out32 == nullptr || (a.table && d->dtype == DSW_BF16), "%s: out32 goes with a bias table and bf16 tensors", who);
    if ((rc = band_rest_tensor(who, d, a, mode))) return rc;
    a.lse = lse;
    a.lse_rest = a.table || d->dtype != DSW_F32 ? nullptr : d->lse_rest;
    a.top = lse && a.table ? lse + (size_t)a.B * a.Hq * a.Lq : nullptr;
    a.out32 = out32;
    hipStream_t st = as_stream(stream);
    if (out32 == nullptr && band_step_plan(*d, a.nrb, a.nsplit)) {
        const size_t need = dsw_band_attn_fwd_workspace(d);
        DSW_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), "%s: workspace of %zu bytes, %zu are needed", who, workspace_bytes, need);
        a.partial = static_cast<float *>(workspace);
        return band_launch_step(a, d->dtype, mode, st);
    }
    DSW_BAND_DISPATCH(d->dtype, a.D, mode, T, DP, MODE, {
        if constexpr (sizeof(T) == 2) {
            if (out32) return launch_fwd<T, DP, MODE, true, true>(a, st);
        }
        return a.table ? launch_fwd<T, DP, MODE, true, false>(a, st) : launch_fwd<T, DP, MODE, false, false>(a, st);
    });
    return DSW_OK;
}
