// Attention over token sequences, forward (see band_attn.hpp for the mathematics and the register layouts).
//
// One workgroup takes 128 query rows of one head, 32 per wave, and walks the key tiles of 64 that its rows can see: the
// sinks' tiles, then the window's.  A tile's K and V rows go through LDS (read by all four waves), the next tile's are
// under way in registers meanwhile.  S^T = K Q^T puts a row's scores into the registers of two lanes, so the running
// maximum costs one exchange per tile; the accumulators are rescaled only when a maximum grew by more than 8 (the
// probabilities then stay below 2^8, and fp32 sums do not care).  Tiles that every row sees whole carry no mask.
// Rows of heads that share keys, and neighbouring row blocks, are handed to one XCD.
#include "band_attn.hpp"

namespace dsw {

template <typename T, int DP, bool BIAS, bool EXACT>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DP == 128 ? 1 : 2)) void band_attn_fwd_kernel(const BandArgs a) {
    constexpr int NB = band_t<T>::nbuf(DP), ELEMS = band_t<T>::template elems<DP>(BAND_TILE);
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T *const lds = reinterpret_cast<T *>(smem);  // [NB][K | V]
    float *const bias = reinterpret_cast<float *>(lds + NB * 2 * ELEMS);

    const int nqb = (a.Lq + BAND_ROWS - 1) / BAND_ROWS;
    const int idx = xcd_remap(blockIdx.x, gridDim.x);
    const int g = idx % a.G, rest = idx / a.G;
    const int qb = nqb - 1 - rest % nqb, bh = rest / nqb;  // (the last rows of a causal call have the most to do: first)
    const int hk = bh % a.Hkv, b = bh / a.Hkv, h = hk * a.G + g;
    const int lane = threadIdx.x & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const BandSeq sq = band_seq(a, b);
    const int i_lo = qb * BAND_ROWS, i0 = i_lo + 32 * wave, i = i0 + l31;
    const bool row_on = i < sq.qn, wave_on = i0 < sq.qn;
    const int p = sq.off + i, w_lo = sq.off + i0, w_hi = sq.off + min(i0 + 31, sq.qn - 1);
    const BandTiles tiles = band_tiles<BAND_TILE>(a, sq.kn, sq.off + i_lo, sq.off + min(i_lo + BAND_ROWS, sq.qn) - 1);

    const T *const qrow = band_row<T>(a.q, b, i, h);
    const T *const kbase = band_row<T>(a.k, b, 0, hk);
    const T *const vbase = band_row<T>(a.v, b, 0, hk);
    if constexpr (BIAS) band_stage_bias(a, h, 1, bias, 256);

    typename band_t<T>::frag qf[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        if (row_on) qf[c] = band_load8(qrow, 16 * c + 8 * hh, a.D, a.q.mode);
        else band_clear(qf[c]);
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) o[db] = band_zero();
    float m = -INFINITY, l = 0.f;

    BandStage<T, DP> ks, vs;
    if (tiles.count) {
        const int j0 = tiles.at(0) * BAND_TILE;
        ks.load(kbase, a.k.s.l, j0, sq.kn, a.D, a.k.mode);
        vs.load(vbase, a.v.s.l, j0, sq.kn, a.D, a.v.mode);
    }
    for (int it = 0; it < tiles.count; ++it) {
        T *const K = lds + (NB == 2 ? (it & 1) : 0) * 2 * ELEMS, *const V = K + ELEMS;
        if constexpr (NB == 1) lds_barrier();
        ks.put(K);
        vs.put(V);
        if (it + 1 < tiles.count) {
            const int j1 = tiles.at(it + 1) * BAND_TILE;
            ks.load(kbase, a.k.s.l, j1, sq.kn, a.D, a.k.mode);
            vs.load(vbase, a.v.s.l, j1, sq.kn, a.D, a.v.mode);
        }
        lds_barrier();
        const int j0 = tiles.at(it) * BAND_TILE, j9 = j0 + BAND_TILE - 1;
        if (!wave_on || j0 > w_hi + a.right || (j9 < w_lo - a.left && j0 >= a.sinks)) continue;
        const bool full = j9 < sq.kn && j9 <= w_lo + a.right && (j0 >= w_hi - a.left || j9 < a.sinks);

        f32x16 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u] = band_zero();
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) s[u] = band_mma(band_rows<DP>(K, 32 * u + l31, c, hh), qf[c], s[u]);
        }
        float bu = 0.f;  // bias of a tile whose distances are all clipped
        bool near = false;
        if constexpr (BIAS) {
            near = j9 - w_lo > -a.M && j0 - w_hi < a.M;
            if (near) {
                const float *br = bias + (j0 + 4 * hh - p + a.M + BAND_MARGIN);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[u][r] = __builtin_fmaf(s[u][r], a.c, br[32 * u + rho(r)]);
            } else {
                bu = bias[j0 > w_hi ? 2 * (a.M + BAND_MARGIN) : 0];
            }
        }
        if (!full) {
            const BandMask mask = band_row_mask(a, p, sq.kn, j0 + 4 * hh);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[u][r] = mask.sees(32 * u + rho(r)) ? s[u][r] : -INFINITY;
        }
        float x = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) x = fmaxf(x, s[u][r]);
        const float c = BIAS && near ? 1.f : a.c;
        x = max_across_halves(__builtin_fmaf(x, c, bu));
        if (__any(x > m + 8.f)) {
            const float mn = fmaxf(m, x), alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
        }
        const float shift = bu - (m == -INFINITY ? 0.f : m);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], c, shift));
                l += s[u][r];
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                typename band_t<T>::frag pf;
                band_pack(s[u], k, pf);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    const auto vf = band_cols<DP>(V, 32 * u + 16 * k, db, lane);
                    o[db] = band_mma(vf, pf, o[db]);
                    if constexpr (EXACT && sizeof(T) == 2) {
                        uint4 rf;
                        band_pack_rest(s[u], k, pf, rf);
                        o[db] = band_mma(vf, rf, o[db]);
                    }
                }
            }
        }
    }

    float bad = 0.f;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = __builtin_fmaf(o[db][r], 0.f, bad);
    if (__any(bad != 0.f))
        band_careful<T, DP, BIAS, BAND_TILE>(a, qrow, kbase, vbase, h, p, row_on, sq.kn, tiles, 0, tiles.count, 1, hh, m, l, o);

    l += __shfl_xor(l, 32, 64);
    const float inv = !row_on || l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)  // rows behind the sequence: zeros, whatever the tiles held
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] = row_on ? o[db][r] : 0.f;
    const bool store = i < a.Lq;
    band_store_row<T, DP>(const_cast<T *>(band_row<T>(a.out, b, i, h)), o, inv, a.D, a.out.mode, hh, store);
    if constexpr (EXACT)
        band_store_row<float, DP>(a.out32 + (((size_t)b * a.Lq + i) * a.Hq + h) * a.D, o, inv, a.D, a.D % 4 ? 2 : 0, hh, store);
    if (a.lse && store && hh == 0)
        a.lse[((size_t)b * a.Hq + h) * a.Lq + i] = !row_on || l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

template <typename T, int DP, bool BIAS, bool EXACT> static int launch_fwd(const BandArgs &a, hipStream_t st) {
    const size_t lds = (size_t)band_t<T>::nbuf(DP) * 2 * band_t<T>::template elems<DP>(BAND_TILE) * sizeof(T) +
                       (BIAS ? (2 * (a.M + BAND_MARGIN) + 1) * sizeof(float) : 0);
    auto kern = band_attn_fwd_kernel<T, DP, BIAS, EXACT>;
    if (lds > 65536) {
        hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return fail(DSW_ELAUNCH, "dsw_band_attn_fwd: %zu bytes of LDS: %s", lds, hipGetErrorString(e));
    }
    const long long grid = (long long)a.B * a.Hq * ((a.Lq + BAND_ROWS - 1) / BAND_ROWS);
    kern<<<dim3((unsigned)grid), 256, lds, st>>>(a);
    return check_launch("dsw_band_attn_fwd");
}

int band_tensor(const char *who, const char *name, const void *p, const dsw_strides *s, int dtype, int D, bool null_ok, BandTensor &t) {
    DSW_REQUIRE((p && s) || null_ok, "%s: null %s", who, name);
    t.p = p;
    t.s = s ? *s : dsw_strides{0, 0, 0};
    const int size = dtype == DSW_F32 ? 4 : 2, wide = 16 / size;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    auto fits = [&](int n) { return D % n == 0 && at % (n * size) == 0 && t.s.b % n == 0 && t.s.l % n == 0 && t.s.h % n == 0; };
    t.mode = fits(wide) ? 0 : fits(4 / size) ? 1 : 2;
    return DSW_OK;
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

#define DSW_BAND_DISPATCH(dtype, D, T, DP, ...)                                   \
    DSW_DISPATCH_DTYPE(dtype, T, {                                                \
        if ((D) <= 32) { constexpr int DP = 32; __VA_ARGS__; }                    \
        else if ((D) <= 64) { constexpr int DP = 64; __VA_ARGS__; }               \
        else { constexpr int DP = 128; __VA_ARGS__; }                             \
    })

extern "C" size_t dsw_band_attn_fwd_workspace(const dsw_band_desc *d) {
    int nrb = 0, nsplit = 0;
    BandArgs a;
    if (band_make_args("dsw_band_attn_fwd_workspace", d, a) || !band_step_plan(*d, nrb, nsplit) || nsplit < 2) return 0;
    // per split and row: D sums, the maximum and the denominator
    return (size_t)d->B * d->Hkv * nrb * nsplit * 32 * (d->D + 2) * sizeof(float);
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
    if ((rc = band_tensor(who, "q", q, sq, d->dtype, a.D, false, a.q)) || (rc = band_tensor(who, "k", k, sk, d->dtype, a.D, no_keys, a.k)) ||
        (rc = band_tensor(who, "v", v, sv, d->dtype, a.D, no_keys, a.v)) || (rc = band_tensor(who, "out", out, so, d->dtype, a.D, false, a.out)))
        return rc;
    DSW_REQUIRE(out32 == nullptr || (a.table && d->dtype == DSW_BF16), "%s: out32 goes with a bias table and bf16 tensors", who);
    a.lse = lse;
    a.out32 = out32;
    hipStream_t st = as_stream(stream);
    if (lse == nullptr && out32 == nullptr && band_step_plan(*d, a.nrb, a.nsplit)) {
        const size_t need = dsw_band_attn_fwd_workspace(d);
        DSW_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), "%s: workspace of %zu bytes, %zu are needed", who, workspace_bytes, need);
        a.partial = static_cast<float *>(workspace);
        return band_launch_step(a, d->dtype, st);
    }
    DSW_BAND_DISPATCH(d->dtype, a.D, T, DP, {
        if constexpr (sizeof(T) == 2) {
            if (out32) return launch_fwd<T, DP, true, true>(a, st);
        }
        return a.table ? launch_fwd<T, DP, true, false>(a, st) : launch_fwd<T, DP, false, false>(a, st);
    });
    return DSW_OK;
}
