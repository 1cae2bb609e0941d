// Attention over token sequences for few query rows: new tokens over a cache, short sequences (see band_attn.hpp for the
// mathematics).
//
// Bound by the bytes of the keys and values, which every query head of a shared key head reads: the Lq * G rows of a key
// head sit side by side on the lane axis of one 32x32 tile (32 rows to a block).  A workgroup takes one block and one of
// `nsplit` shares of the key tiles (32 keys); its four waves take every fourth tile each, on their own - K straight
// from memory into the operand registers, V through a piece of LDS that only the wave touches, no barrier in the loop,
// the next tile under way meanwhile - and meet at the end.  With more than one share the sums, maxima and denominators
// go to the workspace, and a second kernel joins them in the order of the shares.  One token over 8 caches of 4096 to 32768
// keys, 16 heads on 4 of 64, bf16: 151 MB in 29 us, 5.2 TB/s, and 4 us for the join; over windows of 1028 keys of 128, 16
// sequences of 8 key heads: 65 MB in 24 us, two tiles a wave, bound by latency.  For bf16 tensors the probabilities enter the
// product with V in bf16 and are divided by the sum of the rounded ones, as in the forward of many rows.
#include "band_attn.hpp"

namespace dsw {

constexpr int STEP_KEYS = 32;

// an element of the result, and what its rounding left behind
template <typename T> __device__ __forceinline__ void step_store(const BandArgs &a, int b, int i, int h, int d, float v) {
    io<T>::st(const_cast<T *>(band_row<T>(a.out, b, i, h)) + d, v);
    if constexpr (sizeof(T) == 2) {
        if (a.rest) a.rest[(((size_t)b * a.Lq + i) * a.Hq + h) * a.D + d] = f32_to_bf16(v - bf16_to_f32(f32_to_bf16(v)));
    }
}

template <typename T, int DP, int MODE, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DP == 128 ? 1 : 2)) void band_attn_step_kernel(const BandArgs a) {
    constexpr int ELEMS = band_t<T>::template elems<DP>(STEP_KEYS);
    constexpr int SLOTS = DP / 8, NV = STEP_KEYS * SLOTS / 64, STEP = 64 / SLOTS;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // [heads of the key head][2 M + 1] biases, where two workgroups a CU leave the room; then four V tiles, where the waves' sums
    // meet in the end
    float *const bias_of = reinterpret_cast<float *>(smem);
    unsigned char *const room = smem + (BIAS ? a.staged * sizeof(float) : 0);
    T *const V = reinterpret_cast<T *>(room) + wave * ELEMS;

    const int sp = blockIdx.x % a.nsplit, rest = blockIdx.x / a.nsplit;
    const int rb = rest % a.nrb, bh = rest / a.nrb, hk = bh % a.Hkv, b = bh / a.Hkv;
    const BandSeq sq = band_seq(a, b);
    const int row = rb * 32 + l31, R = a.Lq * a.G;
    const int i = row / a.G, h = hk * a.G + row - i * a.G;
    const bool row_on = row < R && i < sq.qn;
    const int p = sq.off + i;
    const int i_lo = rb * 32 / a.G, i_hi = min((rb * 32 + 31) / a.G, sq.qn - 1);
    const int p_lo = sq.off + i_lo, p_hi = sq.off + i_hi;
    const BandTiles tiles = band_tiles<STEP_KEYS>(a, sq.kn, p_lo, p_hi);
    const int share = (tiles.count + a.nsplit - 1) / a.nsplit, t_end = min((sp + 1) * share, tiles.count);
    const int t_begin = sp * share + wave;

    const float *const bias_row = bias_of + (row - i * a.G) * (2 * a.M + 1) + a.M;
    if (BIAS && a.staged) {
        const int n = 2 * a.M + 1;
        for (int e = threadIdx.x; e < a.G * n; e += 256) {
            const int g = e / n;
            bias_of[e] = band_bias_at(a, hk * a.G + g, e - g * n - a.M);
        }
        __syncthreads();
    }
    const T *const qrow = band_row<T>(a.q, b, i, h);
    const T *const kbase = band_row<T>(a.k, b, 0, hk);
    const T *const vbase = band_row<T>(a.v, b, 0, hk);
    typename band_t<T>::frag qf[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        band_clear(qf[c]);
        if (row_on) qf[c] = band_load8<MODE>(qrow, 16 * c + 8 * hh, a.D);
        if constexpr (MODE == 1) {
            // K's piece there is the one that ends with the row (see load below): the query's columns go where it has them
            const int col = 16 * c + 8 * hh, back = col + 8 - a.D;
            if (row_on && back > 0) {
                T e[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) e[k] = k >= back ? qrow[a.D - 8 + k] : (T)0;
                __builtin_memcpy(&qf[c], e, sizeof(e));
            }
        }
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) o[db] = band_zero();
    float m = -INFINITY, l = 0.f;

    typename band_t<T>::frag kf[DP / 16], vf[NV];
    // Keys that no row of the block sees are not read (they may be uninitialised parts of a cache): a visible one stands in
    // for them, and the mask drops it.
    const int j_lo = max(0, p_lo - a.left), j_hi = min(sq.kn - 1, p_hi + a.right);
    auto load = [&](int j0) {
        auto stand_in = [&](int j) { return min(j >= j_lo || j < a.sinks ? j : j_lo, j_hi); };
        const T *kr = kbase + (long long)stand_in(j0 + l31) * a.k.s.l;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
            const int col = 16 * c + 8 * hh;
            if constexpr (MODE == 1) kf[c] = band_piece(kr + min(col, a.D - 8));
            else kf[c] = band_load8<MODE>(kr, col, a.D);
        }
        const int r = lane / SLOTS, col = 8 * (lane % SLOTS);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const T *vr = vbase + (long long)stand_in(j0 + r + n * STEP) * a.v.s.l;
            if constexpr (MODE == 1) vf[n] = band_piece(vr + min(col, a.D - 8));
            else vf[n] = band_load8<MODE>(vr, col, a.D);
        }
    };
    auto put = [&]() {
        const int r = lane / SLOTS, slot = lane % SLOTS;
        if (MODE != 1 || 8 * slot + 8 <= a.D) {
#pragma unroll
            for (int n = 0; n < NV; ++n) band_put<DP>(V, r + n * STEP, slot, vf[n]);
        } else if (8 * slot < a.D) {
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                T e[8];
                __builtin_memcpy(e, &vf[n], sizeof(e));
#pragma unroll
                for (int k = 0; k < 8; ++k) V[band_at<T, DP>(r + n * STEP, a.D - 8 + k)] = e[k];
            }
        }
    };
    if (MODE == 1 && a.D < DP)  // the columns past D, which put() leaves alone
        for (int e = lane; e < STEP_KEYS * (DP - a.D); e += 64) V[band_at<T, DP>(e / (DP - a.D), a.D + e % (DP - a.D))] = (T)0;
    if (t_begin < t_end) load(tiles.at(t_begin) * STEP_KEYS);
    for (int t = t_begin; t < t_end; t += 4) {
        const int j0 = tiles.at(t) * STEP_KEYS;
        band_fence();  // (the last tile's reads of V come first, this one's after: a wave's LDS accesses complete in order)
        put();
        band_fence();
        f32x16 s = band_zero();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) s = band_mma(kf[c], qf[c], s);
        if (t + 4 < t_end) load(tiles.at(t + 4) * STEP_KEYS);
        const BandMask mask = band_row_mask(a, p, sq.kn, j0 + 4 * hh);
        float x = -INFINITY, bias[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = j0 + rho(r) + 4 * hh;
            bias[r] = 0.f;
            if constexpr (BIAS) {
                if (a.staged) bias[r] = bias_row[min(max(j - p, -a.M), a.M)];
                else if (row < R) bias[r] = band_bias_at(a, h, j - p);
            }
            s[r] = mask.sees(rho(r)) ? s[r] : -INFINITY;
            x = fmaxf(x, __builtin_fmaf(s[r], a.c, bias[r]));
        }
        x = max_across_halves(x);
        if (__any(x > m + 8.f)) {
            const float mn = fmaxf(m, x), alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
        }
        const float shift = m == -INFINITY ? 0.f : m;
        const bool remote = BIAS && band_remote(shift);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(band_exponent(s[r], a.c, bias[r], shift, remote));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            typename band_t<T>::frag pf;
            band_pack(s, k, pf);
            l = band_sum(pf, l);  // (the weights as they enter the product: they then sum to one)
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) o[db] = band_mma(band_cols<DP>(V, 16 * k, db, lane), pf, o[db]);
        }
    }
    float bad = 0.f;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = __builtin_fmaf(o[db][r], 0.f, bad);
    float lift = 0.f;
    if (__any(bad != 0.f || (BIAS && row_on && band_strayed(m, l + __shfl_xor(l, 32, 64)))))
        band_careful<T, DP, BIAS, STEP_KEYS>(a, qrow, kbase, vbase, h, p, row_on, sq.kn, tiles, t_begin, t_end, 4, hh, m, lift, l, o);

    // the four waves meet: maxima and denominators first, then the sums, scaled to the common maximum
    l += __shfl_xor(l, 32, 64);
    __syncthreads();
    const int nrow = min(32, R - rb * 32);
    constexpr int PART = BIAS ? 3 : 2;                   // reference, denominator, lift
    float *const ml = reinterpret_cast<float *>(room);  // [4][32][PART]
    float *const os = ml + 4 * 32 * PART;                // [4][nrow][D]
    // the common reference of a row of the block, and the largest lift beside it
    auto meet = [&](int r, float &mx, float &top) {
        mx = -INFINITY, top = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, ml[(w * 32 + r) * PART]);
        if constexpr (BIAS) {
            top = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float *const x = ml + (w * 32 + r) * PART;
                top = fmaxf(top, x[0] == -INFINITY ? -INFINITY : (x[0] - mx) + x[2]);
            }
            top = mx == -INFINITY ? 0.f : top;
        }
    };
    float *const mine = ml + (wave * 32 + l31) * PART;
    if (hh == 0) {
        mine[0] = m;
        if constexpr (BIAS) mine[2] = lift;
    }
    __syncthreads();
    float mt, top;
    meet(l31, mt, top);
    const float mul = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(BIAS ? (m - mt) + (lift - top) : m - mt);
    if (hh == 0) mine[1] = m == -INFINITY ? 0.f : l * mul;
    if (l31 < nrow) {
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * db + rho(r) + 4 * hh;
                // (a wave without visible keys holds zeros, or what a row it must not see left there)
                if (d < a.D) os[(wave * nrow + l31) * a.D + d] = m == -INFINITY ? 0.f : o[db][r] * mul;
            }
    }
    __syncthreads();
    const int n = nrow * a.D;
    for (int e = threadIdx.x; e < n; e += 256) {
        const int rl = e / a.D, d = e - rl * a.D;
        float mx, den = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) den += ml[(w * 32 + rl) * PART + 1];
        if (d == 0) meet(rl, mx, top);
        const float sum = (os[e] + os[n + e]) + (os[2 * n + e] + os[3 * n + e]);
        if (a.nsplit == 1) {
            const int ro = rb * 32 + rl, io_ = ro / a.G, ho = hk * a.G + ro - io_ * a.G;
            const bool off = den == 0.f || io_ >= sq.qn;
            step_store<T>(a, b, io_, ho, d, off ? 0.f : sum / den);
            if (a.lse && d == 0) band_keep(a, ((size_t)b * a.Hq + ho) * a.Lq + io_, off, mx, top, den);
        } else {
            const int W = a.D + PART;
            float *const ws = a.partial + ((((size_t)bh * a.nrb + rb) * a.nsplit + sp) * 32 + rl) * W;
            ws[d] = sum;
            if (d == 0) {
                ws[a.D] = mx, ws[a.D + 1] = den;
                if constexpr (BIAS) ws[a.D + 2] = top;
            }
        }
    }
}

// A workgroup joins the shares of one row: every thread weighs a share or two, then each wave adds every fourth share.
constexpr int STEP_MAX_SPLITS = 512;
template <typename T> __global__ __launch_bounds__(256) void band_attn_join_kernel(const BandArgs a) {
    __shared__ float weight[STEP_MAX_SPLITS], red[8], sums[4][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, R = a.Lq * a.G;
    const int bh = blockIdx.x / R, row = blockIdx.x - bh * R, b = bh / a.Hkv, hk = bh % a.Hkv;
    const int i = row / a.G, h = hk * a.G + row - i * a.G, W = band_share_floats(a);
    const size_t step = (size_t)32 * W;
    const float *const ws = a.partial + ((size_t)bh * a.nrb + row / 32) * a.nsplit * step + (row & 31) * W;
    const int s0 = threadIdx.x, s1 = threadIdx.x + 256;
    const float m0 = s0 < a.nsplit ? ws[s0 * step + a.D] : -INFINITY, m1 = s1 < a.nsplit ? ws[s1 * step + a.D] : -INFINITY;
    const float d0 = s0 < a.nsplit ? ws[s0 * step + a.D + 1] : 0.f, d1 = s1 < a.nsplit ? ws[s1 * step + a.D + 1] : 0.f;
    const float mt = block_max(fmaxf(m0, m1), red);
    // exponents of the shares' weights beside the common reference; with a bias less the largest of them (the step kernel's lift)
    float x0 = m0 == -INFINITY ? -INFINITY : m0 - mt, x1 = m1 == -INFINITY ? -INFINITY : m1 - mt, top = 0.f;
    if (a.table) {
        if (m0 != -INFINITY) x0 += ws[s0 * step + a.D + 2];
        if (m1 != -INFINITY) x1 += ws[s1 * step + a.D + 2];
        top = block_max(fmaxf(x0, x1), red);
        top = mt == -INFINITY ? 0.f : top;
        x0 -= top, x1 -= top;
    }
    const float w0 = __builtin_amdgcn_exp2f(x0), w1 = __builtin_amdgcn_exp2f(x1);
    if (s0 < a.nsplit) weight[s0] = w0;
    if (s1 < a.nsplit) weight[s1] = w1;
    const float den = block_sum(__builtin_fmaf(d0, w0, d1 * w1), red + 4);  // (its barriers cover the weights)
    float o0 = 0.f, o1 = 0.f;
    const int c0 = min(lane, a.D - 1), c1 = min(lane + 64, a.D - 1);
#pragma unroll 4
    for (int s = wave; s < a.nsplit; s += 4) {
        // (a share without a visible key weighs nothing, and its sums are zeros)
        o0 = __builtin_fmaf(ws[s * step + c0], weight[s], o0);
        o1 = __builtin_fmaf(ws[s * step + c1], weight[s], o1);
    }
    sums[wave][lane] = o0;
    sums[wave][lane + 64] = o1;
    __syncthreads();
    const bool off = den == 0.f || i >= band_seq(a, b).qn;
    const int d = threadIdx.x;
    if (d < a.D) step_store<T>(a, b, i, h, d, off ? 0.f : ((sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d])) / den);
    if (a.lse && d == 0) band_keep(a, ((size_t)b * a.Hq + h) * a.Lq + i, off, mt, top, den);
}

// Few rows: at most 32 rows of a key head, or too few of the other kernel's workgroups (128 rows of a head) for the chip.
bool band_step_plan(const dsw_band_desc &d, int &nrb, int &nsplit) {
    if (d.B == 0 || d.Lq == 0 || d.Hq == 0 || d.Hkv == 0) return false;
    const long long R = (long long)d.Lq * (d.Hq / d.Hkv);
    if (R > 32 && (long long)d.B * d.Hq * ((d.Lq + BAND_ROWS - 1) / BAND_ROWS) >= 256) return false;
    nrb = (int)((R + 31) / 32);
    const long long G = d.Hq / d.Hkv, tokens = d.Lq < 31 / G + 2 ? d.Lq : 31 / G + 2;  // of a block of 32 rows
    const long long span = d.left < 0 || d.right < 0 ? d.Lk : (long long)d.left + tokens + d.right + d.sinks + 2 * STEP_KEYS;
    const long long tiles = ((span < d.Lk ? span : d.Lk) + STEP_KEYS - 1) / STEP_KEYS, units = (long long)d.B * d.Hkv * nrb;
    // as many workgroups as are resident at a time (two a CU in wide heads' registers, else four), with two tiles per wave at
    // least.  One token over 16 x 8 windows of 1028 keys of 128: 31 us at 2 to 4 shares, 35 at 1, 40 at 6 and 8; over 8 x 4
    // caches of up to 32768 keys of 64: 44 us at 32 shares, 47 at 16 and at 64 (graph replays, with the join).  Where there are
    // several row blocks, one workgroup a CU: their many rows make the join dear (2 x 777 rows of 4 heads of 48, window 255,
    // fp32: 23.5 us at one share, 23.3 and 12.7 for the join at two).
    const long long want = nrb > 1 ? 256 : d.D > 64 ? 512 : 1024, most = (tiles + 7) / 8;
    long long n = want / units;
    n = n < most ? n : most;
    nsplit = (int)(n < 1 ? 1 : n > STEP_MAX_SPLITS ? STEP_MAX_SPLITS : n);
    return true;
}

// Biases through LDS (two dependent loads for each of a tile's 1024 otherwise: 32 us for 28, 3 x 1098 tokens, 3 heads of 32,
// window 183, fp32, with three shares) while two workgroups fit on a CU beside the widest one's 66 KB.
constexpr int STEP_BIAS_FLOATS = 3584;
template <typename T, int DP, int MODE, bool BIAS> static int launch_step(BandArgs &a, hipStream_t st) {
    const int R = a.Lq * a.G, nrow = R < 32 ? R : 32;
    const size_t tile = (size_t)4 * band_t<T>::template elems<DP>(STEP_KEYS) * sizeof(T);
    const size_t meet = (size_t)(4 * 32 * (BIAS ? 3 : 2) + 4 * nrow * a.D) * sizeof(float), n_bias = (size_t)a.G * (2 * a.M + 1);
    a.staged = BIAS && n_bias <= STEP_BIAS_FLOATS ? (int)((n_bias + 3) & ~(size_t)3) : 0;
    const size_t lds = (tile > meet ? tile : meet) + a.staged * sizeof(float);
    auto kern = band_attn_step_kernel<T, DP, MODE, BIAS>;
    if (int rc = band_allow_lds("dsw_band_attn_fwd", kern, lds)) return rc;
    const long long grid = (long long)a.B * a.Hkv * a.nrb * a.nsplit;
    if (grid >= (1LL << 31)) return fail(DSW_EUNSUPPORTED, "dsw_band_attn_fwd: %lld workgroups", grid);
    kern<<<dim3((unsigned)grid), 256, lds, st>>>(a);
    int rc = check_launch("dsw_band_attn_fwd");
    if (rc || a.nsplit == 1) return rc;
    const long long rows = (long long)a.B * a.Hkv * R;
    if (rows >= (1LL << 31)) return fail(DSW_EUNSUPPORTED, "dsw_band_attn_fwd: %lld rows", rows);
    band_attn_join_kernel<T><<<dim3((unsigned)rows), 256, 0, st>>>(a);
    return check_launch("dsw_band_attn_fwd (join)");
}

int band_launch_step(BandArgs &a, int dtype, int mode, hipStream_t st) {
    DSW_BAND_DISPATCH(dtype, a.D, mode, T, DP, MODE, return a.table ? launch_step<T, DP, MODE, true>(a, st) : launch_step<T, DP, MODE, false>(a, st));
    return DSW_OK;
}

}  // namespace dsw
