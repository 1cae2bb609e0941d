// Norm of every head's query and key row with the rotation by position behind it, one pass forward and one backward.
//
//   x: a head's D columns of one token      r = 1 / sqrt(mean(x^2) + eps)      u = w * x * r
//   y = u with its first 2 * axes * pairs columns turned pair by pair: pair c = a * pairs + i stands in columns
//   (c, c + axes * pairs), or (2c, 2c + 1) when interleaved, and turns by pos[token][a] * freqs[a][i]
//   backward: du = dy turned back, dw = sum over rows of du * x * r, dn = du * w, dx = r (dn - x r mean(dn * x r))
//
// Forward reads x and writes y, backward reads x and dy and writes dx: bound by memory where pieces of 16 bytes are
// possible (4 sequences of 8192 tokens, 40 rows of 128, bf16: 671 MB in 134 us, 5.0 TB/s, the rate of a plain copy), by
// vector instructions and by the number of narrow accesses where they are not (heads of 30, 131072 tokens of 12 rows:
// forward 189 MB in 48 us, backward 283 MB in 80 us, 3.5 to 3.9 TB/s).  The angles need the accurate path (positions in
// the millions: the product with the frequency is
// taken in 64 bits and reduced to a part of one turn before sine and cosine), which costs more than a row's norm; they
// are the same for all heads of a token, so a workgroup takes all heads of a few tokens and keeps the sines and cosines
// in LDS.  A row is held by RL lanes in units of two Q-element pieces, chosen so that both columns of a pair are
// in one lane: the rotation needs no exchange, the norm log2(RL) of them.  Q is the widest piece (16 bytes at most)
// that the head dim, the pair count, the strides and the addresses allow; Q = 1 takes any of them.  Loads and sums run
// without branches, over masked registers: with branches around the pieces that a row does not have, and the weights'
// sums joined by exchanges, the two kernels took 57 and 107 us.
#include "common.hpp"

namespace dsw {

struct RotOperand {
    const void *p;
    dsw_strides s;
};
struct RotArgs {
    RotOperand x[2], dy[2];  // q, k
    RotOperand y[2];         // forward: results, backward: dx
    const float *w[2];       // null: ones
    const float *freqs;
    const void *pos;         // int32 or int64 [.., axes], or null: the token's index in its sequence on every axis
    int pos_bytes;
    long long pos_batch;     // elements between the positions of two sequences (0: shared)
    float *partial;          // backward: [blocks][2][D] or null
    long long tokens;
    int L, Hq, Hkv, D, axes, pairs, rl_log, units, tpw;
    int mul_n, mul_pairs;    // e / n = e * mul_n >> 18 for e below 2^11 and n up to 64; c / pairs = c * mul_pairs >> 16 for c below 64
    float eps;
};

// Q consecutive elements, aligned to their size (16 bytes at most): loaded as WORDS registers, unpacked later
template <typename T, int Q> struct piece;
template <int Q> struct piece<bf16_t, Q> {
    static constexpr int WORDS = Q == 1 ? 1 : Q / 2;
    __device__ static __forceinline__ void ld(const bf16_t *p, uint32_t *w) {
        if constexpr (Q == 8) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else if constexpr (Q == 4) {
            const uint2 u = *reinterpret_cast<const uint2 *>(p);
            w[0] = u.x, w[1] = u.y;
        } else if constexpr (Q == 2) {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
            w[0] = *p;
        }
    }
    __device__ static __forceinline__ void unpack(const uint32_t *w, float *v) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            if constexpr (Q > 1) v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ static __forceinline__ void st(bf16_t *p, const float *v) {
        if constexpr (Q == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        else if constexpr (Q == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
        else if constexpr (Q == 2) *reinterpret_cast<uint32_t *>(p) = pack_bf16(v[0], v[1]);
        else *p = f32_to_bf16(v[0]);
    }
};
template <int Q> struct piece<float, Q> {
    static constexpr int WORDS = Q;
    __device__ static __forceinline__ void ld(const float *p, uint32_t *w) {
        if constexpr (Q == 4) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else if constexpr (Q == 2) {
            const uint2 u = *reinterpret_cast<const uint2 *>(p);
            w[0] = u.x, w[1] = u.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        }
    }
    __device__ static __forceinline__ void unpack(const uint32_t *w, float *v) {
#pragma unroll
        for (int i = 0; i < Q; ++i) v[i] = __uint_as_float(w[i]);
    }
    __device__ static __forceinline__ void st(float *p, const float *v) {
        if constexpr (Q == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else if constexpr (Q == 2) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
        else *p = v[0];
    }
};

constexpr int ROT_THREADS = 256;

// cosines and sines of nt tokens' angles, [token][pair], and the two weights [2][D] behind them (forward and backward
// read both per row)
__device__ __forceinline__ void rot_tables(const RotArgs &a, long long token0, int nt, float2 *cs, float *w) {
    const int n = a.axes * a.pairs;
    for (int e = threadIdx.x; e < nt * n; e += ROT_THREADS) {
        const int t = (int)((unsigned)e * (unsigned)a.mul_n >> 18), c = e - t * n, ax = c * a.mul_pairs >> 16;
        const unsigned token = (unsigned)token0 + t, b = token / (unsigned)a.L;  // (fewer than 2^31 tokens)
        const int l = (int)(token - b * a.L);
        const long long at = b * a.pos_batch + (long long)l * a.axes + ax;
        const long long pos = !a.pos ? l : a.pos_bytes == 8 ? static_cast<const long long *>(a.pos)[at] : static_cast<const int *>(a.pos)[at];
        // in turns; two roundings in 64 bits leave less than 2^-24 of a turn up to 2^28 turns
        double turns = (double)pos * ((double)a.freqs[c] * 0.15915494309189533577);
        turns -= rint(turns);
        float s, co;
        sincospif(2.f * (float)turns, &s, &co);
        cs[e] = make_float2(co, s);
    }
    if (w)
        for (int e = threadIdx.x; e < 2 * a.D; e += ROT_THREADS) {
            const float *src = a.w[e >= a.D];
            w[e] = src ? src[e >= a.D ? e - a.D : e] : 1.f;
        }
}

// The units of a lane, the same in all its rows: the columns of their two pieces and which of them exist.  A piece that does
// not is loaded from the row's start and masked to zero: loads under branches are waited for one by one.
template <int Q, int NU, bool INTER> struct RotUnits {
    int ca[NU], cb[NU], at[NU];  // at: first pair of the unit
    uint32_t ma[NU], mb[NU];     // all ones where the piece exists
    bool one[NU], two[NU], turned[NU];
    __device__ __forceinline__ RotUnits(int lane, int RL, int units, int n, int D) {
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            const int u = lane + j * RL;
            at[j] = Q * u;
            turned[j] = Q * u < n;
            ca[j] = turned[j] ? (INTER ? 2 * Q * u : Q * u) : 2 * Q * u;
            cb[j] = turned[j] && !INTER ? n + Q * u : ca[j] + Q;
            one[j] = u < units;
            two[j] = one[j] && cb[j] < D;
            turned[j] = turned[j] && one[j];
            ma[j] = one[j] ? ~0u : 0u, mb[j] = two[j] ? ~0u : 0u;
            if (!one[j]) ca[j] = 0;
            if (!two[j]) cb[j] = 0;
        }
    }
    template <typename T> __device__ __forceinline__ void ld(const T *row, uint32_t (*w)[2 * piece<T, Q>::WORDS]) const {
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            piece<T, Q>::ld(row + ca[j], w[j]);
            piece<T, Q>::ld(row + cb[j], w[j] + piece<T, Q>::WORDS);
        }
    }
    template <typename T> __device__ __forceinline__ void unpack(const uint32_t (*w)[2 * piece<T, Q>::WORDS], uint32_t row, float (*v)[2 * Q]) const {
        constexpr int N = piece<T, Q>::WORDS;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            uint32_t m[2 * N];
#pragma unroll
            for (int i = 0; i < 2 * N; ++i) m[i] = w[j][i] & (i < N ? ma[j] : mb[j]) & row;
            piece<T, Q>::unpack(m, v[j]);
            piece<T, Q>::unpack(m + N, v[j] + Q);
        }
    }
    template <typename T> __device__ __forceinline__ void st(T *row, const float (*v)[2 * Q]) const {
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            if (one[j]) piece<T, Q>::st(row + ca[j], v[j]);
            if (two[j]) piece<T, Q>::st(row + cb[j], v[j] + Q);
        }
    }
};
// the sum over the 2^rl_log lanes of a row (16 at most), in all of them
template <int CTRL> __device__ __forceinline__ float rot_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float rot_row_sum(float v, int rl_log) {
    if (rl_log > 0) v = rot_add<0xb1>(v);   // neighbours
    if (rl_log > 1) v = rot_add<0x4e>(v);   // pairs of a quad
    if (rl_log > 2) v = rot_add<0x141>(v);  // quads of eight lanes
    if (rl_log > 3) v = rot_add<0x140>(v);  // eights of sixteen
    return v;
}
// turn the pairs of a unit; inv: back
template <int Q, bool INTER> __device__ __forceinline__ void rot_turn(float *x, const float2 *cs, bool inv) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        const float2 t = cs[i];
        const float s = inv ? -t.y : t.y;
        float &p = x[INTER ? 2 * i : i], &q = x[INTER ? 2 * i + 1 : Q + i];
        const float p0 = p, q0 = q;
        p = __builtin_fmaf(p0, t.x, -(q0 * s));
        q = __builtin_fmaf(p0, s, q0 * t.x);
    }
}

// The rows (token, head) of a tile that one group of lanes takes, every G-th of them, without a division per row; where the
// tile's tokens begin in each tensor is computed once, into LDS.  (With both per row the kernels were bound by integer
// arithmetic: 83 us forward for 131072 tokens of 12 rows of 30.)
constexpr int ROT_TOKENS = 32;  // of a tile, at most
struct RotRows {
    int t, h, dt, dh, H;
    __device__ __forceinline__ RotRows(int heads, int grp, int G) {
        H = heads > 0 ? heads : 1;  // (no heads: the caller takes no rows)
        dt = G / H, dh = G - dt * H;
        t = grp / H, h = grp - t * H;
    }
    __device__ __forceinline__ void next() {
        t += dt, h += dh;
        const bool over = h >= H;
        h -= over ? H : 0, t += over;
    }
};
// offsets [tensor][token] for x (0, 1), y (2, 3) and, backward, dy (4, 5); a barrier is the caller's
__device__ __forceinline__ void rot_offsets(const RotArgs &a, long long token0, int nt, int tensors, long long *off) {
    if (threadIdx.x >= (unsigned)(tensors * ROT_TOKENS)) return;
    const int k = threadIdx.x / ROT_TOKENS, t = threadIdx.x % ROT_TOKENS;
    if (t >= nt) return;
    const unsigned token = (unsigned)token0 + t, b = token / (unsigned)a.L, l = token - b * a.L;
    const RotOperand &o = k < 2 ? a.x[k] : k < 4 ? a.y[k - 2] : a.dy[k - 4];
    off[k * ROT_TOKENS + t] = b * o.s.b + l * o.s.l;
}

template <typename T, int Q, int NU, bool INTER>
__global__ __launch_bounds__(ROT_THREADS) void qk_norm_rotary_fwd_kernel(const RotArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int n = a.axes * a.pairs, D = a.D;
    const long long token0 = (long long)blockIdx.x * a.tpw;
    const int nt = (int)(a.tokens - token0 < a.tpw ? a.tokens - token0 : a.tpw);
    float *w = reinterpret_cast<float *>(smem);
    float2 *cs = reinterpret_cast<float2 *>(w + ((2 * D + 3) & ~3));
    const int RL = 1 << a.rl_log, lane = threadIdx.x & (RL - 1), grp = threadIdx.x >> a.rl_log, G = ROT_THREADS >> a.rl_log;
    const float inv_d = 1.f / (float)D;
    constexpr int AHEAD = 2;  // rows whose loads are under way together (one: the same; four: 52 us for 48)
    __shared__ long long off[4 * ROT_TOKENS];
    rot_offsets(a, token0, nt, 4, off);
    __syncthreads();
    const RotUnits<Q, NU, INTER> un(lane, RL, a.units, n, D);
    RotRows row(a.Hq + a.Hkv, grp, G);
    bool first = true;
    while (first || row.t < nt) {
        uint32_t raw[AHEAD][NU][2 * piece<T, Q>::WORDS];
        T *dst[AHEAD];
        int tk[AHEAD], kind[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            tk[k] = row.t, kind[k] = row.h >= a.Hq;
            const int which = kind[k], h = row.h - (which ? a.Hq : 0), t = min(row.t, nt - 1);  // (past the tile: any of its rows)
            const T *src = static_cast<const T *>(which ? a.x[1].p : a.x[0].p) + off[which * ROT_TOKENS + t] + h * (which ? a.x[1].s.h : a.x[0].s.h);
            dst[k] = static_cast<T *>(const_cast<void *>(which ? a.y[1].p : a.y[0].p)) + off[(2 + which) * ROT_TOKENS + t] +
                     h * (which ? a.y[1].s.h : a.y[0].s.h);
            un.ld(src, raw[k]);
            row.next();
        }
        if (first) {  // the tables are made while the first rows are on their way
            rot_tables(a, token0, nt, cs, w);
            __syncthreads();
            first = false;
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            float x[NU][2 * Q];
            un.template unpack<T>(raw[k], ~0u, x);
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < NU; ++j)
#pragma unroll
                for (int i = 0; i < 2 * Q; ++i) ss = __builtin_fmaf(x[j][i], x[j][i], ss);
            ss = rot_row_sum(ss, a.rl_log);
            if (tk[k] >= nt) continue;
            const float *wr = w + (kind[k] ? D : 0);
            const float r = rsqrtf(ss * inv_d + a.eps);
#pragma unroll
            for (int j = 0; j < NU; ++j) {
#pragma unroll
                for (int i = 0; i < Q; ++i) {
                    x[j][i] *= r * wr[un.ca[j] + i];
                    x[j][Q + i] *= r * wr[un.cb[j] + i];
                }
                if (un.turned[j]) rot_turn<Q, INTER>(x[j], cs + tk[k] * n + un.at[j], false);
            }
            un.st(dst[k], x);
        }
    }
}

// One workgroup walks token tiles blockIdx.x, + gridDim.x, ...; its share of the weights' gradients stays in registers
// until the end and leaves as one row of `partial`, so that the sums have a fixed order.
template <typename T, int Q, int NU, bool INTER>
__global__ __launch_bounds__(ROT_THREADS) void qk_norm_rotary_bwd_kernel(const RotArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int n = a.axes * a.pairs, D = a.D;
    float *w = reinterpret_cast<float *>(smem);
    float2 *cs = reinterpret_cast<float2 *>(w + ((2 * D + 3) & ~3));
    const int RL = 1 << a.rl_log, lane = threadIdx.x & (RL - 1), grp = threadIdx.x >> a.rl_log, G = ROT_THREADS >> a.rl_log;
    const float inv_d = 1.f / (float)D;
    constexpr int AHEAD = 1;  // rows whose loads are under way together (two: 82 us for 80, four: 86; the registers cost waves)
    __shared__ long long off[6 * ROT_TOKENS];
    const RotUnits<Q, NU, INTER> un(lane, RL, a.units, n, D);
    float dw[2][NU][2 * Q];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < NU; ++j)
#pragma unroll
            for (int i = 0; i < 2 * Q; ++i) dw[m][j][i] = 0.f;
    const int tiles = (int)((a.tokens + a.tpw - 1) / a.tpw);
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long long token0 = (long long)tile * a.tpw;
        const int nt = (int)(a.tokens - token0 < a.tpw ? a.tokens - token0 : a.tpw);
        __syncthreads();  // the last tile's readers are done
        rot_offsets(a, token0, nt, 6, off);
        rot_tables(a, token0, nt, cs, tile == (int)blockIdx.x ? w : nullptr);
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int H = m ? a.Hkv : a.Hq;
            if (H == 0) continue;
            const float *wr = w + m * D;
            RotRows row(H, grp, G);
            while (row.t < nt) {
                uint32_t rx[AHEAD][NU][2 * piece<T, Q>::WORDS], rg[AHEAD][NU][2 * piece<T, Q>::WORDS];
                T *dst[AHEAD];
                int tk[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    tk[k] = row.t;
                    const int t = min(row.t, nt - 1);  // (past the tile: any of its rows)
                    un.ld(static_cast<const T *>(a.x[m].p) + off[m * ROT_TOKENS + t] + row.h * a.x[m].s.h, rx[k]);
                    un.ld(static_cast<const T *>(a.dy[m].p) + off[(4 + m) * ROT_TOKENS + t] + row.h * a.dy[m].s.h, rg[k]);
                    dst[k] = static_cast<T *>(const_cast<void *>(a.y[m].p)) + off[(2 + m) * ROT_TOKENS + t] + row.h * a.y[m].s.h;
                    row.next();
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    float x[NU][2 * Q], g[NU][2 * Q];
                    const uint32_t on = tk[k] < nt ? ~0u : 0u;  // (past the tile: zeros, which add nothing to the weights' gradients)
                    un.template unpack<T>(rx[k], on, x);
                    un.template unpack<T>(rg[k], on, g);
                    float ss = 0.f;
#pragma unroll
                    for (int j = 0; j < NU; ++j)
#pragma unroll
                        for (int i = 0; i < 2 * Q; ++i) ss = __builtin_fmaf(x[j][i], x[j][i], ss);
                    const float r = rsqrtf(rot_row_sum(ss, a.rl_log) * inv_d + a.eps);
                    float dot = 0.f;
#pragma unroll
                    for (int j = 0; j < NU; ++j) {
                        if (un.turned[j]) rot_turn<Q, INTER>(g[j], cs + min(tk[k], nt - 1) * n + un.at[j], true);
#pragma unroll
                        for (int i = 0; i < 2 * Q; ++i) {
                            x[j][i] *= r;  // (zero, like g, in a piece that is not there)
                            dw[m][j][i] = __builtin_fmaf(g[j][i], x[j][i], dw[m][j][i]);
                            g[j][i] *= wr[i < Q ? un.ca[j] + i : un.cb[j] + i - Q];
                            dot = __builtin_fmaf(g[j][i], x[j][i], dot);
                        }
                    }
                    dot = rot_row_sum(dot, a.rl_log) * inv_d;
#pragma unroll
                    for (int j = 0; j < NU; ++j)
#pragma unroll
                        for (int i = 0; i < 2 * Q; ++i) g[j][i] = r * __builtin_fmaf(-x[j][i], dot, g[j][i]);
                    if (tk[k] < nt) un.st(dst[k], g);
                }
            }
        }
    }
    if (a.partial == nullptr) return;
    // the groups' shares through LDS: [group][2][D], summed in a fixed order by four threads for each entry
    __syncthreads();
    float *red = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < NU; ++j)
#pragma unroll
            for (int i = 0; i < 2 * Q; ++i)
                if (i < Q ? un.one[j] : un.two[j]) red[(grp * 2 + m) * D + (i < Q ? un.ca[j] + i : un.cb[j] + i - Q)] = dw[m][j][i];
    __syncthreads();
    for (int e = threadIdx.x >> 2; e < 2 * D; e += ROT_THREADS >> 2) {
        float v = 0.f;
        for (int g = threadIdx.x & 3; g < G; g += 4) v += red[g * 2 * D + e];
        v = rot_row_sum(v, 2);
        if ((threadIdx.x & 3) == 0) a.partial[(size_t)blockIdx.x * 2 * D + e] = v;
    }
}

// dw[2][D]: the workgroups' rows of `partial`, added in a fixed order
__global__ __launch_bounds__(1024) void qk_norm_rotary_weights_kernel(const float *__restrict__ partial, int rows, int cols, float *__restrict__ dw) {
    __shared__ float red[32][33];
    int col;
    float total;
    if (column_sum_32<32>(partial, rows, cols, red, col, total)) dw[col] = total;
}

constexpr int ROT_MAX_D = 128, ROT_BWD_BLOCKS = 1024;  // (four of 256 threads a CU)

// Tokens of a tile: eight rows for each group of lanes (sixteen backward, where a tile costs two barriers), so that the
// angles, computed once per tile, and the tile's start are spread over them, while two thousand workgroups are left; one
// for new tokens.  131072 tokens of 12 rows of 30, forward: 74 us at 8 tokens, 59 at 16; 32768 tokens of 40 rows of 128: 143 us
// at 8, 155 at 16.
static int rot_tokens_per_wg(long long tokens, int heads, int groups, bool bwd) {
    const long long t = tokens / 2048, want = (bwd ? 16LL : 8LL) * groups / (heads > 0 ? heads : 1);
    const long long most = want < 4 ? 4 : want > ROT_TOKENS ? ROT_TOKENS : want;
    return t < 1 ? 1 : t > most ? (int)most : (int)t;
}
// The widest piece that a call's sizes allow; its strides and addresses may ask for a narrower one.  (The backward's number of
// workgroups has to be known before its buffers are there, so it follows from the sizes alone.)
static int rot_widest(int D, int n, int dtype) {
    int Q = dtype == DSW_F32 ? 4 : 8;
    while (Q > 1 && (D % Q || n % Q)) Q >>= 1;
    return Q;
}
static constexpr int rot_units_per_lane(int Q) { return Q == 2 ? 2 : Q == 1 ? 4 : 1; }
// lanes of a row (narrow pieces: several units per lane, so that a row's fixed costs are paid by fewer lanes)
static int rot_lanes_log(int D, int Q) {
    int k = 0;
    while ((1 << k) * rot_units_per_lane(Q) < (D + 2 * Q - 1) / (2 * Q)) ++k;
    return k;
}
static int rot_tile(long long tokens, int heads, int D, int n, int dtype, bool bwd) {
    return rot_tokens_per_wg(tokens, heads, ROT_THREADS >> rot_lanes_log(D, rot_widest(D, n, dtype)), bwd);
}

static bool operand_ok(const RotOperand &o, int heads, long long q, int size) {
    return heads == 0 || (reinterpret_cast<uintptr_t>(o.p) % (q * size) == 0 && o.s.b % q == 0 && o.s.l % q == 0 && o.s.h % q == 0);
}

static int rot_check(const char *who, RotArgs &a, int dtype, int B, bool bwd, int &Q) {
    DSW_REQUIRE(B >= 0 && a.L >= 0 && a.Hq >= 0 && a.Hkv >= 0 && a.axes >= 0 && a.pairs >= 0, "%s: negative size", who);
    if (dtype != DSW_F32 && dtype != DSW_BF16) return fail(DSW_EUNSUPPORTED, "%s: dtype code %d", who, dtype);
    if (a.D < 1 || a.D > ROT_MAX_D) return fail(DSW_EUNSUPPORTED, "%s: head dim %d outside 1..%d", who, a.D, ROT_MAX_D);
    // (64-bit product: two large factors must not wrap into an accepted one)
    DSW_REQUIRE(2LL * a.axes * a.pairs <= a.D, "%s: %d axes of %d pairs need more than the head dim %d", who, a.axes, a.pairs, a.D);
    if (a.axes == 0 || a.pairs == 0) a.axes = a.pairs = 0;
    if ((long long)B * a.L >= (1LL << 31)) return fail(DSW_EUNSUPPORTED, "%s: %lld tokens", who, (long long)B * a.L);
    a.tokens = (long long)B * a.L;
    if (a.tokens == 0 || a.Hq + a.Hkv == 0) return DSW_OK;
    if ((long long)a.Hq + a.Hkv > 4096) return fail(DSW_EUNSUPPORTED, "%s: %d + %d heads", who, a.Hq, a.Hkv);
    DSW_REQUIRE(a.axes == 0 || a.freqs, "%s: null freqs", who);
    DSW_REQUIRE(a.pos == nullptr || a.pos_bytes == 4 || a.pos_bytes == 8, "%s: positions of %d bytes", who, a.pos_bytes);
    for (int m = 0; m < 2; ++m) {
        const int h = m ? a.Hkv : a.Hq;
        DSW_REQUIRE(h == 0 || (a.x[m].p && a.y[m].p && (!bwd || a.dy[m].p)), "%s: null pointer", who);
    }
    const int n = a.axes * a.pairs, size = dtype == DSW_F32 ? 4 : 2;
    for (Q = rot_widest(a.D, n, dtype); Q > 1; Q >>= 1) {
        bool ok = true;
        for (int m = 0; m < 2 && ok; ++m) {
            const int h = m ? a.Hkv : a.Hq;
            ok = operand_ok(a.x[m], h, Q, size) && operand_ok(a.y[m], h, Q, size) && (!bwd || operand_ok(a.dy[m], h, Q, size));
        }
        if (ok) break;
    }
    a.units = (a.D + 2 * Q - 1) / (2 * Q);
    a.rl_log = rot_lanes_log(a.D, Q);
    a.tpw = rot_tile(a.tokens, a.Hq + a.Hkv, a.D, n, dtype, bwd);
    if (n) a.mul_n = (1 << 18) / n + 1, a.mul_pairs = (1 << 16) / a.pairs + 1;
    return DSW_OK;
}

template <typename T, int Q, int NU>
static int rot_launch(const RotArgs &a, bool bwd, bool interleaved, hipStream_t st) {
    const long long tiles = (a.tokens + a.tpw - 1) / a.tpw;
    size_t lds = ((2 * a.D + 3) & ~3) * 4 + (size_t)a.tpw * a.axes * a.pairs * 8;
    if (bwd) {
        const size_t shares = (size_t)(ROT_THREADS >> a.rl_log) * 2 * a.D * 4;  // (32 KB at most)
        if (a.partial && lds < shares) lds = shares;
        const dim3 grid((unsigned)(tiles < ROT_BWD_BLOCKS ? tiles : ROT_BWD_BLOCKS));
        if (interleaved) qk_norm_rotary_bwd_kernel<T, Q, NU, true><<<grid, ROT_THREADS, lds, st>>>(a);
        else qk_norm_rotary_bwd_kernel<T, Q, NU, false><<<grid, ROT_THREADS, lds, st>>>(a);
    } else {
        const dim3 grid((unsigned)tiles);
        if (interleaved) qk_norm_rotary_fwd_kernel<T, Q, NU, true><<<grid, ROT_THREADS, lds, st>>>(a);
        else qk_norm_rotary_fwd_kernel<T, Q, NU, false><<<grid, ROT_THREADS, lds, st>>>(a);
    }
    return check_launch(bwd ? "dsw_qk_norm_rotary_bwd" : "dsw_qk_norm_rotary_fwd");
}

static int rot_dispatch(const RotArgs &a, int dtype, int Q, bool bwd, bool interleaved, hipStream_t st) {
    if (dtype == DSW_BF16 && Q == 8) return rot_launch<bf16_t, 8, 1>(a, bwd, interleaved, st);
    DSW_DISPATCH_DTYPE(dtype, T, {
        if (Q == 4) return rot_launch<T, 4, 1>(a, bwd, interleaved, st);
        if (Q == 2) return rot_launch<T, 2, rot_units_per_lane(2)>(a, bwd, interleaved, st);
        return rot_launch<T, 1, rot_units_per_lane(1)>(a, bwd, interleaved, st);
    });
    return DSW_OK;
}

}  // namespace dsw

using namespace dsw;

extern "C" int dsw_qk_norm_rotary_fwd(const void *q, const dsw_strides *sq, const void *k, const dsw_strides *sk, int dtype, int B,
                                      int L, int Hq, int Hkv, int D, const float *wq, const float *wk, float eps, const float *freqs,
                                      int axes, int pairs, const void *pos, int pos_bytes, long long pos_batch, int interleaved, void *oq,
                                      const dsw_strides *soq, void *ok, const dsw_strides *sok, void *stream) {
    DSW_REQUIRE(sq && sk && soq && sok, "dsw_qk_norm_rotary_fwd: null strides");
    RotArgs a = {};
    a.x[0] = {q, *sq}, a.x[1] = {k, *sk}, a.y[0] = {oq, *soq}, a.y[1] = {ok, *sok};
    a.w[0] = wq, a.w[1] = wk, a.freqs = freqs, a.pos = pos, a.pos_bytes = pos_bytes, a.pos_batch = pos_batch;
    a.L = L, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.axes = axes, a.pairs = pairs, a.eps = eps;
    int Q = 1;
    const int rc = rot_check("dsw_qk_norm_rotary_fwd", a, dtype, B, false, Q);
    if (rc || a.tokens == 0 || Hq + Hkv == 0) return rc;
    return rot_dispatch(a, dtype, Q, false, interleaved != 0, as_stream(stream));
}

extern "C" int dsw_qk_norm_rotary_blocks(int dtype, int B, int L, int Hq, int Hkv, int D, int axes, int pairs) {
    const long long tokens = (long long)B * L;
    if (B < 0 || L < 0 || tokens >= (1LL << 31) || Hq < 0 || Hkv < 0 || (long long)Hq + Hkv > 4096 || D < 1 || D > ROT_MAX_D || axes < 0 ||
        pairs < 0 || 2LL * axes * pairs > D)
        return 0;
    const int tile = rot_tile(tokens, Hq + Hkv, D, axes * pairs, dtype, true);
    const long long tiles = (tokens + tile - 1) / tile;
    return (int)(tiles < ROT_BWD_BLOCKS ? tiles : ROT_BWD_BLOCKS);
}

extern "C" int dsw_qk_norm_rotary_bwd(const void *q, const dsw_strides *sq, const void *k, const dsw_strides *sk, const void *dyq,
                                      const dsw_strides *sdyq, const void *dyk, const dsw_strides *sdyk, int dtype, int B, int L,
                                      int Hq, int Hkv, int D, const float *wq, const float *wk, float eps, const float *freqs,
                                      int axes, int pairs, const void *pos, int pos_bytes, long long pos_batch, int interleaved, void *dq,
                                      const dsw_strides *sdq, void *dk, const dsw_strides *sdk, float *partial, float *dw, void *stream) {
    DSW_REQUIRE(sq && sk && sdyq && sdyk && sdq && sdk, "dsw_qk_norm_rotary_bwd: null strides");
    RotArgs a = {};
    a.x[0] = {q, *sq}, a.x[1] = {k, *sk}, a.dy[0] = {dyq, *sdyq}, a.dy[1] = {dyk, *sdyk}, a.y[0] = {dq, *sdq}, a.y[1] = {dk, *sdk};
    a.w[0] = wq, a.w[1] = wk, a.freqs = freqs, a.pos = pos, a.pos_bytes = pos_bytes, a.pos_batch = pos_batch, a.partial = partial;
    a.L = L, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.axes = axes, a.pairs = pairs, a.eps = eps;
    int Q = 1;
    int rc = rot_check("dsw_qk_norm_rotary_bwd", a, dtype, B, true, Q);
    DSW_REQUIRE((partial == nullptr) == (dw == nullptr), "dsw_qk_norm_rotary_bwd: partial and dw go together");
    if (rc || a.tokens == 0 || Hq + Hkv == 0) return rc;
    rc = rot_dispatch(a, dtype, Q, true, interleaved != 0, as_stream(stream));
    if (rc || dw == nullptr) return rc;
    const int rows = dsw_qk_norm_rotary_blocks(dtype, B, L, Hq, Hkv, D, axes, pairs);
    qk_norm_rotary_weights_kernel<<<dim3((2 * D + 31) / 32), 1024, 0, as_stream(stream)>>>(partial, rows, 2 * D, dw);
    return check_launch("dsw_qk_norm_rotary_bwd (weights)");
}
