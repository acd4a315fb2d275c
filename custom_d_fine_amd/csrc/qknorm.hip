// A2 / A6 - norms of queries and keys for each head, with the position rotation in the same pass, forward and backward.
//
// The token streams' attention (src/d_fine/arch/hybrid_encoder.py:243-290, src/d_fine/arch/dfine_decoder.py:200,233-255) scores q k^T as the
// projection leaves them; this is the step in between for a block that norms each head's query and key and rotates them by the token's position.
//   x: the D channels of one head of one token.  i = rsqrt(mean x^2 + eps), n = x i w;  pair (a, b) of the first R channels - halves (j, j + R/2) or
//   neighbours (2j, 2j + 1) - y_a = n_a c - n_b s, y_b = n_b c + n_a s with the token's row of the cosine / sine table; channels past R pass.
//   backward: dn_a = dy_a c + dy_b s, dn_b = dy_b c - dy_a s;  dw = sum dn x i;  dx = i (w dn - x i mean(x i w dn)).
// Bound: HBM (one read and one write of q and k forward, two reads and one write backward; ~10 vector instructions per element).
// A lane holds V consecutive channels of a head (one 16-byte load; 8-byte ones in 16 bits where half of R is no multiple of 8), the lanes of a head sit
// next to each other (a power of two of them), and a wave walks through the heads of its tokens with the table row and the weights in registers, so the
// table - 4 bytes per channel against 2 of data - is read once per token and not once per head.  The partner of a pair comes from its lane as raw
// storage (a shuffle of 16 bytes) and is normed again here: cheaper than exchanging the 32-bit results.
// Measured: 4 x 8192 tokens of 32 + 8 heads of 128 channels, bf16, forward 145 - 165 us (671 MB, 4.1 - 4.6 TB/s; a large copy reaches 4.9), backward 199 - 202 us (1007 MB,
// 5.0 TB/s) and 5 us for the weights' sums; 32 x 492 tokens of 8 + 8 heads of 32 channels 13 - 16, 17 - 18 and 4 us (32 MB, 48 MB); 16 x 900 tokens of 16 + 16 heads of 24
// channels in fp32 20 - 22, 29 and 4 us (88 MB, 133 MB); one token each of 16 sequences 4.5 us (a launch).
// All arithmetic is in 32 bits; the one rounding is the store.  The weight gradients leave as one partial row per workgroup, added up in order.
#include "common.h"

namespace dfine {

constexpr int kQkThreads = 256;

struct QkNormArgs {
    const void *x[2], *dy[2];             // q, k [B, L, heads, D]
    void *y[2];                           // forward: results; backward: dx
    const void *w[2];                     // [D] or null
    const float *cosv, *sinv;             // [T, R / 2]
    const void *pos;                      // [B or 1, L] or null: the token's index
    float *part;                          // backward: [grid][2][D]
    int64_t xs[2][3], ds[2][3];           // strides (batch, token, head) of x and dy in elements; y is contiguous
    int64_t pos_b;
    int heads[2], B, L, D, R, T, pos64, wbf16[2], wvec[2], paired;
    int lpr, hs, hchunk;                  // lanes per head, heads side by side, heads per workgroup column
    float eps;
};

template <typename T, int V> struct QkVec;
template <> struct QkVec<uint16_t, 8> { uint32_t r[4]; };
template <> struct QkVec<uint16_t, 4> { uint32_t r[2]; };
template <> struct QkVec<float, 4> { uint32_t r[4]; };

template <typename T, int V> __device__ __forceinline__ QkVec<T, V> qk_load(const T *p) {
    QkVec<T, V> v;
    if constexpr (sizeof(v) == 16) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        v.r[0] = u.x; v.r[1] = u.y; v.r[2] = u.z; v.r[3] = u.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        v.r[0] = u.x; v.r[1] = u.y;
    }
    return v;
}
template <typename T, int V> __device__ __forceinline__ void qk_unpack(const QkVec<T, V> &v, float *f) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) { f[2 * j] = __uint_as_float(v.r[j] << 16); f[2 * j + 1] = __uint_as_float(v.r[j] & 0xffff0000u); }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = __uint_as_float(v.r[j]);
    }
}
template <typename T, int V> __device__ __forceinline__ void qk_store(T *p, const float *f) {
    if constexpr (sizeof(T) == 2) {
        uint32_t r[V / 2];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) r[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
        if constexpr (V == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(r[0], r[1], r[2], r[3]);
        else *reinterpret_cast<uint2 *>(p) = make_uint2(r[0], r[1]);
    } else {
        *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
}
template <typename T, int V> __device__ __forceinline__ QkVec<T, V> qk_from_lane(const QkVec<T, V> &v, int lane) {
    QkVec<T, V> o;
#pragma unroll
    for (int j = 0; j < (int)(sizeof(v.r) / 4); ++j) o.r[j] = (uint32_t)__shfl((int)v.r[j], lane);
    return o;
}

// sum over the lpr (a power of two) neighbouring lanes of a head; up to 16 lanes inside the vector unit (DPP), wider through the shuffle network
__device__ __forceinline__ float qk_row_sum(float v, int lpr) {
#define QK_DPP(ctrl) __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
    if (lpr > 1) v += QK_DPP(0xB1);       // lane ^ 1
    if (lpr > 2) v += QK_DPP(0x4E);       // lane ^ 2
    if (lpr > 4) v += QK_DPP(0x141);      // mirrored in 8: the other group of 4
    if (lpr > 8) v += QK_DPP(0x140);      // mirrored in 16: the other group of 8
#undef QK_DPP
    if (lpr > 16) v += __shfl_xor(v, 16);
    if (lpr > 32) v += __shfl_xor(v, 32);
    return v;
}

// V weights from channel e on (0 past D; 1 without weights): one or two 16-byte loads where the pointer allows it
template <int V> __device__ __forceinline__ void qk_weights(const void *w, int bf16, bool vec, int e, int D, float *f) {
    if (!w || e >= D || e < 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = e >= D || e < 0 ? 0.f : 1.f;
    } else if (vec && bf16) {
        const uint2 *p = reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(w) + e);
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const uint2 u = p[j / 4];
            f[j] = __uint_as_float(u.x << 16); f[j + 1] = __uint_as_float(u.x & 0xffff0000u);
            f[j + 2] = __uint_as_float(u.y << 16); f[j + 3] = __uint_as_float(u.y & 0xffff0000u);
        }
    } else if (vec) {
        const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(w) + e);
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const float4 u = p[j / 4];
            f[j] = u.x; f[j + 1] = u.y; f[j + 2] = u.z; f[j + 3] = u.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(w)[e + j]) : reinterpret_cast<const float *>(w)[e + j];
    }
}

// grid.x: workgroups over tokens (strided), grid.y: chunks of heads
template <typename T, int V, bool BWD>
__global__ __launch_bounds__(kQkThreads) void qk_norm_rotate_kernel(const QkNormArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lpr = a.lpr, slot = lane / lpr, li = lane & (lpr - 1);
    const int hs = a.hs, ts = 64 / (lpr * hs), h0 = slot & (hs - 1), t0 = slot / hs;
    const int e = li * V, half = a.R >> 1;
    const bool live = e < a.D;
    // role in the rotation: the channels' column in the table, the partner's lane, the sign of the partner's term (0: passes through)
    int tcol = 0, plane = lane;
    float sign = 0.f;
    if (!a.paired && e < a.R) {
        const bool low = e < half;
        tcol = low ? e : e - half;
        plane = low ? lane + half / V : lane - half / V;
        sign = low ? -1.f : 1.f;
    } else if (a.paired && e < a.R) {
        tcol = e >> 1;
        sign = 1.f;
    }
    const bool turns = sign != 0.f;
    float w[2][V], wp[2][V];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (a.heads[s] == 0) continue;
        qk_weights<V>(a.w[s], a.wbf16[s], a.wvec[s], e, a.D, w[s]);
        if (!a.paired && !BWD) qk_weights<V>(a.w[s], a.wbf16[s], a.wvec[s], e + (plane - lane) * V, a.D, wp[s]);
    }
    float dw[2][V];
#pragma unroll
    for (int j = 0; j < V; ++j) dw[0][j] = dw[1][j] = 0.f;

    const int tokens = a.B * a.L;                                  // (host: fewer than 2^31 less the largest step)
    const float inv_d = 1.f / (float)a.D;
    const int64_t step = (int64_t)gridDim.x * (kQkThreads / 64) * ts;
    for (int64_t tok0 = ((int64_t)blockIdx.x * (kQkThreads / 64) + wave) * ts; tok0 < tokens; tok0 += step) {
        const int tok = (int)tok0 + t0;
        const bool tlive = tok < tokens;
        const int b = tlive ? tok / a.L : 0, l = tlive ? tok - b * a.L : 0;
        float c[V], s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) { c[j] = 1.f; s[j] = 0.f; }
        if (turns && tlive) {
            int64_t p = l;
            if (a.pos) p = a.pos64 ? reinterpret_cast<const int64_t *>(a.pos)[b * a.pos_b + l] : (int64_t)reinterpret_cast<const int *>(a.pos)[b * a.pos_b + l];
            const bool inside = p >= 0 && p < a.T;                 // a position outside the table: not a number, never a read outside it
            const float *cr = a.cosv + (inside ? p : 0) * half + tcol, *sr = a.sinv + (inside ? p : 0) * half + tcol;
            const float bad = __int_as_float(0x7fc00000);
            if (a.paired) {                                        // (rows of R / 2 floats, R a multiple of 8: 8-byte loads are on their border)
#pragma unroll
                for (int j = 0; j < V / 2; j += 2) {
                    const float2 cc = *reinterpret_cast<const float2 *>(cr + j), ss = *reinterpret_cast<const float2 *>(sr + j);
                    c[2 * j] = c[2 * j + 1] = cc.x; c[2 * j + 2] = c[2 * j + 3] = cc.y;
                    s[2 * j] = s[2 * j + 1] = ss.x; s[2 * j + 2] = s[2 * j + 3] = ss.y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const float4 cc = *reinterpret_cast<const float4 *>(cr + j), ss = *reinterpret_cast<const float4 *>(sr + j);
                    c[j] = cc.x; c[j + 1] = cc.y; c[j + 2] = cc.z; c[j + 3] = cc.w;
                    s[j] = ss.x; s[j + 1] = ss.y; s[j + 2] = ss.z; s[j + 3] = ss.w;
                }
            }
            if (!inside) {
#pragma unroll
                for (int j = 0; j < V; ++j) c[j] = s[j] = bad;
            }
        }
#pragma unroll
        for (int set = 0; set < 2; ++set) {                        // queries, then keys
            const int H = a.heads[set], hend = min(H, (int)(blockIdx.y + 1) * a.hchunk);
            const T *xb = reinterpret_cast<const T *>(a.x[set]) + (int64_t)b * a.xs[set][0] + (int64_t)l * a.xs[set][1] + e;
            const T *db = reinterpret_cast<const T *>(a.dy[set]) + (int64_t)b * a.ds[set][0] + (int64_t)l * a.ds[set][1] + e;
            T *yb = reinterpret_cast<T *>(a.y[set]) + (int64_t)tok * H * a.D + e;
            for (int hb = blockIdx.y * a.hchunk; hb < hend; hb += hs) {
                const int h = hb + h0;
                const bool ok = live && tlive && h < hend;
                QkVec<T, V> xr{}, gr{};
                if (ok) xr = qk_load<T, V>(xb + (int64_t)h * a.xs[set][2]);
                if (BWD && ok) gr = qk_load<T, V>(db + (int64_t)h * a.ds[set][2]);
                float x[V], out[V];
                qk_unpack<T, V>(xr, x);
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < V; ++j) ss += x[j] * x[j];
                const float i = rsqrtf(qk_row_sum(ss, lpr) * inv_d + a.eps);
                if (!BWD) {
                    float n[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) n[j] = x[j] * i * w[set][j];
                    if (a.paired) {
#pragma unroll
                        for (int j = 0; j < V; j += 2) {
                            out[j] = turns ? n[j] * c[j] - n[j + 1] * s[j] : n[j];       // (not n 1 - n' 0: a channel that passes takes nothing of its neighbour)
                            out[j + 1] = turns ? n[j + 1] * c[j] + n[j] * s[j] : n[j + 1];
                        }
                    } else {
                        float xp[V];
                        qk_unpack<T, V>(qk_from_lane<T, V>(xr, plane), xp);
#pragma unroll
                        for (int j = 0; j < V; ++j) out[j] = turns ? n[j] * c[j] + sign * (xp[j] * i * wp[set][j]) * s[j] : n[j];
                    }
                } else {
                    float g[V], dn[V];
                    qk_unpack<T, V>(gr, g);
                    if (a.paired) {
#pragma unroll
                        for (int j = 0; j < V; j += 2) {
                            dn[j] = turns ? g[j] * c[j] + g[j + 1] * s[j] : g[j];
                            dn[j + 1] = turns ? g[j + 1] * c[j] - g[j] * s[j] : g[j + 1];
                        }
                    } else {
                        float gp[V];
                        qk_unpack<T, V>(qk_from_lane<T, V>(gr, plane), gp);
#pragma unroll
                        for (int j = 0; j < V; ++j) dn[j] = turns ? g[j] * c[j] - sign * gp[j] * s[j] : g[j];
                    }
                    float dot = 0.f;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        x[j] *= i;                                 // x i
                        if (ok) dw[set][j] += dn[j] * x[j];
                        dn[j] *= w[set][j];
                        dot += dn[j] * x[j];
                    }
                    dot = qk_row_sum(dot, lpr) * inv_d;
#pragma unroll
                    for (int j = 0; j < V; ++j) out[j] = i * (dn[j] - x[j] * dot);
                }
                if (ok) qk_store<T, V>(yb + (int64_t)h * a.D, out);
            }
        }
    }
    if (BWD) {                                                     // this workgroup's weight gradients: lanes of the same channels, then waves, in order
        __shared__ float sum[2][4][256];
#pragma unroll
        for (int set = 0; set < 2; ++set)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float v = dw[set][j];
                for (int d = lpr; d < 64; d <<= 1) v += __shfl_xor(v, d);
                if (slot == 0 && e + j < 256) sum[set][wave][e + j] = v;
            }
        __syncthreads();
        float *p = a.part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.D;
        for (int i = threadIdx.x; i < 2 * a.D; i += kQkThreads) {
            const int set = i >= a.D, ch = i - set * a.D;
            p[i] = (sum[set][0][ch] + sum[set][1][ch]) + (sum[set][2][ch] + sum[set][3][ch]);
        }
    }
}

// dw[set][ch] = sum over the partial rows: 32 channels per workgroup, the rows in 32 interleaved runs, 8 loads in flight
__global__ __launch_bounds__(1024) void qk_dw_kernel(const float *__restrict__ part, void *dwq, void *dwk, int qbf16, int kbf16, int rows, int D) {
    __shared__ float s[32][33];
    const int col = threadIdx.x & 31, run = threadIdx.x >> 5, i = blockIdx.x * 32 + col;
    float v = 0.f;
    if (i < 2 * D) {
#pragma unroll 8
        for (int r = run; r < rows; r += 32) v += part[(int64_t)r * 2 * D + i];
    }
    s[run][col] = v;
    __syncthreads();
    if (run || i >= 2 * D) return;
#pragma unroll
    for (int r = 1; r < 32; ++r) v += s[r][col];
    const bool k = i >= D;
    void *dst = k ? dwk : dwq;
    if (!dst) return;
    const int ch = k ? i - D : i;
    if (k ? kbf16 : qbf16) reinterpret_cast<uint16_t *>(dst)[ch] = f32_to_bf16(v);
    else reinterpret_cast<float *>(dst)[ch] = v;
}

}  // namespace dfine

using namespace dfine;

extern "C" {

// shape: see include/dfine_hip.h
static int qk_norm_setup(QkNormArgs &a, const int64_t *s, const float *cosv, const float *sinv, const void *pos, float eps, int *vec, int *gx, int *gy,
                         bool bwd) {
    const int64_t B = s[0], L = s[1], Hq = s[2], Hk = s[3], D = s[4], R = s[5], T = s[6], dt = s[7];
    if (B < 0 || L < 0 || Hq < 0 || Hk < 0 || B > 0x7fffffff || L > 0x7fffffff || B * L > 0x7fffffff - 0x10000 || Hq > 4096 || Hk > 4096 || D < 8 || D > 256 || D % 8 || R < 0 || R > D || R % 8 ||
        (dt != 0 && dt != 1))
        return DFINE_E_BADARG;
    if (R && (!cosv || !sinv || ((uintptr_t)cosv | (uintptr_t)sinv) & 15 || T < 1 || (!pos && T < L))) return DFINE_E_BADARG;
    a.B = (int)B; a.L = (int)L; a.D = (int)D; a.R = (int)R; a.T = (int)(T > 0x7fffffff ? 0x7fffffff : T);
    a.heads[0] = (int)Hq; a.heads[1] = (int)Hk;
    a.paired = s[8] != 0; a.pos64 = s[9] != 0; a.pos_b = s[10];
    a.wbf16[0] = s[11] != 0; a.wbf16[1] = s[12] != 0;
    a.cosv = cosv; a.sinv = sinv; a.pos = pos; a.eps = eps;
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 3; ++j) { a.xs[i][j] = s[13 + 3 * i + j]; a.ds[i][j] = s[19 + 3 * i + j]; }
    const int V = dt == 0 ? 4 : (!a.paired && (R / 2) % 8) ? 4 : 8;
    *vec = V;
    int lpr = 1;
    while (lpr * V < D) lpr <<= 1;
    const int slots = 64 / lpr, hmax = (int)(Hq > Hk ? Hq : Hk);
    int hs = 1;
    while (hs < slots && hs < hmax) hs <<= 1;
    a.lpr = lpr; a.hs = hs;
    const int64_t per_wave = slots / hs, waves = (B * L + per_wave - 1) / per_wave, groups = (waves + 3) / 4;
    // few tokens: the heads go over workgroups too, down to one load per lane; many: a wave takes all heads of its tokens (one read of the table row).
    // All heads in a wave / up to 1024 / up to 4096 workgroups: 16 tokens of 32 heads 6.1 / 4.7 / 4.6 us, one token of 64 heads 14.5 / 4.8 / 4.8, 160 tokens of 32
    // heads 11.5 / 6.0 / 6.0, 16 x 900 tokens of 16 heads (fp32) 21 / 21 / 24.
    int chunk = hmax;
    while (chunk > hs && groups * ((hmax + chunk - 1) / chunk) < 1024) chunk = (chunk / 2 + hs - 1) / hs * hs;
    a.hchunk = chunk < hs ? hs : chunk;
    *gy = hmax ? (hmax + a.hchunk - 1) / a.hchunk : 1;
    // backward: at most 1024 partial rows of weight gradients.  512 / 1024 / 2048 rows: 267 / 200 / 201 us and 4.9 / 4.9 / 8.0 for their sums at 4 x 8192 tokens of
    // 40 heads, 20.6 / 17.8 / 24.1 and 3.8 / 3.8 / 6.2 at 32 x 492 of 16
    const int64_t most = bwd ? 1024 / (*gy < 1024 ? *gy : 1024) : 65536;
    *gx = (int)(groups < most ? groups : most);
    return DFINE_OK;
}

static void qk_norm_weights(QkNormArgs &a, const void *wq, const void *wk) {
    a.w[0] = wq; a.w[1] = wk;
    for (int i = 0; i < 2; ++i) a.wvec[i] = ((uintptr_t)a.w[i] & (a.wbf16[i] ? 7 : 15)) == 0;
}

int64_t dfine_qk_norm_rotate_ws_floats(const int64_t *shape) {
    QkNormArgs a{};
    int vec, gx, gy;
    if (!shape || qk_norm_setup(a, shape, (const float *)16, (const float *)16, (const void *)1, 0.f, &vec, &gx, &gy, true)) return -1;
    return (int64_t)gx * gy * 2 * a.D;
}

#define QK_LAUNCH(BWD_)                                                                                                                     \
    if (shape[7] == 0) hipLaunchKernelGGL((qk_norm_rotate_kernel<float, 4, BWD_>), dim3(gx, gy), dim3(kQkThreads), 0, (hipStream_t)stream, a);   \
    else if (vec == 8) hipLaunchKernelGGL((qk_norm_rotate_kernel<uint16_t, 8, BWD_>), dim3(gx, gy), dim3(kQkThreads), 0, (hipStream_t)stream, a); \
    else hipLaunchKernelGGL((qk_norm_rotate_kernel<uint16_t, 4, BWD_>), dim3(gx, gy), dim3(kQkThreads), 0, (hipStream_t)stream, a);

int dfine_qk_norm_rotate_fwd(const void *q, const void *k, const void *wq, const void *wk, const float *cosv, const float *sinv, const void *pos,
                             void *yq, void *yk, const int64_t *shape, float eps, void *stream) {
    if (!shape) return DFINE_E_BADARG;
    QkNormArgs a{};
    int vec, gx, gy;
    if (int e = qk_norm_setup(a, shape, cosv, sinv, pos, eps, &vec, &gx, &gy, false)) return e;
    if (shape[0] == 0 || shape[1] == 0 || shape[2] + shape[3] == 0) return DFINE_OK;
    if ((a.heads[0] && (!q || !yq)) || (a.heads[1] && (!k || !yk))) return DFINE_E_BADARG;
    a.x[0] = q; a.x[1] = k; a.y[0] = yq; a.y[1] = yk;
    qk_norm_weights(a, wq, wk);
    QK_LAUNCH(false)
    return check_launch();
}

int dfine_qk_norm_rotate_bwd(const void *q, const void *k, const void *wq, const void *wk, const float *cosv, const float *sinv, const void *pos,
                             const void *dyq, const void *dyk, void *dq, void *dk, void *dwq, void *dwk, float *ws, const int64_t *shape, float eps,
                             void *stream) {
    if (!shape) return DFINE_E_BADARG;
    QkNormArgs a{};
    int vec, gx, gy;
    if (int e = qk_norm_setup(a, shape, cosv, sinv, pos, eps, &vec, &gx, &gy, true)) return e;
    if (!ws) return DFINE_E_BADARG;
    int rows = gx * gy;
    if (shape[0] == 0 || shape[1] == 0 || shape[2] + shape[3] == 0) {
        rows = 0;                                                   // no rows: the weights' gradients are zero
    } else {
        if ((a.heads[0] && (!q || !dyq || !dq)) || (a.heads[1] && (!k || !dyk || !dk))) return DFINE_E_BADARG;
        a.x[0] = q; a.x[1] = k; a.dy[0] = dyq; a.dy[1] = dyk; a.y[0] = dq; a.y[1] = dk; a.part = ws;
        qk_norm_weights(a, wq, wk);
        QK_LAUNCH(true)
        if (int e = check_launch()) return e;
    }
    if (!dwq && !dwk) return DFINE_OK;
    hipLaunchKernelGGL(qk_dw_kernel, dim3((2 * a.D + 31) / 32), dim3(1024), 0, (hipStream_t)stream, (const float *)ws, dwq, dwk, a.wbf16[0], a.wbf16[1], rows,
                       a.D);
    return check_launch();
}
#undef QK_LAUNCH

}  // extern "C"
