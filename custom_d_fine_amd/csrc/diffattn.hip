// A2 / A6 - differential attention of the token streams, forward and backward.
//
// Next to the softmax attention of attn.hip (src/d_fine/arch/hybrid_encoder.py:243-290, src/d_fine/arch/dfine_decoder.py:200,233-255): every head
// has two query and two key vectors per token, and reads its values through the DIFFERENCE of two softmax maps,
//   A_t = softmax(scale q_t k_t^T + mask), t = 0, 1 (a row that sees no key: 0),   U = A_0 V - l_h A_1 V,
//   l_h = exp(x0 . x1) - exp(x2 . x3) + init (the head's learned vectors),          Y = (1 - init) norm(U) g   (or Y = U without a norm weight),
// norm(U) = U r, r = rsqrt(mean U^2 + eps) over the head's dv channels.  Backward, with D_t = dU . (A_t V):
//   dU = (1 - init) r (g dY - U r^2 mean(U g dY)), dP = dU V^T, dS_0 = A_0 (dP - D_0), dS_1 = -l A_1 (dP - D_1),
//   dq_t = scale dS_t k_t, dk_t = scale dS_t^T q_t, dV = (A_0 - l A_1)^T dU, dl = - sum D_1, dx0 = dl exp(x0 . x1) x1 and its like.
//
// Rows.  The G = H / Hk query heads of a shared key head read the same keys: their rows (query i, head g) form one list r = i G + g, and a wave takes 32
// rows of it.  One token of G heads therefore fills G columns of one matrix tile, and the gradients of a shared key head add up in registers.
// Products (32 x 32 matrix instructions).  Forward and dQ: S^T = K Q^T puts ONE row of the list (a lane's column) against 16 keys per lane and tile in the
// order 8 a + 4 h + b (h = lane / 32, a and b the register), which is the order the transposed read of V delivers the second product's other operand in, so
// the probabilities go from registers to the matrix unit as they are.  dK and dV: S = Q K^T, one KEY per lane, the same way with dU and Q transposed.
// LDS tiles hold rows of 16-byte units, unit u of row r at u ^ f(r) (da_swz): both kinds of reads fall on different banks without padding.
// Types: bf16 (v_mfma_f32_32x32x16_bf16; probabilities and dS are rounded to bf16 for the second products, as the values they meet are) and fp32
// (v_mfma_f32_32x32x2_f32).  Scores, softmax statistics, sums and norms are 32-bit.  Head dims up to 64 with values up to 128, multiples of 8, run on the
// next of three sizes with zero-filled tiles.
#include "common.h"

namespace dfine {

typedef __attribute__((ext_vector_type(16))) float da_f16v;
typedef __attribute__((ext_vector_type(8))) __bf16 da_bf16x8;
typedef short da_tr4 __attribute__((ext_vector_type(4)));
typedef short da_tr8 __attribute__((ext_vector_type(8)));

constexpr int kDaThreads = 256;
constexpr int kDaSplitWgs = 256, kDaRunKeys = 256, kDaOneRun = 1024, kDaManyRows = 256;      // diff_attn_splits

struct DiffArgs {
    const void *q, *k, *v;                      // [B, N, H, 2, d], [B, M, Hk, 2, d], [B, M, Hk, dv]
    const void *lam, *weight;                   // [4, H or 1, d], [dv] or null
    const uint64_t *rowbits, *colbits, *some;   // mask forms (1 = may attend): [Bm][N][M64], [Bm][M][N64], any of 64 queries [Bm][N64][M64]; null: no mask
    const uint8_t *tiles;                       // [Bm][N64][M64] 0 free, 1 mixed, 2 blocked
    const int *kvlen, *qstart_dev;              // [B] or null
    void *out, *o2;                             // [B, N, H, dv]; o2 = W and u = U (null: not kept) are read by the backward pass
    float *u;
    float *stats;                               // [4][B, H, N]: lse of the two maps in the exp2 domain (+inf: an empty row), r, beta
    int64_t qs[4], ks[4], vs[3];                // strides (batch, token, head, map)
    int64_t mask_b;                             // 0: one mask for the batch
    int64_t qstart;
    uint32_t g_mul;                             // n / G = umulhi(2 n, g_mul) >> g_shift for n < 2^31
    int g_shift;
    int B, N, M, H, Hk, G, d, dv, causal, lam_heads, lam_bf16, w_bf16;
    float scale, scale_log2e, init, post, eps;  // post = 1 - init with a norm weight
    // backward
    const void *dy;
    int64_t dys[3];
    void *du, *dq, *dk, *dvv;
    float *rowstat;                             // [4][B, H, N]: -lse_0 / c, -(lse_1 - log2 |l|) / c, -D_0, sign(l) (D_1 - D_0), c = scale_log2e (diff_attn_prep_kernel)
    float *lpart, *wpart;                       // per workgroup of the first kernel: sum of D_1, sums of dg
    float *kvpart;                              // dK | dV sums of each run of the rows, fp32 [runs][B, M, Hk, 2 d + dv] (null: one run)
    int kvruns;
};

template <typename T> struct Da;
template <> struct Da<uint16_t> {
    static constexpr int KPF = 16;              // contraction length of one fragment (16 bytes per lane)
    static __device__ __forceinline__ da_f16v mma(uint4 a, uint4 b, da_f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(da_bf16x8, a), __builtin_bit_cast(da_bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Da<float> {
    static constexpr int KPF = 8;
    static __device__ __forceinline__ da_f16v mma(uint4 a, uint4 b, da_f16v c) {
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
    }
};

// sizes of one instantiation: DK channels per map, 2 DK value channels
template <typename T, int DK> struct DaCfg {
    static constexpr int ES = sizeof(T), DV = 2 * DK, ROWB = 2 * DK * ES, U = ROWB / 16, NF = DK / Da<T>::KPF, NFV = DV / Da<T>::KPF, MT = DV / 32 ? DV / 32 : 1,
                         MTK = DK / 32 ? DK / 32 : 1, FPT = 32 / Da<T>::KPF;      // fragments per 32 keys
    static_assert(DV % 32 == 0, "a value tile is 32 channels");
};

// f(row): a b128 read serves 16 lanes at a time (rows 16 apart in some order, one u), a transposed read 32 lanes (4 rows from a multiple of 4 on, 4 units from a
// multiple of 4 on): f takes all values over 16 rows and, in its bits from 2 on, over 4 (256 bytes = all banks; rows shorter than that share them).
// Measured per wave: b128 4 cycles, transposed 3 (plain rows of 256 bytes: 64 and 8; u ^ 2 (row % 8): 8 and 4).  fp32 reads its transposed operand in 4-byte
// pieces, 32 columns of rows 4 apart: there bit 2 of the row goes on top.
template <typename T, int U> __device__ __forceinline__ int da_swz(int row) {
    if (sizeof(T) == 4) return U >= 16 ? ((row >> 2) & 1) << 3 | (row & 3) << 1 | ((row >> 3) & 1) : (row >> 1) & 7;
    return U >= 16 ? (row & 3) << 2 | ((row >> 2) & 3) : U == 8 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : (row >> 2) & 3;
}

typedef __attribute__((ext_vector_type(4))) uint32_t da_u4v;
typedef __attribute__((address_space(3))) const da_u4v *da_lds_u4;
typedef __attribute__((address_space(3))) const uint32_t *da_lds_u1;

// A lane's way through a tile of rows of U units (byte addresses in LDS; tiles start on 512-byte borders): everything that depends on the lane is one register
// per kind of read, the fragment only flips bits of it (below 512: the tiles' own borders)
template <typename T, int DK> struct DaLane {
    using C = DaCfg<T, DK>;
    uint32_t row, tr[sizeof(T) == 2 ? 1 : 4];
    __device__ __forceinline__ void init(int lane) {
        const int h = lane >> 5, l32 = lane & 31;
        row = l32 * C::ROWB + ((h ^ da_swz<T, C::U>(l32)) << 4);
        if constexpr (sizeof(T) == 2) {
            const int i16 = lane & 15, r = 4 * h + (i16 >> 2), u = ((lane >> 4) & 1) * 2 + ((i16 & 3) >> 1);
            tr[0] = r * C::ROWB + ((u ^ da_swz<T, C::U>(r)) << 4) + 8 * (i16 & 1);
        } else {
#pragma unroll
            for (int b = 0; b < 4; ++b) tr[b] = (4 * h + b) * C::ROWB + (((l32 >> 2) ^ da_swz<T, C::U>(4 * h + b)) << 4) + (l32 & 3) * 4;
        }
    }
    // row-major operand: row lane % 32 of the 32 rows at `tile`, fragment f
    __device__ __forceinline__ uint4 frag(uint32_t tile, int f) const { return __builtin_bit_cast(uint4, *(da_lds_u4)(uintptr_t)((tile + row) ^ (f << 5))); }
    // transposed operand: contraction over rows KPF f .. of the 32 rows at `tile` in the order 8 a + 4 h + b, column 32 x + lane % 32
    __device__ __forceinline__ uint4 frag_tr(uint32_t tile, int f, int x) const {
        if constexpr (sizeof(T) == 2) {
            const uint32_t p = ((tile + tr[0]) ^ (x << 6)) + f * 16 * C::ROWB, q = ((tile + tr[0]) ^ (x << 6) ^ 32) + (f * 16 + 8) * C::ROWB;
            const da_tr4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((da_tr4 __attribute__((address_space(3))) *)(uintptr_t)p);
            const da_tr4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((da_tr4 __attribute__((address_space(3))) *)(uintptr_t)q);
            return __builtin_bit_cast(uint4, (da_tr8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            uint32_t r[4];
#pragma unroll
            for (int b = 0; b < 4; ++b)
                r[b] = *(da_lds_u1)(uintptr_t)(((tile + tr[b]) ^ (x << 7) ^ (C::U >= 16 && (f & 1) ? 16 : 0) ^ (C::U == 8 && (f & 1) ? 64 : 0)) + f * 8 * C::ROWB);
            return make_uint4(r[0], r[1], r[2], r[3]);
        }
    }
};

// N fragments through D registers in flight: rd(i) asks for fragment i, use(i, fragment) multiplies.  The order is held against the scheduler, which would
// ask for each fragment right in front of its product and wait out the LDS latency N times; vector instructions may move across.
template <int N, int D, class RD, class USE> __device__ __forceinline__ void da_ring(RD rd, USE use) {
    uint4 fr[D];
#pragma unroll
    for (int i = 0; i < D && i < N; ++i) fr[i] = rd(i);
    __builtin_amdgcn_sched_barrier(0x406);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        use(i, fr[i % D]);
        if (i + D < N) fr[i % D] = rd(i + D);
        __builtin_amdgcn_sched_barrier(0x406);
    }
}

// N products with the vector work of 16 elements between them: after product i the elements [16 i / N, 16 (i + 1) / N).  The matrix unit runs a product in 32 cycles of
// which the wave issues for 4; vector work of the SAME wave that the products do not wait for fills the rest, and here it stands in that order.  fr: the first two
// fragments, asked for in front.
template <int N, class RD, class USE, class VEC> __device__ __forceinline__ void da_between(uint4 *fr, RD rd, USE use, VEC vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        use(i, fr[i & 1]);
        if (i + 2 < N) fr[i & 1] = rd(i + 2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 16 * i / N; r < 16 * (i + 1) / N; ++r) vec(r);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// -1 where bit `pos` of v is set, else 0 (assembly: written as an expression it becomes an and, a compare and a select for each use)
template <int POS> __device__ __forceinline__ uint32_t da_bit(uint32_t v) {
    uint32_t r;
    asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(r) : "v"(v), "n"(POS));
    return r;
}
// scores of keys (rows) that the lane's row (key) does not see: -inf
template <int R = 0> __device__ __forceinline__ void da_hide(da_f16v &s, uint32_t mine) {
    if constexpr (R < 16) {
        const uint32_t on = da_bit<8 * (R >> 2) + (R & 3)>(mine);
        s[R] = __uint_as_float((__float_as_uint(s[R]) & on) | (0xff800000u & ~on));
        da_hide<R + 1>(s, mine);
    }
}
// Two floats to bf16 as a conversion the compiler sees (common.h's pack_bf16x2 is inline assembly): it has to put two wait states between the
// conversion and a matrix instruction that reads it, which it does not do behind assembly.
typedef __attribute__((ext_vector_type(2))) float da_f2;
typedef __attribute__((ext_vector_type(2))) __bf16 da_bf2;
__device__ __forceinline__ uint32_t da_pk(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((da_f2){a, b}, da_bf2)); }

// fragment f of 32 values per lane pair (accumulator order) as a matrix operand
template <typename T> __device__ __forceinline__ uint4 da_pack(const da_f16v &p, int f) {
    if constexpr (sizeof(T) == 2)
        return make_uint4(da_pk(p[8 * f], p[8 * f + 1]), da_pk(p[8 * f + 2], p[8 * f + 3]), da_pk(p[8 * f + 4], p[8 * f + 5]),
                          da_pk(p[8 * f + 6], p[8 * f + 7]));
    else
        return make_uint4(__float_as_uint(p[4 * f]), __float_as_uint(p[4 * f + 1]), __float_as_uint(p[4 * f + 2]), __float_as_uint(p[4 * f + 3]));
}

__device__ __forceinline__ float da_exp2(float x) { return __builtin_amdgcn_exp2f(x); }     // arguments <= 0 or -inf: no range handling needed
__device__ __forceinline__ float da_load1(const void *p, int64_t i, int bf16) {
    return bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[i]) : reinterpret_cast<const float *>(p)[i];
}
template <typename T> __device__ __forceinline__ void da_store4(T *p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
    else *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
}
template <typename T> __device__ __forceinline__ float da_round(float v) { return sizeof(T) == 2 ? bf16_to_f32(f32_to_bf16(v)) : v; }
template <typename T> __device__ __forceinline__ void da_load4(const T *p, float *f) {
    if constexpr (sizeof(T) == 2) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
        f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
    } else {
        const float4 u = *reinterpret_cast<const float4 *>(p);
        f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
    }
}

__device__ __forceinline__ int da_div_g(const DiffArgs &a, int n) { return (int)(__umulhi(2u * (uint32_t)n, a.g_mul) >> a.g_shift); }

// sum over the 64 lanes, the same in every lane
__device__ __forceinline__ float da_wave_sum(float v) {
#define DA_DPP(ctrl) __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
    v += DA_DPP(0xB1);                          // lane ^ 1
    v += DA_DPP(0x4E);                          // lane ^ 2
    v += DA_DPP(0x141);                         // mirrored in 8
    v += DA_DPP(0x140);                         // mirrored in 16
#undef DA_DPP
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// exp(x0 . x1) and exp(x2 . x3) of a head, by a whole wave: one channel per lane
__device__ __forceinline__ float4 da_lambda_vectors(const DiffArgs &a, int h) {
    const int j = threadIdx.x & 63;
    const int64_t st = (int64_t)a.lam_heads * a.d, o = (a.lam_heads == 1 ? 0 : (int64_t)h * a.d) + j;
    if (j >= a.d) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.lam_bf16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(a.lam) + o;
        return make_float4(bf16_to_f32(p[0]), bf16_to_f32(p[st]), bf16_to_f32(p[2 * st]), bf16_to_f32(p[3 * st]));
    }
    const float *p = reinterpret_cast<const float *>(a.lam) + o;
    return make_float4(p[0], p[st], p[2 * st], p[3 * st]);
}
__device__ __forceinline__ void da_lambda_parts(const float4 &x, float &e1, float &e2) {
    e1 = expf(da_wave_sum(x.x * x.y));
    e2 = expf(da_wave_sum(x.z * x.w));
}
__device__ __forceinline__ float da_lambda(const DiffArgs &a, const float4 &x) {
    float e1, e2;
    da_lambda_parts(x, e1, e2);
    return e1 - e2 + a.init;
}
__device__ __forceinline__ float da_lambda(const DiffArgs &a, int h) { return da_lambda(a, da_lambda_vectors(a, h)); }
// (1 - init) g of N channels from c0 on (1 without a norm), channels from dv on 0: one test of the type, all loads at once
template <int N> __device__ __forceinline__ void da_weights(const DiffArgs &a, int c0, float *w) {
    if (!a.weight) {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = c0 + j < a.dv ? 1.f : 0.f;
    } else if (a.w_bf16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(a.weight) + c0;
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = c0 + j < a.dv ? bf16_to_f32(p[j]) * a.post : 0.f;
    } else {
        const float *p = reinterpret_cast<const float *>(a.weight) + c0;
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = c0 + j < a.dv ? p[j] * a.post : 0.f;
    }
}
// l of each lane's own head, for a wave whose rows start at w0: its rows' heads are min(G, 32) in a row (a whole wave calls this)
__device__ __forceinline__ float da_lambda_rows(const DiffArgs &a, int hk, int w0, int head) {
    if (a.lam_heads == 1) return da_lambda(a, 0);
    if (a.G == 1) return da_lambda(a, hk);
    const int g0 = w0 - da_div_g(a, w0) * a.G, n = min(a.G, 32);
    float lam = 0.f;
    for (int x = 0; x < n; ++x) {
        const int h = hk * a.G + (g0 + x) % a.G;
        const float l = da_lambda(a, h);
        if (h == head) lam = l;
    }
    return lam;
}

// keys that row i of batch b may look at end here
__device__ __forceinline__ int da_limit(const DiffArgs &a, int len, int64_t start, int i) {
    if (!a.causal) return len;
    const int64_t e = start + i + 1;
    return e < 0 ? 0 : e < len ? (int)e : len;
}
__device__ __forceinline__ int64_t da_start(const DiffArgs &a, int b) { return a.qstart_dev ? (int64_t)a.qstart_dev[b] : a.qstart; }
// keys of batch b that any of its queries may see: what lies behind is never read
__device__ __forceinline__ int da_len(const DiffArgs &a, int b) {
    int len = a.kvlen ? min(max(a.kvlen[b], 0), a.M) : a.M;
    if (a.causal) {
        const int64_t e = da_start(a, b) + a.N;
        len = e < 0 ? 0 : e < len ? (int)e : len;
    }
    return len;
}

// 16 bytes global -> LDS without registers; the LDS side is lane-linear from lds_addr (wave-uniform).  Inline assembly, waited for by hand (da_wait_copies,
// da_copies_done_barrier):
// behind the builtin the compiler waits for every copy in front of the next LDS read, which would end the overlap of copies and products.
__device__ __forceinline__ void da_copy16(const void *src, uint32_t lds_addr) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(src), "s"(lds_addr) : "memory");
}
template <int N> __device__ __forceinline__ void da_wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void da_copies_done_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// Makes the compiler wait for a loaded value HERE: it does not see the waits above, and would put its own in front of the value's first use in the loop -
// which is a wait for the copies that are on their way by then
__device__ __forceinline__ void da_pin(uint4 &v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
__device__ __forceinline__ void da_pin(float &v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void da_pin(uint32_t &v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void da_pin(uint64_t &v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void da_lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __attribute__((aligned(16))) uint32_t da_zero_page[4];            // what rows and channels that are not there are copied from

// One operand's way into LDS: `ROWS` rows of U units by NT threads (a workgroup or a wave), this thread's part
template <typename T, int DK, int ROWS, int NT> struct DaCopy {
    using C = DaCfg<T, DK>;
    static constexpr int J = ROWS * C::U / NT, STEP = NT / C::U, P = STEP >= 16 ? 1 : 16 / STEP;     // the swizzle repeats every 16 rows
    static_assert(J >= 1 && STEP >= 1 && J % P == 0, "");
    const T *at[P];                                     // row r0 (+ p STEP) of the block at hand, this thread's channels
    int64_t hop;                                        // P STEP rows, in elements
    uint32_t ok;                                        // bit p: the channels are there
    int r0;
    __device__ __forceinline__ void init(const T *src, int64_t ld, int64_t map, int nch, bool maps, int t) {
        r0 = t / C::U;
        ok = 0;
        hop = ld * (P * STEP);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int u = (t % C::U) ^ da_swz<T, C::U>(r0 + p * STEP), half = maps ? u / (C::U / 2) : 0;
            const int c = (maps ? u % (C::U / 2) : u) * (16 / C::ES);
            ok |= c < nch ? 1u << p : 0u;
            at[p] = src + (int64_t)(r0 + p * STEP) * ld + half * map + c;
        }
    }
    __device__ __forceinline__ void move(int64_t elements) {
#pragma unroll
        for (int p = 0; p < P; ++p) at[p] += elements;
    }
    // the block into the tile at lds (this wave's first byte); rows >= valid, rows whose live bit is 0 and channels that are not there become zeros.
    // rows: all ROWS rows are there and live; full: all channels are
    __device__ __forceinline__ void run(uint32_t lds, int valid, uint64_t live, bool rows, bool full) const {
        const T *p[P];
#pragma unroll
        for (int q = 0; q < P; ++q) p[q] = at[q];
        if (rows && full) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                da_copy16(p[j % P], __builtin_amdgcn_readfirstlane(lds + j * NT * 16));
                p[j % P] += hop;
            }
            return;
        }
        const T *zero = reinterpret_cast<const T *>(da_zero_page);
        uint32_t on = 0;                                // bit j: copy j is of a row and channels that are there
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int r = r0 + j * STEP;
            on |= ((ok >> (j % P)) & 1) && (rows || (r < valid && ((live >> r) & 1))) ? 1u << j : 0u;
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            da_copy16((on >> j) & 1 ? p[j % P] : zero, __builtin_amdgcn_readfirstlane(lds + j * NT * 16));
            p[j % P] += hop;
        }
    }
};

// The kernel's arguments read again: what a loop does not need is not held in scalar registers over it (held, it spills to vector registers and comes back lane by
// lane, eight instructions for each copy).
__device__ __forceinline__ const DiffArgs &da_again() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();    // (DiffArgs is the first argument of every kernel)
    asm volatile("" : "+s"(p));
    return *(const DiffArgs *)p;
}

__device__ __forceinline__ float da_other_half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float da_both_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// the rows of a wave: what the forward pass knows about the lane's row and the wave's range of queries
struct DaRows {
    int row, i, head, limit, lim_lo, lim_hi, q_lo, q_hi;           // lim_*: ends of the first and last query's keys; q_*: their 64-query tiles
    bool live, alive;                                         // this row / any row of the wave exists
};
__device__ __forceinline__ DaRows da_rows(const DiffArgs &a, int hk, int w0, int l32, int len, int64_t start) {
    DaRows w;
    const int R = a.N * a.G, wl = min(w0 + 31, R - 1);
    w.row = w0 + l32;
    w.live = w.row < R;
    w.alive = w0 < R;
    w.i = w.live ? da_div_g(a, w.row) : 0;
    w.head = hk * a.G + (w.live ? w.row - w.i * a.G : 0);
    w.limit = w.live ? da_limit(a, len, start, w.i) : 0;
    const int i_lo = w.alive ? da_div_g(a, w0) : 0, i_hi = w.alive ? da_div_g(a, wl) : 0;
    w.lim_lo = da_limit(a, len, start, i_lo);
    w.lim_hi = w.alive ? da_limit(a, len, start, i_hi) : 0;
    w.q_lo = i_lo >> 6; w.q_hi = i_hi >> 6;
    return w;
}
// What the mask says about tiles of 64 keys for the 64-query tiles qt0 .. qt1 of a workgroup and q_lo, q_hi of a wave: 64 tiles at a time as bit sets, one tile
// per lane, so that the loop over the keys reads no mask state but the bits of mixed tiles.
struct DaWalk {
    uint64_t need, part, mixed, hide;                         // workgroup: not all hidden, not all free; wave: mixed, all hidden
    int base;
    __device__ __forceinline__ void load(const DaRows &w, int64_t mb, int qt0, int qt1, int chunk, int M64, int N64) {
        const int kt = chunk * 64 + (threadIdx.x & 63);
        bool n = false, p = false, x = false, y = true;
        if (kt < M64) {
            const uint8_t *tp = da_again().tiles + mb * N64 * M64 + kt;
            for (int qt = qt0; qt <= qt1; ++qt) {
                const int c = tp[(int64_t)qt * M64];
                n = n || c != 2;
                p = p || c != 0;
            }
            const int c0 = tp[(int64_t)w.q_lo * M64], c1 = tp[(int64_t)w.q_hi * M64];
            x = c0 != c1 || c0 == 1;
            y = c0 == 2 && c1 == 2;
        }
        need = __ballot(n); part = __ballot(p); mixed = __ballot(x); hide = __ballot(y);
        base = chunk;
    }
    // the first block at or after k0 that any row of the workgroup may see part of
    __device__ __forceinline__ int next(const DiffArgs &a, const DaRows &w, int64_t mb, int qt0, int qt1, int M64, int N64, int k0, int end) {
        if (!a.tiles) return k0;
        while (k0 < end) {
            const int kt = k0 >> 6;
            if (kt >> 6 != base) load(w, mb, qt0, qt1, kt >> 6, M64, N64);
            const uint64_t m = need >> (kt & 63);
            if (m & 1) break;
            k0 = m ? (kt + __builtin_ctzll(m)) << 6 : ((kt >> 6) + 1) << 12;
        }
        return k0;
    }
    __device__ __forceinline__ int code(const DiffArgs &a, int k0) const {
        const int x = (k0 >> 6) & 63;
        return !a.tiles ? 0 : (mixed >> x) & 1 ? 1 : (hide >> x) & 1 ? 2 : 0;
    }
    // keys (from k0 on) that some query of the workgroup's tiles may see: the others are copied as zeros
    __device__ __forceinline__ uint64_t live(const DiffArgs &a, int64_t mb, int qt0, int qt1, int M64, int N64, int k0) const {
        if (!a.tiles || !((part >> ((k0 >> 6) & 63)) & 1)) return ~0ull;
        uint64_t m = 0;
        const uint64_t *some = da_again().some;
        for (int qt = qt0; qt <= qt1; ++qt) m |= some[(mb * N64 + qt) * M64 + (k0 >> 6)];
        return m >> (k0 & 63);
    }
};

template <typename T, int DK> struct DaState {
    using C = DaCfg<T, DK>;
    da_f16v o[2][C::MT];
    float m[2], l[2];                                         // running maximum (exp2 domain) and this lane's part of the sum
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            m[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
            for (int x = 0; x < C::MT; ++x)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[t][x][r] = 0.f;
        }
    }
};

template <typename T, int DK> __device__ __forceinline__ void da_load_q(const DiffArgs &a, const DaRows &w, int b, int h2, uint4 (*qf)[DaCfg<T, DK>::NF]) {
    const T *qp = reinterpret_cast<const T *>(a.q) + b * a.qs[0] + w.i * a.qs[1] + w.head * a.qs[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int f = 0; f < DaCfg<T, DK>::NF; ++f) {
            const int c = f * Da<T>::KPF + h2 * (Da<T>::KPF / 2);
            qf[t][f] = w.live && c < a.d ? *reinterpret_cast<const uint4 *>(qp + t * a.qs[3] + c) : make_uint4(0, 0, 0, 0);
        }
}

// 32 keys (rows r0 .. of the tiles in LDS) against the wave's 32 rows.  vis: bit per key of the lane's row, looked at where `masked`.
// The running maximum moves only when some row's grows by more than 2^8 (in the exp2 domain, 8): the accumulators are then rescaled; below that the
// probabilities are at most 256 times what the true maximum would give, which 32-bit sums and bf16's exponent hold without loss.
template <typename T, int DK>
__device__ __forceinline__ void da_fwd_tile(DaState<T, DK> &st, const uint4 (*qf)[DaCfg<T, DK>::NF], const DaLane<T, DK> &ln, uint32_t tk, uint32_t tv, bool masked, uint32_t vis, float c,
                                            int lane) {
    using C = DaCfg<T, DK>;
    const uint32_t mine = vis >> (4 * (lane >> 5));
    da_f16v s[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.f;
    float mu[2], sum[2] = {0.f, 0.f};
    auto scores = [&](int t) {                                // hides what is hidden, moves the maximum of map t where it has to
        if (masked) da_hide(s[t], mine);
        float bm = s[t][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) bm = fmaxf(bm, s[t][r]);
        bm = da_other_half_max(bm) * c;
        if (__any(bm > st.m[t] + 8.f)) {
            const float mn = fmaxf(st.m[t], bm), alpha = mn == -INFINITY ? 1.f : da_exp2(st.m[t] - mn);
            st.m[t] = mn;
            st.l[t] *= alpha;
#pragma unroll
            for (int x = 0; x < C::MT; ++x)
#pragma unroll
                for (int r = 0; r < 16; ++r) st.o[t][x][r] *= alpha;
        }
        mu[t] = st.m[t] == -INFINITY ? 0.f : st.m[t];
    };
    auto vec = [&](int t, int r) {
        s[t][r] = da_exp2(fmaf(s[t][r], c, -mu[t]));
        sum[t] += s[t][r];
    };
    auto value = [&](int i) { return ln.frag_tr(tv, i / C::MT, i % C::MT); };
    uint4 fr[2], pf[C::FPT];
    da_ring<C::NF, 2>([&](int i) { return ln.frag(tk, i); }, [&](int i, const uint4 &f) { s[0] = Da<T>::mma(f, qf[0][i], s[0]); });
    fr[0] = ln.frag(tk, C::NF);
    if (C::NF > 1) fr[1] = ln.frag(tk, C::NF + 1);
    scores(0);
    // the first map's exponentials between the second's products, the second's between the first map's products with the values
    da_between<C::NF>(fr, [&](int i) { return ln.frag(tk, C::NF + i); }, [&](int i, const uint4 &f) { s[1] = Da<T>::mma(f, qf[1][i], s[1]); }, [&](int r) { vec(0, r); });
    fr[0] = value(0);
    fr[1] = value(1);
#pragma unroll
    for (int f = 0; f < C::FPT; ++f) pf[f] = da_pack<T>(s[0], f);
    scores(1);
    da_between<C::FPT * C::MT>(fr, value, [&](int i, const uint4 &f) { st.o[0][i % C::MT] = Da<T>::mma(f, pf[i / C::MT], st.o[0][i % C::MT]); }, [&](int r) { vec(1, r); });
    st.l[0] += sum[0];
    st.l[1] += sum[1];
#pragma unroll
    for (int f = 0; f < C::FPT; ++f) pf[f] = da_pack<T>(s[1], f);
    da_ring<C::FPT * C::MT, 2>(value, [&](int i, const uint4 &f) { st.o[1][i % C::MT] = Da<T>::mma(f, pf[i / C::MT], st.o[1][i % C::MT]); });
}

// A wave's 32 rows x W channels from accumulator order to memory in whole rows: four channels at a time into LDS (unit u of row r at u ^ r % units), then 16
// bytes per lane, a row's units on neighbouring lanes.  (Stores straight from the accumulators are 8-byte pieces of 32 rows each: the forward pass of 32 x 492
// tokens spent 15 of its 40 us in them.)
template <typename T, int W> struct DaRowsOut {
    static constexpr int UN = W * (int)sizeof(T) / 16, RP = 64 / UN;               // units of a row, rows of one round
    char *buf;
    __device__ __forceinline__ void put(int r, int c, float a, float b, float d, float e) const {
        const int at = c * (int)sizeof(T);
        da_store4(reinterpret_cast<T *>(buf + r * W * sizeof(T) + (((at >> 4) ^ (r & (UN < 16 ? UN - 1 : 15))) << 4) + (at & 15)), a, b, d, e);
    }
    // dst(row, channel): where the 16 bytes from `channel` on of row `row` go, or null
    template <class F> __device__ __forceinline__ void flush(int lane, F dst) const {
        da_lds_done();
#pragma unroll
        for (int n = 0; n < 32 / RP; ++n) {
            const int r = n * RP + lane / UN, u = lane % UN;
            const uint4 v = *reinterpret_cast<const uint4 *>(buf + r * W * sizeof(T) + ((u ^ (r & (UN < 16 ? UN - 1 : 15))) << 4));
            T *p = dst(r, u * 16 / (int)sizeof(T));
            if (p) *reinterpret_cast<uint4 *>(p) = v;
        }
        da_lds_done();
    }
};

__device__ __forceinline__ float da_inv(float l) { return l > 0.f ? 1.f / l : l; }                 // an empty row: 0; not a number stays that
// the norm's factor from sum U^2; a row that sees no key: 0, so that its result is 0 with eps = 0 too (1 / sqrt(0) times 0 is not a number)
__device__ __forceinline__ float da_norm(float ss, const DiffArgs &a, bool empty) { return empty ? 0.f : rsqrtf(ss / (float)a.dv + a.eps); }
__device__ __forceinline__ float da_lse(float m, float l) { return l > 0.f ? m + log2f(l) : l == 0.f ? INFINITY : l; }

// ------------------------------------------------------------------------------------------------------------------
// forward, many rows: workgroup = (batch, key head, 128 rows), a wave owns 32 rows; the keys stream through two LDS buffers of KB, copied while the block
// in front is worked on (one barrier per block).
// 128 rows read a key once from L2 for 4 waves; two waves per SIMD (registers: DK = 64) hide each other's LDS and matrix latencies.  Bound: the vector unit for
// heads up to 32 channels (16 exponentials, maxima, sums and conversions per 12 products of 32 cycles), vector and matrix unit about alike at 64.
// Measured (kernel alone under the tracer, several cards): 8192 causal tokens, 16 heads on 4, 2 x 64 channels bf16 470 - 520 us (790 - 880 TFLOP/s; a plain 8192^3 product
// reaches 1177 here); 32 x 492 tokens with their group mask, 4 heads of 2 x 32, results for the backward kept, 30 - 33 us; 8 x 900 tokens, 8 heads of 2 x 24, 46 - 51 us;
// 16 x 396 tokens of 4 heads in fp32, results kept, 60 - 64 us.
template <typename T, int DK>
__global__ __launch_bounds__(kDaThreads, DK == 16 || sizeof(T) == 2 ? 2 : 1) void diff_attn_fwd_kernel(const DiffArgs a) {
    using C = DaCfg<T, DK>;
    constexpr int KB = sizeof(T) == 2 ? 64 : 32, TILE = KB * C::ROWB;
    extern __shared__ __attribute__((aligned(512))) char lds[];      // (512: DaLane)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h2 = lane >> 5, l32 = lane & 31;
    const int nbh = a.B * a.Hk, bh = blockIdx.x % nbh, nblk = gridDim.x / nbh, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int blk = a.causal ? nblk - 1 - (int)(blockIdx.x / nbh) : (int)(blockIdx.x / nbh);          // causal: the longest first
    const int len = da_len(a, b);
    const int64_t start = da_start(a, b);
    const int R = a.N * a.G, blk0 = blk * 128;
    const int M64 = (a.M + 63) >> 6, N64 = (a.N + 63) >> 6;
    const int64_t mb = a.mask_b ? b : 0;
    const DaRows w = da_rows(a, hk, blk0 + wave * 32, l32, len, start);
    const int i_end = da_div_g(a, min(blk0 + 127, R - 1));
    const int wg_end = da_limit(a, len, start, i_end), qt0 = da_div_g(a, blk0) >> 6, qt1 = i_end >> 6;

    DaCopy<T, DK, KB, kDaThreads> ck, cv;
    ck.init(reinterpret_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[2], a.ks[1], a.ks[3], a.d, true, tid);
    cv.init(reinterpret_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[2], a.vs[1], 0, a.dv, false, tid);
    const bool full = a.d == DK && a.dv == C::DV;
    const uint32_t tile0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds, lds0 = tile0 + wave * 1024;
    DaLane<T, DK> ln;
    ln.init(lane);
    DaWalk walk;
    walk.base = -1;
    auto next = [&](int k0) { return walk.next(a, w, mb, qt0, qt1, M64, N64, k0, wg_end); };
    const int64_t ldk = a.ks[1], ldv = a.vs[1];
    int stand = 0;                                            // the block that the copies stand at
    auto issue = [&](int k0, int buf) {
        const int valid = len - k0;
        const uint64_t live = walk.live(a, mb, qt0, qt1, M64, N64, k0), all = KB == 64 ? ~0ull : 0xffffffffull;
        const bool rows = valid >= KB && (live & all) == all;
        ck.move((k0 - stand) * ldk);
        cv.move((k0 - stand) * ldv);
        stand = k0;
        ck.run(lds0 + buf * 2 * TILE, valid, live, rows, full);
        cv.run(lds0 + buf * 2 * TILE + TILE, valid, live, rows, full);
    };
    auto bits = [&](int k0) {                                 // a mixed tile's keys as this lane's row sees them
        return w.live ? da_again().rowbits[(mb * a.N + w.i) * M64 + (k0 >> 6)] >> (k0 & 63) : 0ull;
    };
    int k0 = next(0), buf = 0, code = 0;
    uint64_t vis = ~0ull;
    if (k0 < wg_end) {
        code = walk.code(a, k0);
        if (code == 1) vis = bits(k0);
        issue(k0, 0);
    }
    uint4 qf[2][C::NF];
    da_load_q<T, DK>(a, w, b, h2, qf);
    DaState<T, DK> st;
    st.init();
#pragma unroll
    for (int f = 0; f < 2 * C::NF; ++f) da_pin(qf[f / C::NF][f % C::NF]);
    __shared__ __attribute__((aligned(16))) float sLam[128], sW[C::DV];         // (not held in registers over the loop)
    if (tid < C::DV) da_weights<1>(a, tid, sW + tid);
    {
        const float l = da_lambda_rows(a, hk, blk0 + wave * 32, w.head);
        if (h2 == 0) sLam[wave * 32 + l32] = l;
    }
    while (k0 < wg_end) {
        const int kn = next(k0 + KB), code_n = kn < wg_end ? walk.code(a, kn) : 0;
        uint64_t vis_n = ~0ull;
        da_copies_done_barrier();                             // block k0 is there for every wave, and every wave is done with the buffer in front
        da_pin(vis);
        if (code_n == 1) vis_n = bits(kn);                    // (in front of the copies: the wait for it is a wait for what comes before it)
        if (kn < wg_end) issue(kn, buf ^ 1);
        if (code != 2 && k0 < w.lim_hi) {
            const bool cut = k0 + KB > w.lim_lo, masked = cut || code == 1;
            if (cut) vis &= w.limit <= k0 ? 0ull : w.limit >= k0 + 64 ? ~0ull : (1ull << (w.limit - k0)) - 1;
            const uint32_t tk = tile0 + buf * 2 * TILE, tv = tk + TILE;
#pragma unroll 1
            for (int nt = 0; nt < KB / 32; ++nt) {
                const uint32_t at = nt * 32 * C::ROWB;
                da_fwd_tile<T, DK>(st, qf, ln, tk + at, tv + at, masked, (uint32_t)(vis >> (32 * nt)), a.scale_log2e, lane);
            }
        }
        k0 = kn;
        code = code_n;
        vis = vis_n;
        buf ^= 1;
    }
    const DiffArgs &e = da_again();
    const float lam = sLam[wave * 32 + l32], l0 = da_both_halves(st.l[0]), l1 = da_both_halves(st.l[1]), inv0 = da_inv(l0), inv1 = da_inv(l1);
    float ss = 0.f, us = 0.f;
#pragma unroll
    for (int x = 0; x < C::MT; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            st.o[1][x][r] *= inv1;
            st.o[0][x][r] = st.o[0][x][r] * inv0 - lam * st.o[1][x][r];
            ss += st.o[0][x][r] * st.o[0][x][r];
            us += st.o[0][x][r] * st.o[1][x][r];
        }
    ss = da_both_halves(ss);
    us = da_both_halves(us);
    const float beta = e.weight && ss > 0.f ? us / ss : 0.f;  // what is kept of A_1 V is its part at right angles to U (diff_attn_prep_kernel)
    const float rn = e.weight ? da_norm(ss, e, l0 == 0.f) : 1.f;
    int row = blk0 + wave * 32 + l32;
    asm volatile("" : "+v"(row));                             // (worked out again: the row's numbers are not held over the loop either)
    if (e.stats && h2 == 0 && row < R) {
        const int i = da_div_g(e, row);
        const int64_t bhn = (int64_t)e.B * e.H * e.N, at = ((int64_t)b * e.H + hk * e.G + row - i * e.G) * e.N + i;
        e.stats[at] = da_lse(st.m[0], l0);
        e.stats[bhn + at] = da_lse(st.m[1], l1);
        e.stats[2 * bhn + at] = rn;
        e.stats[3 * bhn + at] = beta;
    }
    __syncthreads();                                          // every wave is done with the tiles
    char *own = lds + wave * 32 * C::DV * 4;
    const DaRowsOut<T, C::DV> rows{own};
    const int w0 = blk0 + wave * 32;
    auto to = [&](auto rows, auto *base) {
        rows.flush(lane, [&](int r, int c) {
            const int row = w0 + r, i = da_div_g(e, min(row, R - 1));
            return row < R && c < e.dv ? base + (((int64_t)b * e.N + i) * e.H + hk * e.G + row - i * e.G) * e.dv + c : nullptr;
        });
    };
#pragma unroll
    for (int x = 0; x < C::MT; ++x)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const int c = x * 32 + 8 * q4 + 4 * h2;
            const float4 g = *reinterpret_cast<const float4 *>(sW + c);
            rows.put(l32, c, st.o[0][x][4 * q4] * g.x * rn, st.o[0][x][4 * q4 + 1] * g.y * rn, st.o[0][x][4 * q4 + 2] * g.z * rn, st.o[0][x][4 * q4 + 3] * g.w * rn);
        }
    to(rows, reinterpret_cast<T *>(e.out));
    if (!e.o2) return;
    {
        const DaRowsOut<float, C::DV> rows{own};
#pragma unroll
        for (int x = 0; x < C::MT; ++x)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                rows.put(l32, x * 32 + 8 * q4 + 4 * h2, st.o[0][x][4 * q4], st.o[0][x][4 * q4 + 1], st.o[0][x][4 * q4 + 2], st.o[0][x][4 * q4 + 3]);
        to(rows, e.u);
    }
#pragma unroll
    for (int x = 0; x < C::MT; ++x)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            float o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = st.o[1][x][4 * q4 + j] - beta * st.o[0][x][4 * q4 + j];
            rows.put(l32, x * 32 + 8 * q4 + 4 * h2, o[0], o[1], o[2], o[3]);
        }
    to(rows, reinterpret_cast<T *>(e.o2));
}

// One row of the result from its two maps' sums in plain order: LPR neighbouring lanes of NE channels each (c0: the lane's first), O normalised
template <typename T, int NE, int LPR>
__device__ __forceinline__ void da_finish_row(const DiffArgs &a, int b, int i, int head, float lam, int c0, const float *g, float *o0, float *o1, float lse0,
                                              float lse1, bool first) {
    float ss = 0.f, us = 0.f;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
        o0[j] -= lam * o1[j];
        ss += o0[j] * o0[j];
        us += o0[j] * o1[j];
    }
#pragma unroll
    for (int x = 1; x < LPR; x <<= 1) { ss += __shfl_xor(ss, x); us += __shfl_xor(us, x); }
    const float beta = a.weight && ss > 0.f ? us / ss : 0.f;
    const float rn = a.weight ? da_norm(ss, a, lse0 == INFINITY) : 1.f;
    const int64_t orow = (((int64_t)b * a.N + i) * a.H + head) * a.dv;
#pragma unroll
    for (int j = 0; j < NE; j += 4) {
        const int c = c0 + j;
        if (c >= a.dv) continue;
        da_store4(reinterpret_cast<T *>(a.out) + orow + c, o0[j] * g[j] * rn, o0[j + 1] * g[j + 1] * rn, o0[j + 2] * g[j + 2] * rn, o0[j + 3] * g[j + 3] * rn);
        if (a.o2) {
            da_store4(a.u + orow + c, o0[j], o0[j + 1], o0[j + 2], o0[j + 3]);
            da_store4(reinterpret_cast<T *>(a.o2) + orow + c, o1[j] - beta * o0[j], o1[j + 1] - beta * o0[j + 1], o1[j + 2] - beta * o0[j + 2], o1[j + 3] - beta * o0[j + 3]);
        }
    }
    if (a.stats && first) {
        const int64_t bhn = (int64_t)a.B * a.H * a.N, at = ((int64_t)b * a.H + head) * a.N + i;
        a.stats[at] = lse0;
        a.stats[bhn + at] = lse1;
        a.stats[2 * bhn + at] = rn;
        a.stats[3 * bhn + at] = beta;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// forward, few rows: workgroup = (batch, key head, 32 rows, one of nsplit runs of the keys), its waves take every fourth tile of 32 keys of the run, each
// through two LDS buffers of its own (no barrier until the end).  The waves' sums meet in LDS; with one run the rows are finished here, else the run's sums
// go to `part` (rows x nsplit x 2 DV, with maxima and sums in `ml`) for diff_attn_join_kernel.
// Bound: HBM, every key and value once for all heads of the group.  Measured: one token of 16 heads over 16 caches of up to 32768 keys (835 MB) 161 - 165 us, 5.1 - 5.2 TB/s,
// in fp32 (1670 MB) 507 - 520 us: one buffer per wave there, so a wave's copies (340 us at a large copy's rate) and fp32 products (260 us) follow each other;
// 17 tokens over 4 x 10001 keys 21 - 23 us (41 MB: 11 us of it are the first loads, the joins in LDS and the last stores); 300 tokens of one image 10.2 - 10.6 us.
template <typename T, int DK>
__global__ __launch_bounds__(kDaThreads, DK * sizeof(T) <= 64 ? 2 : 1) void diff_attn_fwd_split_kernel(const DiffArgs a, int nsplit, float *__restrict__ part, float4 *__restrict__ ml) {
    using C = DaCfg<T, DK>;
    constexpr int TILE = 32 * C::ROWB, NE = C::DV / 8, UO = 2 * C::DV / 4;
    constexpr int NBUF = C::ROWB > 256 ? 1 : 2;               // (fp32 heads of 64: two buffers for four waves would not fit LDS)
    constexpr int WBYTES = NBUF * 2 * TILE;                   // a wave's buffers, later its sums
    static_assert(WBYTES >= 32 * 2 * C::DV * 4, "");
    extern __shared__ __attribute__((aligned(512))) char lds[];      // (512: DaLane)
    __shared__ float sM[2][4][32], sS[2][4][32], sLam[32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h2 = lane >> 5, l32 = lane & 31;
    const int nbh = a.B * a.Hk, bh = blockIdx.x % nbh, rest = blockIdx.x / nbh, sp = rest % nsplit, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int blk = rest / nsplit, R = a.N * a.G;
    const int len = da_len(a, b);
    const int64_t start = da_start(a, b);
    const int M64 = (a.M + 63) >> 6, N64 = (a.N + 63) >> 6;
    const int64_t mb = a.mask_b ? b : 0;
    const DaRows w = da_rows(a, hk, blk * 32, l32, len, start);
    const int tiles = (w.lim_hi + 31) >> 5, per = (tiles + nsplit - 1) / nsplit, t_end = min(tiles, (sp + 1) * per);

    DaCopy<T, DK, 32, 64> ck, cv;
    constexpr int NCOPY = 2 * DaCopy<T, DK, 32, 64>::J;
    ck.init(reinterpret_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[2], a.ks[1], a.ks[3], a.d, true, lane);
    cv.init(reinterpret_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[2], a.vs[1], 0, a.dv, false, lane);
    const bool full = a.d == DK && a.dv == C::DV;
    char *mine = lds + wave * WBYTES;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)mine;
    DaLane<T, DK> ln;
    ln.init(lane);
    DaWalk walk;
    walk.base = -1;
    auto next = [&](int t) {
        for (; a.tiles && t < t_end; t += 4) {
            if (t >> 7 != walk.base) walk.load(w, mb, w.q_lo, w.q_hi, t >> 7, M64, N64);
            if (walk.code(a, t * 32) != 2) break;
        }
        return t;
    };
    const int64_t ldk = a.ks[1], ldv = a.vs[1];
    int stand = 0;                                            // the key that the copies stand at
    auto bits = [&](int t) {
        uint32_t v = w.live ? (uint32_t)(da_again().rowbits[(mb * a.N + w.i) * M64 + (t >> 1)] >> (t & 1 ? 32 : 0)) : 0u;
        da_pin(v);
        return v;
    };
    auto issue = [&](int t, int buf) {
        const int k0 = t * 32, valid = len - k0;
        const uint64_t live = walk.live(a, mb, w.q_lo, w.q_hi, M64, N64, k0);
        const bool rows = valid >= 32 && (uint32_t)live == ~0u;
        ck.move((k0 - stand) * ldk);
        cv.move((k0 - stand) * ldv);
        stand = k0;
        ck.run(lds0 + buf * 2 * TILE, valid, live, rows, full);
        cv.run(lds0 + buf * 2 * TILE + TILE, valid, live, rows, full);
    };
    int t = next(sp * per + wave), buf = 0, code = 0;
    uint32_t vis = ~0u;
    if (t < t_end) {
        code = walk.code(a, t * 32);
        if (code == 1) vis = bits(t);
        if (NBUF == 2) issue(t, 0);
    }
    uint4 qf[2][C::NF];
    da_load_q<T, DK>(a, w, b, h2, qf);
    DaState<T, DK> st;
    st.init();
#pragma unroll
    for (int f = 0; f < 2 * C::NF; ++f) da_pin(qf[f / C::NF][f % C::NF]);
    if (wave == 0 && nsplit == 1) {
        const float lam = da_lambda_rows(a, hk, blk * 32, w.head);
        if (h2 == 0) sLam[l32] = lam;
    }
    while (t < t_end) {
        if (NBUF == 1) {
            da_lds_done();
            issue(t, 0);
        }
        const int tn = next(t + 4), code_n = tn < t_end ? walk.code(a, tn * 32) : 0, k0 = t * 32;
        uint32_t vis_n = ~0u;
        if (code_n == 1) vis_n = bits(tn);
        da_lds_done();                                        // the buffer in front has been read
        if (NBUF == 2 && tn < t_end) {
            issue(tn, buf ^ 1);
            da_wait_copies<NCOPY>();                          // tile t is there; tile tn may be on its way
        } else {
            da_wait_copies<0>();
        }
        const bool cut = k0 + 32 > w.lim_lo, masked = cut || code == 1;
        if (cut) vis &= w.limit <= k0 ? 0u : w.limit >= k0 + 32 ? ~0u : (1u << (w.limit - k0)) - 1;
        const uint32_t tk = lds0 + buf * 2 * TILE;
        da_fwd_tile<T, DK>(st, qf, ln, tk, tk + TILE, masked, vis, a.scale_log2e, lane);
        t = tn;
        code = code_n;
        vis = vis_n;
        buf ^= NBUF - 1;
    }
    // the four waves' sums: common maximum, then every wave's share of it through LDS (unit u of row r at u ^ (r % 16))
    da_lds_done();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const float l = da_both_halves(st.l[x]);
        if (h2 == 0) { sM[x][wave][l32] = st.m[x]; sS[x][wave][l32] = l; }
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        float mx = sM[x][0][l32];
#pragma unroll
        for (int v = 1; v < 4; ++v) mx = fmaxf(mx, sM[x][v][l32]);
        const float f = mx == -INFINITY ? 1.f : da_exp2(st.m[x] - mx);
#pragma unroll
        for (int y = 0; y < C::MT; ++y)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const int u = (x * C::DV + y * 32 + 8 * q4 + 4 * h2) >> 2;
                const da_f16v &o = st.o[x][y];
                *reinterpret_cast<float4 *>(mine + l32 * UO * 16 + ((u ^ (l32 & 15)) << 4)) = make_float4(o[4 * q4] * f, o[4 * q4 + 1] * f, o[4 * q4 + 2] * f, o[4 * q4 + 3] * f);
            }
    }
    __syncthreads();
    const int r = tid >> 3, c0 = (tid & 7) * NE;
    const int row = blk * 32 + r;
    if (row >= R) return;
    float g[NE];
    if (nsplit == 1) da_weights<NE>(a, c0, g);
    float o[2][NE], lse[2], mx[2], sum[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        mx[x] = fmaxf(fmaxf(sM[x][0][r], sM[x][1][r]), fmaxf(sM[x][2][r], sM[x][3][r]));
        sum[x] = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[x] += mx[x] == -INFINITY ? sS[x][v][r] : sS[x][v][r] * da_exp2(sM[x][v][r] - mx[x]);
        lse[x] = da_lse(mx[x], sum[x]);
#pragma unroll
        for (int j = 0; j < NE; j += 4) {
            const int u = (x * C::DV + c0 + j) >> 2;
            float4 s4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float4 z = *reinterpret_cast<const float4 *>(lds + v * WBYTES + r * UO * 16 + ((u ^ (r & 15)) << 4));
                s4.x += z.x; s4.y += z.y; s4.z += z.z; s4.w += z.w;
            }
            o[x][j] = s4.x; o[x][j + 1] = s4.y; o[x][j + 2] = s4.z; o[x][j + 3] = s4.w;
        }
    }
    const int i = da_div_g(a, row), head = hk * a.G + row - i * a.G;
    if (nsplit == 1) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const float inv = da_inv(sum[x]);
#pragma unroll
            for (int j = 0; j < NE; ++j) o[x][j] *= inv;
        }
        da_finish_row<T, NE, 8>(a, b, i, head, sLam[r], c0, g, o[0], o[1], lse[0], lse[1], (tid & 7) == 0);
        return;
    }
    const int64_t at = ((int64_t)bh * R + row) * nsplit + sp;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < NE; j += 4) *reinterpret_cast<float4 *>(part + (at * 2 + x) * C::DV + c0 + j) = make_float4(o[x][j], o[x][j + 1], o[x][j + 2], o[x][j + 3]);
    if ((tid & 7) == 0) ml[at] = make_float4(mx[0], sum[0], mx[1], sum[1]);
}

// joins the runs of a row: a wave per row, 8 lanes x DV / 8 channels, 8 runs side by side, in a fixed order.  Bound: latency (a launch, one round of loads, the
// reduction); 9 - 10 us for the two bf16 cases above.
template <typename T, int DV>
__global__ __launch_bounds__(kDaThreads) void diff_attn_join_kernel(const DiffArgs a, int nsplit, const float *__restrict__ part, const float4 *__restrict__ ml) {
    constexpr int NE = DV / 8;
    const int lane = threadIdx.x & 63, sg = lane >> 3, c0 = (lane & 7) * NE;
    const int R = a.N * a.G;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (int64_t)R * a.B * a.Hk) return;
    const int bh = (int)(at / R), b = bh / a.Hk, hk = bh - b * a.Hk;
    const int row = (int)(at - (int64_t)bh * R), i = da_div_g(a, row), head = hk * a.G + row - i * a.G;
    const float4 vectors = da_lambda_vectors(a, head);        // (asked for in front of the sums)
    float g[NE], mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, o[2][NE];
    da_weights<NE>(a, c0, g);
#pragma unroll
    for (int j = 0; j < NE; ++j) o[0][j] = o[1][j] = 0.f;
#pragma unroll 2
    for (int s = sg; s < nsplit; s += 8) {                    // (the sums come with their maximum: no load waits for another)
        const float4 v = ml[at * nsplit + s];
        const float m[2] = {v.x, v.z}, l[2] = {v.y, v.w};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float4 z[NE / 4];
#pragma unroll
            for (int j = 0; j < NE / 4; ++j) z[j] = *reinterpret_cast<const float4 *>(part + ((at * nsplit + s) * 2 + x) * DV + c0 + 4 * j);
            const float mn = fmaxf(mx[x], m[x]), f = mn == -INFINITY ? 1.f : da_exp2(mx[x] - mn), g = mn == -INFINITY ? 1.f : da_exp2(m[x] - mn);
            mx[x] = mn;
            sum[x] = sum[x] * f + l[x] * g;
#pragma unroll
            for (int j = 0; j < NE / 4; ++j) {
                o[x][4 * j] = o[x][4 * j] * f + z[j].x * g;
                o[x][4 * j + 1] = o[x][4 * j + 1] * f + z[j].y * g;
                o[x][4 * j + 2] = o[x][4 * j + 2] * f + z[j].z * g;
                o[x][4 * j + 3] = o[x][4 * j + 3] * f + z[j].w * g;
            }
        }
    }
    const float lam = da_lambda(a, vectors);
#pragma unroll
    for (int x = 0; x < 2; ++x) {                             // the 8 groups, in order of their distance
        float m = mx[x];
#pragma unroll
        for (int y = 8; y < 64; y <<= 1) m = fmaxf(m, __shfl_xor(m, y));
        const float f = m == -INFINITY ? 1.f : da_exp2(mx[x] - m);
        mx[x] = m;
        sum[x] *= f;
#pragma unroll
        for (int j = 0; j < NE; ++j) o[x][j] *= f;
#pragma unroll
        for (int y = 8; y < 64; y <<= 1) {
            sum[x] += __shfl_xor(sum[x], y);
#pragma unroll
            for (int j = 0; j < NE; ++j) o[x][j] += __shfl_xor(o[x][j], y);
        }
    }
    if (sg) return;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const float inv = da_inv(sum[x]);
#pragma unroll
        for (int j = 0; j < NE; ++j) o[x][j] *= inv;
    }
    da_finish_row<T, NE, 8>(a, b, i, head, lam, c0, g, o[0], o[1], da_lse(mx[0], sum[0]), da_lse(mx[1], sum[1]), lane == 0);
}

// ------------------------------------------------------------------------------------------------------------------
// mask [Bm][N][M] bytes (strides sb, sn; non-zero = blocked) -> the forms the kernels read.  Workgroup = tile of 64 queries x 64 keys, a wave takes 16 queries;
// lane = key, one ballot per query, all 16 loads in flight.  4 us for 492 x 492 (a launch and its latency).
__global__ __launch_bounds__(256) void diff_attn_mask_kernel(const uint8_t *__restrict__ mask, int64_t sb, int64_t sn, int N, int M, uint64_t *__restrict__ rowbits,
                                                             uint64_t *__restrict__ colbits, uint64_t *__restrict__ some_, uint8_t *__restrict__ tiles) {
    const int M64 = (M + 63) >> 6, N64 = (N + 63) >> 6;
    const int kt = blockIdx.x % M64, rest = blockIdx.x / M64;
    const int64_t b = rest / N64;
    const int nt = rest - (int)b * N64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, key = kt * 64 + lane, n0 = nt * 64 + wave * 16, n1 = min(16, N - n0);
    const uint64_t inside = M - kt * 64 >= 64 ? ~0ull : (1ull << (M - kt * 64)) - 1;
    const uint8_t *p = mask + b * sb + min(key, M - 1);
    uint32_t v[16], c = 0;
#pragma unroll
    for (int x = 0; x < 16; ++x) v[x] = p[(int64_t)min(n0 + x, N - 1) * sn];
    uint64_t all = inside, some = 0, mine = 0;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        const bool see = v[x] == 0 && key < M && x < n1;
        const uint64_t bits = __ballot(see);
        c |= see ? 1u << x : 0u;
        mine = x == lane ? bits : mine;
        all &= x < n1 ? bits : ~0ull;
        some |= bits;
    }
    __shared__ __attribute__((aligned(8))) uint16_t col[64][4];
    __shared__ uint64_t s_all[4], s_some[4];
    col[lane][wave] = (uint16_t)c;
    if (lane == 0) { s_all[wave] = all; s_some[wave] = some; }
    if (lane < n1) rowbits[(b * N + n0 + lane) * M64 + kt] = mine;
    __syncthreads();
    if (wave == 0 && key < M) colbits[(b * M + key) * N64 + nt] = *reinterpret_cast<const uint64_t *>(col[lane]);
    if (threadIdx.x == 64) {
        some = s_some[0] | s_some[1] | s_some[2] | s_some[3];
        all = s_all[0] & s_all[1] & s_all[2] & s_all[3];
        some_[(b * N64 + nt) * M64 + kt] = some;
        tiles[(b * N64 + nt) * M64 + kt] = some == 0 ? 2 : all == inside ? 0 : 1;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// backward, first: dU (rounded to the type it is multiplied in), D_0, D_1 of every row and the partial sums of dl and dg.  Workgroup = (head, run of
// (batch, query) rows); the lanes of a row sit next to each other.
// With a norm dU stands at right angles to U up to eps: dU . U = r (t . U) eps r^2 with t = (1 - init) g dY.  A_1 V mostly points along U (both are
// near the mean of the values where the maps are flat), so dU . (A_1 V) of rounded vectors would be a small difference of large products.  The forward
// pass therefore keeps W = A_1 V - beta U, beta = (A_1 V . U) / (U . U), and D_1 = r (t . W) + beta (dU . U), D_0 = dU . U + l D_1 (long rows, bf16: error of dl
// and dq against 64 bits 0.0046 with A_1 V itself), and U in 32 bits: dU . U is small for the same reason (with U in bf16 dq was 0.0042 off instead of 0.0030).
// dP is made from the ROUNDED dU: what the rounding adds to D is added here too.
// Bound: HBM (dY, U, W read, dU written: 41 MB and 14 - 15 us at 32 x 492 tokens of 4 heads, 168 MB and 34 - 35 us at 8192 of 16; two rounds of rows per workgroup leave
// latency in the small case; loading a row ahead of its use changed nothing, 14.0 and 34 us).
// The other kernels read the rows' statistics with l worked in - exp2(c s - (lse_1 - log2 |l|)) is |l| A_1, and its sign goes with D_1 and dP - and as the
// numbers that dK's and dV's products start from: S_t at -lse_t / c, dP at -D_0.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void diff_attn_prep_kernel(const DiffArgs a, int nrun) {
    constexpr int RW = 256 / LPR;                                                              // rows at a time, LPR lanes of 8 channels each
    const int head = blockIdx.x % a.H, run = blockIdx.x / a.H;
    const int tid = threadIdx.x, lane = tid % LPR, rr = tid / LPR, c = lane * 8;
    const bool ok = c < a.dv;
    const float lam = da_lambda(a, head), log2l = log2f(fabsf(lam)), sign = lam < 0.f ? -1.f : 1.f, inv_c = 1.f / a.scale_log2e;
    float w[8], dw[8], dsum = 0.f;
    da_weights<8>(a, c, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[j] = 0.f;
    const int64_t rows = (int64_t)a.B * a.N, bhn = rows * a.H;
    for (int64_t r = (int64_t)run * RW + rr; r < rows; r += (int64_t)nrun * RW) {
        const int b = (int)(r / a.N), i = (int)(r - (int64_t)b * a.N);
        const int64_t at = ((int64_t)b * a.H + head) * a.N + i, orow = (r * a.H + head) * a.dv + c;
        float dy[8], u[8], o2[8], du[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) dy[j] = u[j] = o2[j] = 0.f;
        if (ok) {
            const T *yp = reinterpret_cast<const T *>(a.dy) + b * a.dys[0] + i * a.dys[1] + head * a.dys[2] + c;
            const float *up = a.u + orow;
            const T *op = reinterpret_cast<const T *>(a.o2) + orow;
            da_load4(yp, dy); da_load4(yp + 4, dy + 4);
            da_load4(up, u); da_load4(up + 4, u + 4);
            da_load4(op, o2); da_load4(op + 4, o2 + 4);
        }
        const float lse0 = a.stats[at], lse1 = a.stats[bhn + at];
        const bool empty = lse0 == INFINITY;                                                   // sees no key: no gradient, whatever dY holds
        const float rn = a.weight ? a.stats[2 * bhn + at] : 1.f, beta = a.weight ? a.stats[3 * bhn + at] : 0.f;
        float dot = 0.f, d1 = 0.f, e1r = 0.f, e2r = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            dot += u[j] * w[j] * dy[j];
            d1 += w[j] * dy[j] * o2[j];
        }
#pragma unroll
        for (int x = 1; x < LPR; x <<= 1) { dot += __shfl_xor(dot, x); d1 += __shfl_xor(d1, x); }
        float uu = dot;                                                                        // dU . U
        if (a.weight) {
            uu = rn * dot * a.eps * rn * rn;
            d1 = rn * d1 + beta * uu;
            dot *= rn * rn / (float)a.dv;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (a.weight) {
                du[j] = rn * (w[j] * dy[j] - u[j] * dot);
                if (!empty) dw[j] += a.post * rn * u[j] * dy[j];
                const float lost = da_round<T>(du[j]) - du[j];
                e1r += lost * u[j];
                e2r += lost * (o2[j] + beta * u[j]);
            } else {
                du[j] = dy[j];
            }
            if (empty) du[j] = 0.f;
        }
        if (sizeof(T) == 2 && a.weight) {
#pragma unroll
            for (int x = 1; x < LPR; x <<= 1) { e1r += __shfl_xor(e1r, x); e2r += __shfl_xor(e2r, x); }
        }
        float d0 = uu + lam * d1;
        if (empty) d0 = d1 = e1r = e2r = 0.f;
        if (ok) {
            T *dp = reinterpret_cast<T *>(a.du) + orow;
            da_store4(dp, du[0], du[1], du[2], du[3]);
            da_store4(dp + 4, du[4], du[5], du[6], du[7]);
        }
        if (lane == 0) {
            const float dd0 = d0 + e1r + lam * e2r;
            a.rowstat[at] = -lse0 * inv_c;
            a.rowstat[bhn + at] = (log2l - lse1) * inv_c;
            a.rowstat[2 * bhn + at] = -dd0;
            a.rowstat[3 * bhn + at] = (d1 + e2r - dd0) * sign;
            dsum += d1;
        }
    }
    // this workgroup's sums: lanes of the same channels, then waves, in order
    __shared__ float sw[4][LPR * 8], sd[4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int x = LPR; x < 64; x <<= 1) dw[j] += __shfl_xor(dw[j], x);
    }
    dsum = da_wave_sum(dsum);
    if ((tid & 63) < LPR) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sw[tid >> 6][c + j] = dw[j];
        if (lane == 0) sd[tid >> 6] = dsum;
    }
    __syncthreads();
    if (a.weight)
        for (int x = tid; x < a.dv; x += 256) a.wpart[(int64_t)blockIdx.x * a.dv + x] = (sw[0][x] + sw[1][x]) + (sw[2][x] + sw[3][x]);
    if (tid == 0) a.lpart[blockIdx.x] = (sd[0] + sd[1]) + (sd[2] + sd[3]);
}

// gradients of the learned vectors and of the norm weight from the first kernel's partial sums, in a fixed order: one workgroup per head (or one for shared
// vectors), then one per 32 channels of the weight (32 interleaved runs of the partial rows, 8 loads in flight).  4 - 5 us, latency.
__global__ __launch_bounds__(1024) void diff_attn_param_kernel(const DiffArgs a, int nrun, void *dlam, void *dw) {
    const int tid = threadIdx.x;
    __shared__ float s[32][33];
    const int nh = a.lam_heads == 1 ? 1 : a.H;
    if ((int)blockIdx.x < nh) {
        if (!dlam) return;
        // sum over runs (and over all heads where they share the vectors; their exponentials are then one pair)
        const int h0 = a.lam_heads == 1 ? 0 : blockIdx.x, nhead = a.lam_heads == 1 ? a.H : 1;
        float v = 0.f;
        for (int x = tid; x < nrun * nhead; x += 1024) v += a.lpart[(x / nhead) * a.H + h0 + x % nhead];
        v = da_wave_sum(v);
        if ((tid & 63) == 0) s[0][tid >> 6] = v;
        float e1, e2;
        da_lambda_parts(da_lambda_vectors(a, h0), e1, e2);
        __syncthreads();
        float dl = 0.f;
#pragma unroll
        for (int x = 0; x < 16; ++x) dl -= s[0][x];
        const int64_t st = (int64_t)a.lam_heads * a.d, o = (a.lam_heads == 1 ? 0 : (int64_t)h0 * a.d);
        if (tid >= 4 * a.d) return;
        const int vec = tid / a.d, j = tid - vec * a.d;
        const float other = da_load1(a.lam, (vec ^ 1) * st + o + j, a.lam_bf16), gr = dl * (vec < 2 ? e1 : -e2) * other;
        if (a.lam_bf16) reinterpret_cast<uint16_t *>(dlam)[vec * st + o + j] = f32_to_bf16(gr);
        else reinterpret_cast<float *>(dlam)[vec * st + o + j] = gr;
        return;
    }
    if (!dw) return;
    const int col = tid & 31, r0 = tid >> 5, ch = (blockIdx.x - nh) * 32 + col, rows = nrun * a.H;
    float v = 0.f;
    if (ch < a.dv) {
#pragma unroll 8
        for (int r = r0; r < rows; r += 32) v += a.wpart[(int64_t)r * a.dv + ch];
    }
    s[r0][col] = v;
    __syncthreads();
    if (r0 || ch >= a.dv) return;
#pragma unroll
    for (int r = 1; r < 32; ++r) v += s[r][col];
    if (a.w_bf16) reinterpret_cast<uint16_t *>(dw)[ch] = f32_to_bf16(v);
    else reinterpret_cast<float *>(dw)[ch] = v;
}

// ------------------------------------------------------------------------------------------------------------------
// backward, dQ: the forward's decomposition and copies; probabilities from the saved statistics, nothing to rescale.  dS is rounded to bf16 for its product with K (as the keys it meets
// are), dU for its product with V: each adds 0.0017 to dq's relative error, 0.0030 in all with the result's own 0.0017.  Keeping either in two bf16 terms would
// cost a third more products for 0.0025.
// Bound as the forward: 453 - 495 us (830 - 910 TFLOP/s) at 8192 causal tokens, 25 - 27 us at 32 x 492, 56 - 59 us in fp32 at 16 x 396.
template <typename T, int DK>
__device__ __forceinline__ void da_dq_tile(const DiffArgs &a, da_f16v (*dq)[DaCfg<T, DK>::MTK], const uint4 (*qf)[DaCfg<T, DK>::NF], const uint4 *uf, const float *lse, const float *dl,
                                           float sign, const DaLane<T, DK> &ln, uint32_t tk, uint32_t tv, bool masked, uint32_t vis, int lane) {
    using C = DaCfg<T, DK>;
    const float c = a.scale_log2e;
    da_f16v dp, s[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] = s[0][r] = s[1][r] = 0.f;
    const uint32_t mine = vis >> (4 * (lane >> 5));
    da_ring<C::NFV + C::NF, 2>([&](int i) { return i < C::NFV ? ln.frag(tv, i) : ln.frag(tk, i - C::NFV); },
                               [&](int i, const uint4 &f) {
                                   if (i < C::NFV) dp = Da<T>::mma(f, uf[i], dp);
                                   else s[0] = Da<T>::mma(f, qf[0][i - C::NFV], s[0]);
                               });
    uint4 fr[2], sf[C::FPT];
    fr[0] = ln.frag(tk, C::NF);
    if (C::NF > 1) fr[1] = ln.frag(tk, C::NF + 1);
    if (masked) da_hide(s[0], mine);
    // the first map's vector work between the second's scores, the second's between the first map's products with the keys
    da_between<C::NF>(fr, [&](int i) { return ln.frag(tk, C::NF + i); }, [&](int i, const uint4 &f) { s[1] = Da<T>::mma(f, qf[1][i], s[1]); },
                      [&](int r) { s[0][r] = da_exp2(fmaf(s[0][r], c, -lse[0])) * (dp[r] - dl[0]); });
    auto key = [&](int t, int i) { return ln.frag_tr(tk, i / C::MTK, DK < 32 ? 0 : t * (DK / 32) + i % C::MTK); };
    fr[0] = key(0, 0);
    fr[1] = key(0, 1);
#pragma unroll
    for (int f = 0; f < C::FPT; ++f) sf[f] = da_pack<T>(s[0], f);
    if (masked) da_hide(s[1], mine);
    da_between<C::FPT * C::MTK>(fr, [&](int i) { return key(0, i); }, [&](int i, const uint4 &f) { dq[0][i % C::MTK] = Da<T>::mma(f, sf[i / C::MTK], dq[0][i % C::MTK]); },
                                [&](int r) { s[1][r] = da_exp2(fmaf(s[1][r], c, -lse[1])) * fmaf(dp[r], -sign, dl[1]); });
#pragma unroll
    for (int f = 0; f < C::FPT; ++f) sf[f] = da_pack<T>(s[1], f);
    da_ring<C::FPT * C::MTK, 2>([&](int i) { return key(1, i); }, [&](int i, const uint4 &f) { dq[1][i % C::MTK] = Da<T>::mma(f, sf[i / C::MTK], dq[1][i % C::MTK]); });
}

template <typename T, int DK>
__global__ __launch_bounds__(kDaThreads, DK == 16 || sizeof(T) == 2 ? 2 : 1) void diff_attn_dq_kernel(const DiffArgs a) {
    using C = DaCfg<T, DK>;
    constexpr int KB = sizeof(T) == 2 ? 64 : 32, TILE = KB * C::ROWB;
    extern __shared__ __attribute__((aligned(512))) char lds[];      // (512: DaLane)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h2 = lane >> 5, l32 = lane & 31;
    const int nbh = a.B * a.Hk, bh = blockIdx.x % nbh, nblk = gridDim.x / nbh, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int blk = a.causal ? nblk - 1 - (int)(blockIdx.x / nbh) : (int)(blockIdx.x / nbh);          // causal: the longest first
    const int len = da_len(a, b);
    const int64_t start = da_start(a, b);
    const int R = a.N * a.G, blk0 = blk * 128;
    const int M64 = (a.M + 63) >> 6, N64 = (a.N + 63) >> 6;
    const int64_t mb = a.mask_b ? b : 0;
    const DaRows w = da_rows(a, hk, blk0 + wave * 32, l32, len, start);
    const int i_end = da_div_g(a, min(blk0 + 127, R - 1));
    const int wg_end = da_limit(a, len, start, i_end), qt0 = da_div_g(a, blk0) >> 6, qt1 = i_end >> 6;

    DaCopy<T, DK, KB, kDaThreads> ck, cv;
    ck.init(reinterpret_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[2], a.ks[1], a.ks[3], a.d, true, tid);
    cv.init(reinterpret_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[2], a.vs[1], 0, a.dv, false, tid);
    const bool full = a.d == DK && a.dv == C::DV;
    const uint32_t tile0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds, lds0 = tile0 + wave * 1024;
    DaLane<T, DK> ln;
    ln.init(lane);
    DaWalk walk;
    walk.base = -1;
    auto next = [&](int k0) { return walk.next(a, w, mb, qt0, qt1, M64, N64, k0, wg_end); };
    const int64_t ldk = a.ks[1], ldv = a.vs[1];
    int stand = 0;                                            // the block that the copies stand at
    auto issue = [&](int k0, int buf) {
        const int valid = len - k0;
        const uint64_t live = walk.live(a, mb, qt0, qt1, M64, N64, k0), all = KB == 64 ? ~0ull : 0xffffffffull;
        const bool rows = valid >= KB && (live & all) == all;
        ck.move((k0 - stand) * ldk);
        cv.move((k0 - stand) * ldv);
        stand = k0;
        ck.run(lds0 + buf * 2 * TILE, valid, live, rows, full);
        cv.run(lds0 + buf * 2 * TILE + TILE, valid, live, rows, full);
    };
    auto bits = [&](int k0) {                                 // a mixed tile's keys as this lane's row sees them
        return w.live ? da_again().rowbits[(mb * a.N + w.i) * M64 + (k0 >> 6)] >> (k0 & 63) : 0ull;
    };
    int k0 = next(0), buf = 0, code = 0;
    uint64_t vis = ~0ull;
    if (k0 < wg_end) {
        code = walk.code(a, k0);
        if (code == 1) vis = bits(k0);
        issue(k0, 0);
    }

    const float lam = da_lambda_rows(a, hk, blk0 + wave * 32, w.head), sign = lam < 0.f ? -1.f : 1.f;
    const int64_t bhn = (int64_t)a.B * a.H * a.N, at = ((int64_t)b * a.H + w.head) * a.N + w.i;
    uint4 qf[2][C::NF], uf[C::NFV];
    float lse[2], dl[2];
    const T *qp = reinterpret_cast<const T *>(a.q) + b * a.qs[0] + w.i * a.qs[1] + w.head * a.qs[2];
    const T *up = reinterpret_cast<const T *>(a.du) + (((int64_t)b * a.N + w.i) * a.H + w.head) * a.dv;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        lse[t] = w.live ? a.rowstat[t * bhn + at] * -a.scale_log2e : INFINITY;
        dl[t] = w.live ? a.rowstat[(2 + t) * bhn + at] : 0.f;
    }
    dl[1] -= sign * dl[0];
    dl[0] = -dl[0];
    const bool empty = lse[0] == INFINITY;                    // sees no key: its query may hold anything
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int f = 0; f < C::NF; ++f) {
            const int c = f * Da<T>::KPF + h2 * (Da<T>::KPF / 2);
            qf[t][f] = w.live && !empty && c < a.d ? *reinterpret_cast<const uint4 *>(qp + t * a.qs[3] + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
    for (int f = 0; f < C::NFV; ++f) {
        const int c = f * Da<T>::KPF + h2 * (Da<T>::KPF / 2);
        uf[f] = w.live && c < a.dv ? *reinterpret_cast<const uint4 *>(up + c) : make_uint4(0, 0, 0, 0);
    }
    da_f16v dq[2][C::MTK];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        da_pin(lse[t]);
        da_pin(dl[t]);
#pragma unroll
        for (int f = 0; f < C::NF; ++f) da_pin(qf[t][f]);
#pragma unroll
        for (int x = 0; x < C::MTK; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[t][x][r] = 0.f;
    }
#pragma unroll
    for (int f = 0; f < C::NFV; ++f) da_pin(uf[f]);

    while (k0 < wg_end) {
        const int kn = next(k0 + KB), code_n = kn < wg_end ? walk.code(a, kn) : 0;
        uint64_t vis_n = ~0ull;
        da_copies_done_barrier();
        da_pin(vis);
        if (code_n == 1) vis_n = bits(kn);
        if (kn < wg_end) issue(kn, buf ^ 1);
        if (code != 2 && k0 < w.lim_hi) {
            const bool cut = k0 + KB > w.lim_lo, masked = cut || code == 1;
            if (cut) vis &= w.limit <= k0 ? 0ull : w.limit >= k0 + 64 ? ~0ull : (1ull << (w.limit - k0)) - 1;
            const uint32_t tk = tile0 + buf * 2 * TILE, tv = tk + TILE;
#pragma unroll 1
            for (int nt = 0; nt < KB / 32; ++nt) {
                const uint32_t at = nt * 32 * C::ROWB;
                da_dq_tile<T, DK>(a, dq, qf, uf, lse, dl, sign, ln, tk + at, tv + at, masked, (uint32_t)(vis >> (32 * nt)), lane);
            }
        }
        k0 = kn;
        code = code_n;
        vis = vis_n;
        buf ^= 1;
    }
    const DiffArgs &e = da_again();
    __syncthreads();                                          // every wave is done with the tiles
    const DaRowsOut<T, C::DV> rows{lds + wave * 32 * C::DV * C::ES};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < C::MTK; ++x)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const int c = x * 32 + 8 * q4 + 4 * h2;       // heads of up to 16 channels: one tile holds both maps' channels, this map's half counts
                if (DK < 32 && c / DK != t) continue;
                rows.put(l32, DK < 32 ? c : t * DK + c, dq[t][x][4 * q4] * e.scale, dq[t][x][4 * q4 + 1] * e.scale, dq[t][x][4 * q4 + 2] * e.scale,
                         dq[t][x][4 * q4 + 3] * e.scale);
            }
    const int w0 = blk0 + wave * 32;
    rows.flush(lane, [&](int r, int c) -> T * {
        const int row = w0 + r, i = da_div_g(e, min(row, R - 1)), t = c / DK;
        c -= t * DK;
        return row < R && c < e.d ? reinterpret_cast<T *>(e.dq) + (((int64_t)b * e.N + i) * e.H + hk * e.G + row - i * e.G) * 2 * e.d + t * e.d + c : nullptr;
    });
}

// ------------------------------------------------------------------------------------------------------------------
// backward, dK and dV: workgroup = (batch, key head, 128 keys, one of kvruns runs of the rows), a wave owns 32 keys with both operands in registers; the
// queries of the group's heads stream through two LDS buffers of QB rows (Q | dU | four statistics), copied while the block in front is worked on.
// The rows' statistics are what the products start from (S at -lse / c, dP at -D_0): they come from LDS straight into the accumulators.
// Both operands and both results of 64-channel heads are 192 registers of 323, one wave per SIMD: vector and matrix work of a tile follow each other, which bounds it.
// Measured: 765 - 900 us at 8192 causal tokens (610 - 720 TFLOP/s), 34 - 37 us at 32 x 492, 73 - 77 us in fp32 at 16 x 396.  Two waves for the same 32 keys, one map each (two waves per
// SIMD, dP worked out twice), took 942 us where this took 901; both mask forms of a tile as code of their own 1140 (the accumulators change places between them).
template <typename T, int DK>
__device__ __forceinline__ void da_dkdv_tile(const DiffArgs &a, da_f16v (*dk)[DaCfg<T, DK>::MTK], da_f16v *dv, const uint4 (*kf)[DaCfg<T, DK>::NF], const uint4 *vf, float sign,
                                             const DaLane<T, DK> &ln, uint32_t tq, uint32_t tu, uint32_t stat, bool masked, uint32_t vis, int lane) {
    using C = DaCfg<T, DK>;
    const float c = a.scale_log2e;
    const int h2 = lane >> 5;
    // a lane's 16 rows' statistics (64 floats of each kind in LDS) are where the sums start: c S_t - lse_t and dP - D_0 come out of the products
    auto stat16 = [&](int kind, da_f16v &x) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const da_u4v y = *(da_lds_u4)(uintptr_t)(stat + (kind * 64 + 8 * q4 + 4 * h2) * 4);
            x[4 * q4] = __uint_as_float(y.x); x[4 * q4 + 1] = __uint_as_float(y.y); x[4 * q4 + 2] = __uint_as_float(y.z); x[4 * q4 + 3] = __uint_as_float(y.w);
        }
    };
    da_f16v dp, s[2], p, dl;
    const uint32_t mine = vis >> (4 * h2);
    uint4 fr[2], sf[C::FPT], pf[C::FPT];
    stat16(2, dp);
    stat16(0, s[0]);
    da_ring<C::NFV + C::NF, 2>([&](int i) { return i < C::NFV ? ln.frag(tu, i) : ln.frag(tq, i - C::NFV); },
                               [&](int i, const uint4 &f) {
                                   if (i < C::NFV) dp = Da<T>::mma(f, vf[i], dp);
                                   else s[0] = Da<T>::mma(f, kf[0][i - C::NFV], s[0]);
                               });
    stat16(1, s[1]);
    fr[0] = ln.frag(tq, C::NF);
    if (C::NF > 1) fr[1] = ln.frag(tq, C::NF + 1);
    if (masked) da_hide(s[0], mine);
    // the first map's vector work between the second's scores, the second's between the first map's products with the queries
    da_between<C::NF>(fr, [&](int i) { return ln.frag(tq, C::NF + i); }, [&](int i, const uint4 &f) { s[1] = Da<T>::mma(f, kf[1][i], s[1]); },
                      [&](int r) {
                          p[r] = da_exp2(s[0][r] * c);
                          s[0][r] = p[r] * dp[r];
                      });
    auto query = [&](int t, int i) { return ln.frag_tr(tq, i / C::MTK, DK < 32 ? 0 : t * (DK / 32) + i % C::MTK); };
    fr[0] = query(0, 0);
    fr[1] = query(0, 1);
    stat16(3, dl);
#pragma unroll
    for (int f = 0; f < C::FPT; ++f) sf[f] = da_pack<T>(s[0], f);
    if (masked) da_hide(s[1], mine);
    da_between<C::FPT * C::MTK>(fr, [&](int i) { return query(0, i); }, [&](int i, const uint4 &f) { dk[0][i % C::MTK] = Da<T>::mma(f, sf[i / C::MTK], dk[0][i % C::MTK]); },
                                [&](int r) {
                                    const float e = da_exp2(s[1][r] * c);
                                    p[r] = fmaf(e, -sign, p[r]);
                                    s[1][r] = e * fmaf(dp[r], -sign, dl[r]);
                                });
#pragma unroll
    for (int f = 0; f < C::FPT; ++f) { sf[f] = da_pack<T>(s[1], f); pf[f] = da_pack<T>(p, f); }
    constexpr int NK = C::FPT * C::MTK;
    da_ring<NK + C::FPT * C::MT, 2>([&](int i) { return i < NK ? query(1, i) : ln.frag_tr(tu, (i - NK) / C::MT, (i - NK) % C::MT); },
                                    [&](int i, const uint4 &f) {
                                        if (i < NK) dk[1][i % C::MTK] = Da<T>::mma(f, sf[i / C::MTK], dk[1][i % C::MTK]);
                                        else dv[(i - NK) % C::MT] = Da<T>::mma(f, pf[(i - NK) / C::MT], dv[(i - NK) % C::MT]);
                                    });
}

__device__ __attribute__((aligned(16))) float da_no_row[4] = {-__builtin_huge_valf(), -__builtin_huge_valf(), 0.f, 0.f};     // statistics of a row that is not there
__device__ __forceinline__ void da_copy4(const void *src, uint32_t lds_addr) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(src), "s"(lds_addr) : "memory");
}

template <typename T, int DK>
__global__ __launch_bounds__(kDaThreads, DK == 16 || (DK == 32 && sizeof(T) == 2) ? 2 : 1) void diff_attn_dkdv_kernel(const DiffArgs a) {
    using C = DaCfg<T, DK>;
    constexpr int QB = 64, TILE = QB * C::ROWB, BUF = 2 * TILE + 4 * QB * 4;       // (BUF: a multiple of 512 bytes)
    extern __shared__ __attribute__((aligned(512))) char lds[];      // (512: DaLane)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h2 = lane >> 5, l32 = lane & 31;
    const int nbh = a.B * a.Hk, bh = blockIdx.x % nbh, rest = blockIdx.x / nbh, run = rest % a.kvruns, blk = rest / a.kvruns, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int len = da_len(a, b);
    const int64_t start = da_start(a, b);
    const int M64 = (a.M + 63) >> 6, N64 = (a.N + 63) >> 6;
    const int kw0 = blk * 128 + wave * 32, key = kw0 + l32;
    const int64_t mb = a.mask_b ? b : 0, bhn = (int64_t)a.B * a.H * a.N;
    const bool klive = key < len;
    bool seen = false;                                        // some row of this run sees the key; else zeros are written, whatever its lanes met
    const bool wlive = kw0 < len;

    uint4 kf[2][C::NF], vf[C::NFV];
    const T *kp = reinterpret_cast<const T *>(a.k) + b * a.ks[0] + (int64_t)key * a.ks[1] + hk * a.ks[2];
    const T *vp = reinterpret_cast<const T *>(a.v) + b * a.vs[0] + (int64_t)key * a.vs[1] + hk * a.vs[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int f = 0; f < C::NF; ++f) {
            const int c = f * Da<T>::KPF + h2 * (Da<T>::KPF / 2);
            kf[t][f] = klive && c < a.d ? *reinterpret_cast<const uint4 *>(kp + t * a.ks[3] + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
    for (int f = 0; f < C::NFV; ++f) {
        const int c = f * Da<T>::KPF + h2 * (Da<T>::KPF / 2);
        vf[f] = klive && c < a.dv ? *reinterpret_cast<const uint4 *>(vp + c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int f = 0; f < 2 * C::NF; ++f) da_pin(kf[f / C::NF][f % C::NF]);
#pragma unroll
    for (int f = 0; f < C::NFV; ++f) da_pin(vf[f]);
    da_f16v dk[2][C::MTK], dv[C::MT];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < C::MTK; ++x) dk[t][x][r] = 0.f;
#pragma unroll
        for (int x = 0; x < C::MT; ++x) dv[x][r] = 0.f;
    }
    // blocks of QB queries that may see a key of this workgroup, head after head: this run's share
    int qt_first = 0;
    if (a.causal) {
        const int64_t f = (int64_t)blk * 128 - start;
        qt_first = f <= 0 ? 0 : f >= a.N ? N64 : (int)f / QB;
    }
    if (blk * 128 >= len) qt_first = N64;
    const int per_head = N64 - qt_first, total = per_head * a.G;
    const int u0 = (int)((int64_t)total * run / a.kvruns), u1 = (int)((int64_t)total * (run + 1) / a.kvruns);
    const int kt0 = blk * 2, kt1 = min(kt0 + 1, M64 - 1);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    DaLane<T, DK> ln;
    ln.init(lane);
    const bool full = a.d == DK && a.dv == C::DV;
    DaCopy<T, DK, QB, kDaThreads> cq, cu;
    cq.init(reinterpret_cast<const T *>(a.q) + b * a.qs[0], a.qs[1], a.qs[3], a.d, true, tid);
    cu.init(reinterpret_cast<const T *>(a.du) + (int64_t)b * a.N * a.H * a.dv, (int64_t)a.H * a.dv, 0, a.dv, false, tid);
    // the mask's tiles along the queries as bit sets, 64 query blocks from qt_first + 64 base on (one per lane): workgroup and wave
    uint64_t need = ~0ull, mixed = 0, hide = 0;
    int base = -1;
    struct Block { int u, g, x; };                            // the run's block u: query block x of the group's head g
    auto skip = [&](Block p, int n) {                         // n blocks on, and on to one that the mask does not leave out
        for (;;) {
            p.u += n;
            p.x += n;
            if (p.x >= per_head) {
                p.x = 0;
                ++p.g;
            }
            if (p.u >= u1 || !a.tiles) return p;
            if (p.x >> 6 != base) {
                base = p.x >> 6;
                const int qt = qt_first + base * 64 + lane;
                bool n = false, m = false, y = true;
                if (qt < N64) {
                    const uint8_t *tp = da_again().tiles + (mb * N64 + qt) * M64;
                    const int c = wlive ? tp[kw0 >> 6] : 2;
                    n = tp[kt0] != 2 || tp[kt1] != 2;
                    m = c == 1;
                    y = c == 2;
                }
                need = __ballot(n); mixed = __ballot(m); hide = __ballot(y);
            }
            const uint64_t m = need >> (p.x & 63);
            if (m & 1) return p;
            n = m ? __builtin_ctzll(m) : min(64 - (p.x & 63), per_head - p.x);
        }
    };
    auto code_of = [&](const Block &p) {
        if (!a.tiles || p.u >= u1) return 0;
        const int x = p.x & 63;
        return (int)((mixed >> x) & 1 ? 1 : (hide >> x) & 1 ? 2 : 0);
    };
    auto bits = [&](const Block &p) { return klive ? da_again().colbits[(mb * a.M + key) * N64 + qt_first + p.x] : 0ull; };
    const float *stat0 = a.rowstat + ((int64_t)b * a.H + hk * a.G) * a.N, *stat_w = stat0 + wave * bhn;     // of the group's first head; the wave's kind
    auto row_lse = [&](const Block &p) {                      // -lse of this lane's row of the block: -inf where it sees nothing or is not there
        if (p.u >= u1) return -INFINITY;
        const int i = (qt_first + p.x) * QB + lane;
        return i < a.N ? stat0[p.g * a.N + i] : -INFINITY;
    };
    const int64_t step_q = QB * a.qs[1], step_u = QB * (int64_t)a.H * a.dv;
    Block at{0, 0, 0};                                        // the block that the copies stand at, from the head's first query block that counts
    cq.move((int64_t)qt_first * step_q + hk * a.G * a.qs[2]);
    cu.move((int64_t)qt_first * step_u + hk * a.G * (int64_t)a.dv);
    auto issue = [&](const Block &p, int buf, float lse) {
        const int i0 = (qt_first + p.x) * QB, valid = a.N - i0;
        const uint64_t rows = __ballot(lse != -INFINITY);     // rows that see nothing: their queries may hold anything, zeros are copied
        const uint32_t to = lds0 + buf * BUF;
        if (p.g == at.g && p.x == at.x + 1) {
            cq.move(step_q);
            cu.move(step_u);
        } else {
            const DiffArgs &e = da_again();
            cq.move((p.x - at.x) * step_q + (p.g - at.g) * e.qs[2]);
            cu.move((p.x - at.x) * step_u + (p.g - at.g) * (int64_t)e.dv);
        }
        at = p;
        cq.run(to + wave * 1024, valid, rows, rows == ~0ull, full);
        cu.run(to + TILE + wave * 1024, valid, rows, rows == ~0ull, full);
        da_copy4(lane < valid ? stat_w + (p.g * a.N + i0 + lane) : da_no_row + wave, __builtin_amdgcn_readfirstlane(to + 2 * TILE + wave * QB * 4));
    };
    Block now = skip(Block{u0, per_head ? u0 / per_head : 0, per_head ? u0 % per_head : 0}, 0);
    int buf = 0, g_now = -1, code = code_of(now);
    float sign = 1.f;
    uint64_t vis = code == 1 ? bits(now) : ~0ull;
    if (now.u < u1) issue(now, 0, row_lse(now));
    Block then = skip(now, 1);
    int code_n = code_of(then);
    float lse_n = row_lse(then);
    while (now.u < u1) {
        const int i0 = (qt_first + now.x) * QB;
        if (now.g != g_now) {
            g_now = now.g;
            sign = da_lambda(a, hk * a.G + g_now) < 0.f ? -1.f : 1.f;
        }
        da_copies_done_barrier();                             // the block is there for every wave, and every wave is done with the buffer in front
        da_pin(vis);
        da_pin(lse_n);
        const Block third = skip(then, 1);
        const int code_nn = code_of(third);
        const float lse_nn = row_lse(third);                  // (one block ahead of its use: the rows that the next copies leave out)
        const uint64_t vis_n = code_n == 1 && then.u < u1 ? bits(then) : ~0ull;
        if (then.u < u1) issue(then, buf ^ 1, lse_n);
        if (wlive && code != 2) {
            const uint32_t tq = lds0 + buf * BUF, tu = tq + TILE, stat = tu + TILE;
#pragma unroll 1
            for (int nt = 0; nt < QB / 32; ++nt) {
                const int i1 = i0 + nt * 32;
                if (i1 >= a.N || (a.causal && start + i1 + 31 < kw0)) continue;
                const bool cut = a.causal && start + i1 < kw0 + 31;
                uint32_t v = (uint32_t)(vis >> (32 * nt));
                if (cut) {                                    // query i1 + n sees this key from n >= key - start - i1 on
                    const int64_t n0 = (int64_t)key - start - i1;
                    v &= n0 <= 0 ? ~0u : n0 >= 32 ? 0u : ~0u << n0;
                }
                seen = seen || v;
                const uint32_t at = nt * 32 * C::ROWB;
                da_dkdv_tile<T, DK>(a, dk, dv, kf, vf, sign, ln, tq + at, tu + at, stat + nt * 128, cut || code == 1, v, lane);
            }
        }
        now = then; then = third; lse_n = lse_nn;
        code = code_n; code_n = code_nn;
        vis = vis_n;
        buf ^= 1;
    }
    const DiffArgs &e = da_again();
    __syncthreads();                                          // every wave is done with the tiles
    const bool keep = klive && seen;
    const float f = keep ? e.scale : 0.f;
    const int64_t k0 = (int64_t)b * e.M;
    const int w = 2 * e.d + e.dv;
    auto out = [&](auto rows, auto dkv) {                     // dV, then dK, as whole rows; dkv(key): where the key's dK row starts, dV behind it or in its own tensor
#pragma unroll
        for (int x = 0; x < C::MT; ++x)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                rows.put(l32, x * 32 + 8 * q4 + 4 * h2, keep ? dv[x][4 * q4] : 0.f, keep ? dv[x][4 * q4 + 1] : 0.f, keep ? dv[x][4 * q4 + 2] : 0.f, keep ? dv[x][4 * q4 + 3] : 0.f);
        rows.flush(lane, [&](int r, int c) { return kw0 + r < e.M && c < e.dv ? dkv(kw0 + r, 1) + c : nullptr; });
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < C::MTK; ++x)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const int c = x * 32 + 8 * q4 + 4 * h2;
                    if (DK < 32 && c / DK != t) continue;
                    rows.put(l32, DK < 32 ? c : t * DK + c, keep ? dk[t][x][4 * q4] * f : 0.f, keep ? dk[t][x][4 * q4 + 1] * f : 0.f, keep ? dk[t][x][4 * q4 + 2] * f : 0.f,
                             keep ? dk[t][x][4 * q4 + 3] * f : 0.f);
                }
        rows.flush(lane, [&](int r, int c) {
            const int t = c / DK;
            c -= t * DK;
            return kw0 + r < e.M && c < e.d ? dkv(kw0 + r, 0) + t * e.d + c : nullptr;
        });
    };
    if (e.kvpart) {
        float *part = e.kvpart + (int64_t)run * e.B * e.M * e.Hk * w;
        out(DaRowsOut<float, C::DV>{lds + wave * 32 * C::DV * 4}, [&](int key, int v) { return part + ((k0 + key) * e.Hk + hk) * w + v * 2 * e.d; });
    } else {
        out(DaRowsOut<T, C::DV>{lds + wave * 32 * C::DV * C::ES}, [&](int key, int v) {
            return v ? reinterpret_cast<T *>(e.dvv) + ((k0 + key) * e.Hk + hk) * e.dv : reinterpret_cast<T *>(e.dk) + ((k0 + key) * e.Hk + hk) * 2 * e.d;
        });
    }
}

// dK and dV from the runs' sums, in order: a thread per 4 channels.  Bound: HBM (14 us for 67 MB at 8192 tokens).
template <typename T> __global__ __launch_bounds__(256) void diff_attn_kv_sum_kernel(const DiffArgs a) {
    const int w4 = (2 * a.d + a.dv) / 4;
    const int64_t rows = (int64_t)a.B * a.M * a.Hk, n = rows * w4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / w4;
        const int c = (int)(i - row * w4) * 4;
        float4 v = *reinterpret_cast<const float4 *>(a.kvpart + i * 4);
        for (int r = 1; r < a.kvruns; ++r) {
            const float4 z = *reinterpret_cast<const float4 *>(a.kvpart + (r * n + i) * 4);
            v.x += z.x; v.y += z.y; v.z += z.z; v.w += z.w;
        }
        if (c < 2 * a.d) da_store4(reinterpret_cast<T *>(a.dk) + row * 2 * a.d + c, v.x, v.y, v.z, v.w);
        else da_store4(reinterpret_cast<T *>(a.dvv) + row * a.dv + c - 2 * a.d, v.x, v.y, v.z, v.w);
    }
}

}  // namespace dfine

using namespace dfine;

extern "C" {

static int diff_attn_setup(DiffArgs &a, const int64_t *s, float scale, float init, float eps) {
    // shape: see include/dfine_hip.h
    const int64_t B = s[0], N = s[1], M = s[2], H = s[3], Hk = s[4], d = s[5], dv = s[6], dt = s[7];
    if (B < 0 || N < 0 || M < 0 || B > 0xffffff || N > 0x3fffffff || M > 0x3fffffff || H < 1 || Hk < 1 || H > 4096 || H % Hk || d < 8 || d > 64 || d % 8 || dv < 8 ||
        dv > 128 || dv % 8 || (dt != 0 && dt != 1) || !(scale >= 1e-30f) || !(eps >= 0.f))
        return DFINE_E_BADARG;
    if (s[8] != 1 && s[8] != H) return DFINE_E_BADARG;                               // heads of the learned vectors
    if (N * (H / Hk) > 0x7fffff00 || B * Hk > 0xffffff) return DFINE_E_BADARG;       // (rows of a key head: 32-bit)
    a.B = (int)B; a.N = (int)N; a.M = (int)M; a.H = (int)H; a.Hk = (int)Hk; a.G = (int)(H / Hk); a.d = (int)d; a.dv = (int)dv;
    a.g_shift = 0;
    while ((1 << a.g_shift) < a.G) ++a.g_shift;
    a.g_mul = (uint32_t)((((uint64_t)1 << (31 + a.g_shift)) + a.G - 1) / a.G);
    a.lam_heads = (int)s[8]; a.lam_bf16 = s[9] != 0; a.w_bf16 = s[10] != 0;
    a.causal = s[11] != 0; a.qstart = s[12]; a.mask_b = s[13];
    const int unit = dt == 0 ? 4 : 8;                                                // elements of a 16-byte load
    for (int j = 0; j < 4; ++j) { a.qs[j] = s[14 + j]; a.ks[j] = s[18 + j]; if (j < 3) { a.vs[j] = s[22 + j]; a.dys[j] = s[25 + j]; } }
    for (int j = 14; j < 28; ++j) if (s[j] % unit) return DFINE_E_BADARG;
    a.scale = scale; a.scale_log2e = scale * 1.44269504088896340736f; a.init = init; a.eps = eps;
    return DFINE_OK;
}

static bool diff_attn_aligned(const void *p) { return p && ((uintptr_t)p & 15) == 0; }

int64_t dfine_diff_attn_mask_words(int64_t batches, int64_t N, int64_t M) {
    if (batches < 0 || N < 0 || M < 0) return -1;
    const int64_t M64 = (M + 63) / 64, N64 = (N + 63) / 64;
    return batches * (N * M64 + M * N64 + N64 * M64) + (batches * N64 * M64 + 7) / 8;
}

static void diff_attn_forms(DiffArgs &a, const uint64_t *forms, int64_t batches) {
    if (!forms) return;
    const int64_t M64 = (a.M + 63) / 64, N64 = (a.N + 63) / 64;
    a.rowbits = forms;
    a.colbits = forms + batches * a.N * M64;
    a.some = a.colbits + batches * a.M * N64;
    a.tiles = reinterpret_cast<const uint8_t *>(a.some + batches * N64 * M64);
}

int dfine_diff_attn_mask(const uint8_t *mask, int64_t batches, int64_t N, int64_t M, int64_t stride_b, int64_t stride_n, uint64_t *forms, void *stream) {
    if (batches < 0 || N < 0 || M < 0 || N > 0x3fffffff || M > 0x3fffffff || batches > 0xffffff) return DFINE_E_BADARG;
    if (batches == 0 || N == 0 || M == 0) return DFINE_OK;
    if (!mask || !forms) return DFINE_E_BADARG;
    const int64_t M64 = (M + 63) / 64, N64 = (N + 63) / 64;
    if (batches * M64 * N64 > 0x7fffffff) return DFINE_E_BADARG;
    uint64_t *col = forms + batches * N * M64, *some = col + batches * M * N64;
    hipLaunchKernelGGL(diff_attn_mask_kernel, dim3((unsigned)(batches * M64 * N64)), dim3(256), 0, (hipStream_t)stream, mask, stride_b, stride_n, (int)N, (int)M, forms, col,
                       some, reinterpret_cast<uint8_t *>(some + batches * N64 * M64));
    return check_launch();
}

// the smallest of the three sizes that holds the head (values are twice as wide as a map's channels)
static int diff_attn_size(int d, int dv) { return d <= 16 && dv <= 32 ? 16 : d <= 32 && dv <= 64 ? 32 : 64; }

// dispatch on type and size; ROWS16, ROWS32: rows of 2 DK channels in LDS, MORE: bytes beside them; DA_ARGS: the kernel's arguments
#define DA_LAUNCH(K_, BYTES)                                                                                                                                      \
    {                                                                                                                                                            \
        const int by_ = (int)(BYTES);                                                                                                                            \
        if (by_ > 64 * 1024) {                                                                                                                                   \
            if (hipError_t e_ = hipFuncSetAttribute(reinterpret_cast<const void *>(K_), hipFuncAttributeMaxDynamicSharedMemorySize, by_); e_ != hipSuccess) {    \
                set_last_error(e_);                                                                                                                              \
                return DFINE_E_LAUNCH;                                                                                                                           \
            }                                                                                                                                                    \
        }                                                                                                                                                        \
        hipLaunchKernelGGL(K_, grid_, block_, by_, st_, DA_ARGS);                                                                                                \
    }
#define DA_DISPATCH(KERNEL, GRID, ROWS16, ROWS32, MORE)                                                                                                                \
    {                                                                                                                                                            \
        const int dk_ = diff_attn_size(a.d, a.dv);                                                                                                               \
        const dim3 grid_(GRID), block_(kDaThreads);                                                                                                              \
        hipStream_t st_ = (hipStream_t)stream;                                                                                                                   \
        if (shape[7] == 0) {                                                                                                                                     \
            if (dk_ == 16) DA_LAUNCH((KERNEL<float, 16>), (ROWS32) * 128 + (MORE))                                                                                        \
            else if (dk_ == 32) DA_LAUNCH((KERNEL<float, 32>), (ROWS32) * 256 + (MORE))                                                                                   \
            else DA_LAUNCH((KERNEL<float, 64>), (ROWS32) * 512 + (MORE))                                                                                                  \
        } else {                                                                                                                                                 \
            if (dk_ == 16) DA_LAUNCH((KERNEL<uint16_t, 16>), (ROWS16) * 64 + (MORE))                                                                                      \
            else if (dk_ == 32) DA_LAUNCH((KERNEL<uint16_t, 32>), (ROWS16) * 128 + (MORE))                                                                                \
            else DA_LAUNCH((KERNEL<uint16_t, 64>), (ROWS16) * 256 + (MORE))                                                                                               \
        }                                                                                                                                                        \
    }

// Runs of the keys a forward pass is cut into: 0 = the kernel for many rows (128 rows per workgroup, all keys), n >= 1 = the kernel for few (32 rows per
// workgroup, n runs).
// kDaManyRows: many rows are those that make 256 workgroups (one per CU).  us of the kernel for many and the one for few, forward without results for the backward,
// 4 heads, at 64 / 128 / 160 / 192 / 224 / 256 / 512 workgroups of 128 rows: 492 tokens of 2 x 32 bf16 19 and 11 / 20 and 14 / 20 and 21 / 20 and 21 / 20 and 24 / 20 and
// 24 / 27 and 45; 512 tokens of 2 x 64 bf16 24 and 15 / 24 and 28 / 24 and 40 / 24 and 40 / 25 and 52 / 25 and 53 / 41 and 111; 396 tokens of 2 x 32 fp32 54 and 24 / 55
// and 46 / 54 and 67 / 55 and 68 / 55 and 68 / 55 and 89 / 94 and 161.  The choice holds from 256 on and up to 64; from about 150 on (wide heads: from
// fewer than 128) the kernel for many is the faster already.
// kDaSplitWgs: the runs fill the chip once, 256 workgroups.  One token over 16 caches of 32768 keys (4 key heads): 170 / 177 / 184 / 212 us with 256 / 512 / 1024 /
// 2048 workgroups; 17 tokens over 4 x 10001 keys 36 / 46 / 66 us with 256 / 512 / 1024: every run costs a prologue, its sums and a share of the join.
// kDaRunKeys: a run has 256 keys at least (two tiles for each of its four waves): one token of 16 heads over 4096 keys, runs + join, 19.4 / 19.5 / 21.5 / 26.8 / 35.9 us
// with runs of 128 / 256 / 512 / 1024 / 2048 keys.
// kDaOneRun: up to 1024 keys stay one run (8 us and 4.9 for every 512 keys, against 10.7 and a join of 8): 300 tokens of one image 10.6 us, in two runs 15.0.
static int diff_attn_splits(const DiffArgs &a) {
    const int64_t R = (int64_t)a.N * a.G, bh = (int64_t)a.B * a.Hk;
    if ((R + 127) / 128 * bh >= kDaManyRows) return 0;
    if (a.M <= kDaOneRun) return 1;
    const int64_t wgs = (R + 31) / 32 * bh, most = ((int64_t)a.M + kDaRunKeys - 1) / kDaRunKeys;
    int64_t n = kDaSplitWgs / wgs;
    if (n > most) n = most;
    if (n > 256) n = 256;
    return (int)(n < 1 ? 1 : n);
}

static int64_t da_up(int64_t x) { return (x + 255) / 256 * 256; }
static int64_t diff_attn_rows(const DiffArgs &a) { return (int64_t)a.N * a.G * a.B * a.Hk; }
int64_t dfine_diff_attn_fwd_ws_bytes(const int64_t *shape) {
    DiffArgs a{};
    if (!shape || diff_attn_setup(a, shape, 1.f, 0.f, 0.f)) return -1;
    if (a.B == 0 || a.N == 0) return 0;
    const int n = diff_attn_splits(a);
    return n <= 1 ? 0 : da_up(diff_attn_rows(a) * n * 16) + diff_attn_rows(a) * n * 16 * diff_attn_size(a.d, a.dv);
}

int dfine_diff_attn_fwd(const void *q, const void *k, const void *v, const void *lam, const void *weight, const uint64_t *mask_forms, const int *kv_len,
                        const int *q_start, void *out, float *u, void *o2, float *stats, void *ws, const int64_t *shape, float scale, float init, float eps, void *stream) {
    if (!shape) return DFINE_E_BADARG;
    DiffArgs a{};
    if (int e = diff_attn_setup(a, shape, scale, init, eps)) return e;
    if (a.B == 0 || a.N == 0) return DFINE_OK;
    if (!diff_attn_aligned(q) || !diff_attn_aligned(out) || !lam || (a.M && (!diff_attn_aligned(k) || !diff_attn_aligned(v)))) return DFINE_E_BADARG;
    if ((o2 != nullptr) != (stats != nullptr) || (o2 != nullptr) != (u != nullptr) || (o2 && (!diff_attn_aligned(o2) || !diff_attn_aligned(u)))) return DFINE_E_BADARG;
    a.q = q; a.k = k; a.v = v; a.lam = lam; a.weight = weight; a.kvlen = kv_len; a.qstart_dev = q_start;
    a.out = out; a.u = u; a.o2 = o2; a.stats = stats;
    a.post = weight ? 1.f - init : 1.f;
    diff_attn_forms(a, mask_forms, a.mask_b ? a.B : 1);
    const int n = diff_attn_splits(a);
    const int64_t R = (int64_t)a.N * a.G, blocks = n ? (R + 31) / 32 * a.B * a.Hk * n : (R + 127) / 128 * a.B * a.Hk;
    if (blocks > 0x7fffffff) return DFINE_E_BADARG;
    if (n == 0) {
        #define DA_ARGS a
        DA_DISPATCH(diff_attn_fwd_kernel, (unsigned)blocks, 256, 128, 0)
#undef DA_ARGS
        return check_launch();
    }
    if (n > 1 && (!ws || ((uintptr_t)ws & 255))) return DFINE_E_BADARG;
    float4 *ml = reinterpret_cast<float4 *>(ws);
    float *part = n > 1 ? reinterpret_cast<float *>(reinterpret_cast<char *>(ws) + da_up(diff_attn_rows(a) * n * 16)) : nullptr;
#define DA_ARGS a, n, part, ml
    DA_DISPATCH(diff_attn_fwd_split_kernel, (unsigned)blocks, 512, dk_ == 64 ? 256 : 512, 0)
#undef DA_ARGS
    if (int e = check_launch()) return e;
    if (n == 1) return DFINE_OK;
    const int64_t joins = (diff_attn_rows(a) + 3) / 4;
    if (joins > 0x7fffffff) return DFINE_E_BADARG;
    const int dk = diff_attn_size(a.d, a.dv);
    const dim3 grid((unsigned)joins), block(kDaThreads);
    hipStream_t st = (hipStream_t)stream;
#define DA_JOIN(T_, DV_) hipLaunchKernelGGL((diff_attn_join_kernel<T_, DV_>), grid, block, 0, st, a, n, (const float *)part, (const float4 *)ml)
    if (shape[7] == 0) { if (dk == 16) DA_JOIN(float, 32); else if (dk == 32) DA_JOIN(float, 64); else DA_JOIN(float, 128); }
    else { if (dk == 16) DA_JOIN(uint16_t, 32); else if (dk == 32) DA_JOIN(uint16_t, 64); else DA_JOIN(uint16_t, 128); }
#undef DA_JOIN
    return check_launch();
}

// Workgroups per head of the first backward kernel: 1024 in all, one pass over their rows each at least.  Kernel us at 512 / 1024 / 2048 / 4096: 42 / 33 / 38 / 44 for
// 8192 tokens of 16 heads of 128 channels, 14.2 / 13.5 / 17.2 / 17.4 for 32 x 492 tokens of 4 heads of 64, 11.2 / 11.9 / 10.6 / 11.6 for 16 x 396 in fp32.
static int diff_attn_runs(const DiffArgs &a) {
    const int64_t rw = 2048 / (2 * diff_attn_size(a.d, a.dv)), rows = ((int64_t)a.B * a.N + rw - 1) / rw;       // rows of one pass of a workgroup
    int64_t n = 1024 / a.H;
    if (n < 1) n = 1;
    return (int)(n < rows ? n : rows < 1 ? 1 : rows);
}

// Runs of the rows that dK and dV are summed in, about 512 workgroups in all, each with four blocks of queries at least.  Measured, kernel + sum kernel in us:
// 8192 causal tokens of 4 key heads, bf16 (256 workgroups of very unequal work) 1543 with one run, 898 + 14 with 2, 905 + 23 with 4, 945 + 54 with 8 (one card);
// 32 x 492 tokens of 4 heads (512 workgroups) 37 with one, 45 + 13 with 2; 16 x 396 tokens of 4 heads in fp32 (256 workgroups, 7 blocks of queries) 77 with
// one, 89 + 8 with 2, 105 + 12 with 4.
static int diff_attn_kvruns(const DiffArgs &a) {
    const int64_t wgs = ((int64_t)a.M + 127) / 128 * a.B * a.Hk, units = ((int64_t)a.N + 63) / 64 * a.G;
    if (wgs == 0) return 1;
    int64_t n = 512 / wgs;
    if (n > 8) n = 8;
    if (n > units / 4) n = units / 4;
    return (int)(n < 1 ? 1 : n);
}
// workspace of the backward pass: dU, the rows' statistics, the partial sums of dl and dg, the runs' sums of dK and dV
int64_t dfine_diff_attn_bwd_ws_bytes(const int64_t *shape) {
    DiffArgs a{};
    if (!shape || diff_attn_setup(a, shape, 1.f, 0.f, 0.f)) return -1;
    const int64_t rows = (int64_t)a.B * a.N * a.H, n = (int64_t)diff_attn_runs(a) * a.H, runs = diff_attn_kvruns(a);
    return da_up(rows * a.dv * (shape[7] ? 2 : 4)) + da_up(rows * 16) + da_up(n * 4) + da_up(n * a.dv * 4) +
           (runs > 1 ? runs * a.B * a.M * a.Hk * (2 * a.d + a.dv) * 4 : 0);
}

#define DA_ARGS a
int dfine_diff_attn_bwd(const void *q, const void *k, const void *v, const void *lam, const void *weight, const uint64_t *mask_forms, const int *kv_len,
                        const int *q_start, const float *u, const void *o2, const float *stats, const void *dy, void *dq, void *dk, void *dv,
                        void *dlam, void *dweight, void *ws, const int64_t *shape, float scale, float init, float eps, void *stream) {
    if (!shape) return DFINE_E_BADARG;
    DiffArgs a{};
    if (int e = diff_attn_setup(a, shape, scale, init, eps)) return e;
    if (!lam || !ws || ((uintptr_t)ws & 255)) return DFINE_E_BADARG;
    const bool rows_ = a.B && a.N, keys_ = a.B && a.M;
    if (rows_ && (!diff_attn_aligned(q) || !diff_attn_aligned(u) || !diff_attn_aligned(o2) || !stats || !diff_attn_aligned(dy) ||
                  (dq && !diff_attn_aligned(dq))))
        return DFINE_E_BADARG;
    if ((dk == nullptr) != (dv == nullptr)) return DFINE_E_BADARG;
    if (keys_ && (!diff_attn_aligned(k) || !diff_attn_aligned(v) || (dk && (!diff_attn_aligned(dk) || !diff_attn_aligned(dv))))) return DFINE_E_BADARG;
    a.q = q; a.k = k; a.v = v; a.lam = lam; a.weight = weight; a.kvlen = kv_len; a.qstart_dev = q_start;
    a.u = const_cast<float *>(u); a.o2 = const_cast<void *>(o2); a.stats = const_cast<float *>(stats);
    a.dy = dy; a.dq = dq; a.dk = dk; a.dvv = dv;
    a.post = weight ? 1.f - init : 1.f;
    diff_attn_forms(a, mask_forms, a.mask_b ? a.B : 1);
    const int nrun = diff_attn_runs(a);
    const int64_t rows = (int64_t)a.B * a.N * a.H, n = (int64_t)nrun * a.H;
    char *p = reinterpret_cast<char *>(ws);
    a.du = p; p += da_up(rows * a.dv * (shape[7] ? 2 : 4));
    a.rowstat = reinterpret_cast<float *>(p); p += da_up(rows * 16);
    a.lpart = reinterpret_cast<float *>(p); p += da_up(n * 4);
    a.wpart = reinterpret_cast<float *>(p); p += da_up(n * a.dv * 4);
    a.kvruns = diff_attn_kvruns(a);
    a.kvpart = a.kvruns > 1 ? reinterpret_cast<float *>(p) : nullptr;
    hipStream_t st = (hipStream_t)stream;
    if (n > 0x7fffffff) return DFINE_E_BADARG;
    const int dk_ = diff_attn_size(a.d, a.dv);
#define DA_PREP(T_, L_) hipLaunchKernelGGL((diff_attn_prep_kernel<T_, L_>), dim3((unsigned)n), dim3(256), 0, st, a, nrun)
    if (shape[7] == 0) { if (dk_ == 16) DA_PREP(float, 4); else if (dk_ == 32) DA_PREP(float, 8); else DA_PREP(float, 16); }
    else { if (dk_ == 16) DA_PREP(uint16_t, 4); else if (dk_ == 32) DA_PREP(uint16_t, 8); else DA_PREP(uint16_t, 16); }
#undef DA_PREP
    if (int e = check_launch()) return e;
    if (dlam || dweight) {
        const int nh = a.lam_heads == 1 ? 1 : a.H;
        hipLaunchKernelGGL(diff_attn_param_kernel, dim3(nh + (a.dv + 31) / 32), dim3(1024), 0, st, a, nrun, dlam, weight ? dweight : nullptr);
        if (int e = check_launch()) return e;
    }
    if (rows_ && dq) {
        const int64_t blocks = ((int64_t)a.N * a.G + 127) / 128 * a.B * a.Hk;
        if (blocks > 0x7fffffff) return DFINE_E_BADARG;
        DA_DISPATCH(diff_attn_dq_kernel, (unsigned)blocks, 256, 128, 0)
        if (int e = check_launch()) return e;
    }
    if (keys_ && dk) {
        const int64_t blocks = ((int64_t)a.M + 127) / 128 * a.B * a.Hk * a.kvruns;
        if (blocks > 0x7fffffff) return DFINE_E_BADARG;
        DA_DISPATCH(diff_attn_dkdv_kernel, (unsigned)blocks, 256, 256, 2 * 4 * 64 * 4)
        if (int e = check_launch()) return e;
        if (a.kvruns > 1) {
            const int64_t grid = ((int64_t)a.B * a.M * a.Hk * (2 * a.d + a.dv) / 4 + 255) / 256;
            if (shape[7] == 0) hipLaunchKernelGGL(diff_attn_kv_sum_kernel<float>, dim3((unsigned)(grid < 4096 ? grid : 4096)), dim3(256), 0, st, a);
            else hipLaunchKernelGGL(diff_attn_kv_sum_kernel<uint16_t>, dim3((unsigned)(grid < 4096 ? grid : 4096)), dim3(256), 0, st, a);
            if (int e = check_launch()) return e;
        }
    }
    return DFINE_OK;
}
#undef DA_ARGS
#undef DA_DISPATCH
#undef DA_LAUNCH

}  // extern "C"
