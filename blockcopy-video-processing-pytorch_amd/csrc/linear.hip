// linear.hip -- rows x weights products with the whole epilogue in the kernel, and their gradients.  Part of libblockcopy_hip.so.
//
//   forward     z[m][n] = sum_k x[m][k] w[n][k] + bias[n]          y[m][n] = act(z[m][n]) + residual[m][n]
//   backward    dz = dy * act'(z)     dx[m][k] = sum_n dz[m][n] w[n][k]     dw[n][k] = sum_m dz[m][n] x[m][k]     db[n] = sum_m dz[m][n]
//
// A row is one pixel of a channels-last map (or one token), its features are the map's channels; bc_conv1x1_nhwc is the inference form of the
// same product for packed channel counts, with per-channel affine records around it.  The three products are ONE kernel (k_lin_gemm) over
// operands that either run along the summed index (KC) or across it (MC).  Sums, pre-activations and epilogue are fp32.  Nothing but results
// is rounded to the tensors' type: z is stored in fp32, and a 16-bit dz as two numbers of the type, one after the other through the same
// product (LinParts).  With one number each, z's and dz's roundings made the gradients' error 1.45 times that of rounding the result alone.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "../../include/blockcopy_hip.h"

#define BC_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 *lds_s16x4_ptr;

enum { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };      // the dtype codes of the C ABI

// V elements make 16 bytes
template <int DT> struct LinT { typedef float S; static constexpr int V = 4; };
template <> struct LinT<DT_F16> { typedef _Float16 S; static constexpr int V = 8; };
template <> struct LinT<DT_BF16> { typedef __bf16 S; static constexpr int V = 8; };

inline int lin_status()
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BC_OK : (int)e;
}

// ------------------------------------------------------------------------------------------------------------------ activations
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4, ACT_COUNT = 5 };

// sigmoid(v) = 1 / (1 + e^-v).  fp32 tensors take the library's exponential and the rounded division; for 16-bit ones (result off by 2^-9 or 2^-11
// anyway) the hardware's exp2 and reciprocal, each good to one unit in the last place of fp32: 4 instructions instead of about 25
template <int DT> __device__ __forceinline__ float lin_sigmoid(float v)
{
    if constexpr (DT == DT_F32) return 1.f / (1.f + expf(-v));
    else return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
}

// Phi(z) = erfc(-z / sqrt 2) / 2 and e = exp(-z^2 / 2), to float's relative precision in the lower tail too (1 + erf would cancel there).  16-bit
// tensors: with x = |z| / sqrt 2 and t = 1 / (1 + p x), exp(x^2) erfc(x) / 2 = t Q(t) for 0 <= t <= 1; Q of degree 7 and p = 0.46 by a weighted minimax fit
// (linear program over 1200 Chebyshev points), off by at most 7e-7 of the value, 1e-6 as evaluated -- 17 instructions, and the derivative needs
// the same exponential (a 5-term form of absolute precision, off by 1 % at z = -8: 62.4 us against 63.6 for bf16 17408 x 512 x 2048).  The library's functions are
// several times that: an epilogue of 256 x 256 outputs spent 17 us on erff, more than eight steps of products
template <int DT> __device__ __forceinline__ float lin_phi(float z, float &e)
{
    if constexpr (DT == DT_F32) {
        e = expf(-0.5f * z * z);
        return 0.5f * erfcf(z * -0.70710678118654752f);
    } else {
        e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
        const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.46f * 0.70710678118654752f, 1.f));
        float q = fmaf(t, 0.0338571444f, -0.113314524f);
        q = fmaf(t, q, 0.0845953226f);
        q = fmaf(t, q, 0.026305452f);
        q = fmaf(t, q, 0.0934238359f);
        q = fmaf(t, q, 0.115590952f);
        q = fmaf(t, q, 0.129778638f);
        q = t * e * fmaf(t, q, 0.129763529f);
        return z < 0.f ? q : 1.f - q;
    }
}

// gelu_tanh is z * (1 + tanh(u)) / 2 = z * sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3): one exponential, nothing cancels
constexpr float GELU_A = 0.7978845608028654f, GELU_B = 0.044715f;

template <int DT, int ACT> __device__ __forceinline__ float lin_act1(float z)
{
    float e;
    if constexpr (ACT == ACT_RELU) return z > 0.f || z != z ? z : 0.f;
    else if constexpr (ACT == ACT_GELU) return z * lin_phi<DT>(z, e);
    else if constexpr (ACT == ACT_GELU_TANH) return z * lin_sigmoid<DT>(2.f * GELU_A * z * fmaf(GELU_B * z, z, 1.f));
    else return z * lin_sigmoid<DT>(z);
}

// act'(z).  From +-128 on every derivative is 0 or 1 to the last bit of float (the slowest, silu', differs by |z| e^-|z| < 2^-177 there); the clamp keeps
// 0 * infinity out of the products (NaN passes through)
template <int DT, int ACT> __device__ __forceinline__ float lin_dact1(float z)
{
    const float c = z > 128.f ? 128.f : (z < -128.f ? -128.f : z);
    if constexpr (ACT == ACT_RELU) return z != z ? z : (z > 0.f ? 1.f : 0.f);
    else if constexpr (ACT == ACT_GELU) {
        float e;
        const float p = lin_phi<DT>(c, e);
        return fmaf(c * e, 0.3989422804014327f, p);
    } else if constexpr (ACT == ACT_GELU_TANH) {
        const float s = lin_sigmoid<DT>(2.f * GELU_A * c * fmaf(GELU_B * c, c, 1.f));
        return s + c * s * (1.f - s) * 2.f * GELU_A * fmaf(3.f * GELU_B * c, c, 1.f);
    } else {
        const float s = lin_sigmoid<DT>(c);
        return s * fmaf(c, 1.f - s, 1.f);
    }
}

// W values at once, the choice outside: their chains of dependent instructions run side by side (a choice per value kept them apart: one
// exponential's latency after the other)
template <int DT, int ACT, int W> __device__ __forceinline__ void lin_acts1(float *v)
{
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = lin_act1<DT, ACT>(v[e]);
}

template <int DT, int W> __device__ __forceinline__ void lin_acts(float *v, int act)
{
    switch (act) {
    case ACT_RELU: return lin_acts1<DT, ACT_RELU, W>(v);
    case ACT_GELU: return lin_acts1<DT, ACT_GELU, W>(v);
    case ACT_GELU_TANH: return lin_acts1<DT, ACT_GELU_TANH, W>(v);
    case ACT_SILU: return lin_acts1<DT, ACT_SILU, W>(v);
    }
}

template <int DT, int ACT, int W> __device__ __forceinline__ void lin_dacts1(float *g, const float *z)      // g *= act'(z)
{
#pragma unroll
    for (int e = 0; e < W; ++e) g[e] *= lin_dact1<DT, ACT>(z[e]);
}

template <int DT, int W> __device__ __forceinline__ void lin_dacts(float *g, const float *z, int act)
{
    switch (act) {
    case ACT_RELU: return lin_dacts1<DT, ACT_RELU, W>(g, z);
    case ACT_GELU: return lin_dacts1<DT, ACT_GELU, W>(g, z);
    case ACT_GELU_TANH: return lin_dacts1<DT, ACT_GELU_TANH, W>(g, z);
    case ACT_SILU: return lin_dacts1<DT, ACT_SILU, W>(g, z);
    }
}

// ------------------------------------------------------------------------------------------------------------------ the product
struct LinOperand {
    const void *p;
    long long ld;       // elements between consecutive rows of memory
    int run;            // readable elements of a row of memory
};

struct LinEpi {
    void *y, *z;                // z: the pre-activations (NULL: not kept), in fp32 for an activation with a curve, else in the tensors' type
    const void *bias, *res;
    long long ldr;
    int bias_f32, act;
};

// relu' asks for z's sign alone, and without an activation nothing is asked: the tensors' type will do.  Other derivatives take all of z
__host__ __device__ constexpr bool lin_curved(int act) { return act > ACT_RELU; }

// dz = gy act'(z) of a curved activation in 16 bits: hi + lo.  PRE dz = hi + what is left, lo = LO times that; the sum of products is (hi's + lo's / LO) / PRE.
// Two numbers hold twice the type's bits of any dz: of float16 LO = 2^11 keeps what is left of small values above the subnormal numbers, PRE = 1/2 keeps
// dz (up to 1.13 gy) below the type's end; bfloat16 has float's range and needs neither
template <int DT> struct LinParts { static constexpr float PRE = 1.f, LO = 1.f; };
template <> struct LinParts<DT_F16> { static constexpr float PRE = 0.5f, LO = 2048.f; };

struct LinArgs {
    LinOperand a, b;            // a: the operand of the output's columns (n), b: of its rows (m)
    int M, N, K;
    int kspan;                  // summed indexes of one slice (a multiple of BK): slice s takes [s kspan, (s + 1) kspan)
    unsigned tiles_m, tiles_n;
    float *part;                // [slices][M][N] sums of the slices, or NULL: one slice, epilogue in place
    size_t b_lo;                // bytes from b's data to its lower part (LinParts); 0: one part
    LinEpi ep;
};

template <int DT> __device__ __forceinline__ void lin_mma(f32x4 &d, const uint4 &a, const uint4 &b)
{
    if constexpr (DT == DT_F16)
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
    else if constexpr (DT == DT_BF16)
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), d, 0, 0, 0);
    else {      // fp32: exact products, four k-steps of the 16 x 16 x 4 instruction; lane group g holds k = 4 g + j for step j on both sides
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) d = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[j], fb[j], d, 0, 0, 0);
    }
}

// One staged operand tile: R rows (output rows or columns) x C vectors of 16 bytes along the summed index (C = 8 or 4)
//   KC (memory runs along the summed index): image [row][C vectors], vector c of row r at c ^ lin_turn(r): the 16 rows x 4 vectors that one
//      fragment read touches cover all banks
//   MC (memory runs across it): image [k][R / V vectors], vectors exchanged by lin_swz(k); 16-bit fragments are transposed by the LDS read
//      itself (ds_read_b64_tr_b16: a group of 16 lanes addresses 4 k x 16 rows and lane i receives row i's four k), fp32 ones read word by word
template <int C> __device__ __forceinline__ int lin_turn(int row) { return C == 8 ? row & 7 : (row >> 1) & 3; }

template <int DT, int R> __device__ __forceinline__ int lin_swz(int k)
{
    if constexpr (DT == DT_F32) return ((k >> 2) & 3) * 4;
    else return ((k & 3) * 2 + ((k >> 3) & 1) * 8) & (R / 8 - 1);
}

// place of the tile's v-th vector (in the order of memory: runs of C or of R / V) inside its image
template <int DT, bool MC, int R, int C> __device__ __forceinline__ int lin_place(int v)
{
    constexpr int V = LinT<DT>::V;
    if constexpr (MC) return v / (R / V) * (R / V) + ((v % (R / V)) ^ lin_swz<DT, R>(v / (R / V)));
    else return v / C * C + ((v % C) ^ lin_turn<C>(v / C));
}

template <int DT, bool MC, int R, int C> __device__ __forceinline__ uint4 lin_frag(const uint4 *img, int row0, int ks, int lane)
{
    constexpr int V = LinT<DT>::V, CPR = R / V;
    const int r = lane & 15, g = lane >> 4;
    if constexpr (!MC) {
        const int row = row0 + r;
        return img[row * C + ((ks * 4 + g) ^ lin_turn<C>(row))];
    } else if constexpr (DT == DT_F32) {
        const float *f = (const float *)img;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = ks * 16 + 4 * g + j;
            v[j] = f[k * R + ((((row0 + r) >> 2) ^ lin_swz<DT, R>(k)) << 2) + (r & 3)];
        }
        return uint4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    } else {
        const int k = ks * 32 + 8 * g + (r >> 2), c = (row0 >> 3) + ((r & 3) >> 1);
        const short *s = (const short *)img + ((k * CPR + (c ^ lin_swz<DT, R>(k))) * 8 + (r & 1) * 4);
        const short *t = (const short *)img + (((k + 4) * CPR + (c ^ lin_swz<DT, R>(k + 4))) * 8 + (r & 1) * 4);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)s), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)t);
        const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
        return uint4{a.x, a.y, b.x, b.y};
    }
}

// 16 bytes of an operand starting at (row, k); elements outside the matrix (or the slice, k >= kend) are zero.  The vector asks for the
// alignment of an element only (the hardware takes unaligned vectors): rows may start anywhere
template <int DT, bool MC> __device__ __forceinline__ uint4 lin_fetch(const LinOperand &o, int rows, int kend, int row, int k)
{
    constexpr int V = LinT<DT>::V;
    typedef typename LinT<DT>::S S;
    typedef S SV __attribute__((ext_vector_type(V), aligned(sizeof(S))));
    const int run = MC ? row : k, run_end = MC ? rows : kend;       // the index that memory runs along
    if ((MC ? k >= kend : row >= rows) || run >= run_end) return uint4{0u, 0u, 0u, 0u};
    const S *p = (const S *)o.p + (MC ? (size_t)k * o.ld + row : (size_t)row * o.ld + k);
    SV v;
    if (run + V <= run_end) v = *(const SV *)p;
    else
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = run + e < run_end ? p[e] : (S)0.f;
    return __builtin_bit_cast(uint4, v);
}

// W consecutive elements, of which `cnt` exist (the vector asks for the alignment of an element only)
template <typename S, int W> __device__ __forceinline__ void lin_load(float *f, const S *p, int cnt)
{
    typedef S SW __attribute__((ext_vector_type(W), aligned(sizeof(S))));
    if (cnt >= W) {
        const SW v = *(const SW *)p;
#pragma unroll
        for (int e = 0; e < W; ++e) f[e] = (float)v[e];
    } else
#pragma unroll
        for (int e = 0; e < W; ++e) f[e] = e < cnt ? (float)p[e] : 0.f;
}

template <typename S, int W> __device__ __forceinline__ void lin_save(S *p, const float *f, int cnt)
{
    typedef S SW __attribute__((ext_vector_type(W), aligned(sizeof(S))));
    if (cnt >= W) {
        SW v;
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = (S)f[e];
        *(SW *)p = v;
    } else
#pragma unroll
        for (int e = 0; e < W; ++e)
            if (e < cnt) p[e] = (S)f[e];
}

// W consecutive outputs (m, n ..; 16 bytes' worth), cnt of them inside the matrix: sums v -> z, y.  The bias b and the residual r are loaded by the caller, ahead
template <int DT, int W = LinT<DT>::V> __device__ __forceinline__ void lin_residual(float *r, const LinEpi &ep, int N, int m, int n)
{
    typedef typename LinT<DT>::S S;
    lin_load<S, W>(r, (const S *)ep.res + (size_t)m * ep.ldr + n, N - n);
}

// the bias of W columns (a lane keeps its columns: loaded once)
template <int DT, int W = LinT<DT>::V> __device__ __forceinline__ void lin_bias(float *b, const LinEpi &ep, int N, int n)
{
    typedef typename LinT<DT>::S S;
#pragma unroll
    for (int e = 0; e < W; ++e) b[e] = 0.f;
    if (!ep.bias || n >= N) return;
    if (ep.bias_f32) lin_load<float, W>(b, (const float *)ep.bias + n, N - n);
    else lin_load<S, W>(b, (const S *)ep.bias + n, N - n);
}

// the smallest number above zero
template <int DT> __device__ constexpr float lin_least() { return DT == DT_F16 ? 0x1p-24f : DT == DT_BF16 ? 0x1p-133f : 0x1p-149f; }

template <int DT, int W = LinT<DT>::V> __device__ __forceinline__ void lin_epilogue(const LinEpi &ep, int N, int m, int n, float *v, const float *b, const float *r)
{
    typedef typename LinT<DT>::S S;
    const int cnt = N - n;
    const size_t at = (size_t)m * N + n;
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] += b[e];
    if (ep.z) {
        if (DT == DT_F32 || lin_curved(ep.act)) lin_save<float, W>((float *)ep.z + at, v, cnt);
        else {
            float s[W];         // (a positive z that rounds to 0 stays positive: relu's derivative)
#pragma unroll
            for (int e = 0; e < W; ++e) s[e] = v[e] > 0.f && v[e] < lin_least<DT>() ? lin_least<DT>() : v[e];
            lin_save<S, W>((S *)ep.z + at, s, cnt);
        }
    }
    lin_acts<DT, W>(v, ep.act);
    if (ep.res)
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] += r[e];
    lin_save<S, W>((S *)ep.y + at, v, cnt);
}

// ---- direct copies global -> LDS.  A wave moves 64 x 16 bytes per instruction: lane l's bytes land at lds + 16 l, its source is base + off, so
// an image's exchanged vector order is made by the lanes' source offsets.  The descriptor is a plain range of bytes (no stride, no limit:
// every offset that is used lies inside the matrix).  Written in assembly because the compiler waits for all outstanding copies before any
// LDS read once it sees one; the kernel waits itself (lin_arrived), and there is no register that a copy in flight could overwrite.
typedef int i32x4 __attribute__((ext_vector_type(4)));

// N (1, 2 or 4) of them, STEP bytes apart in the LDS.  The waits are part of the block, the compiler sees none of its instructions: a buffer access
// may come 5 states after a vector instruction wrote one of its scalar registers (a lane read, a reload), and one state after m0 was written
template <int N, int STEP> __device__ __forceinline__ void lin_copy16(const void *base, const unsigned *off, unsigned lds)
{
    static_assert(N == 1 || N == 2 || N == 4, "copies of a block");
    const unsigned long long b = (unsigned long long)base;
    const i32x4 r = {(int)(unsigned)b, (int)(unsigned)(b >> 32) & 0xffff, -1, 0x00027000};
#define LIN_NEXT(V) "\n\ts_add_u32 m0, m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 " V ", %1, 0 offen lds"
    if constexpr (N == 1)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %3, %1, 0 offen lds" : : "s"(lds), "s"(r), "i"(STEP), "v"(off[0]) : "memory", "m0", "scc");
    else if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %3, %1, 0 offen lds" LIN_NEXT("%4")
                     : : "s"(lds), "s"(r), "i"(STEP), "v"(off[0]), "v"(off[1]) : "memory", "m0", "scc");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %3, %1, 0 offen lds" LIN_NEXT("%4") LIN_NEXT("%5") LIN_NEXT("%6")
                     : : "s"(lds), "s"(r), "i"(STEP), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]) : "memory", "m0", "scc");
#undef LIN_NEXT
}

// everything this wave copied is in the LDS and everything it read from there in registers, then all waves meet
__device__ __forceinline__ void lin_meet()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

// out[m][n] = sum_k A(n, k) B(m, k).  A workgroup of WM x WN waves owns a BM x BN tile; the column operand is the matrix instruction's first
// one, so a lane ends up with four consecutive columns of one row.  Two LDS images of a step's operands, C vectors (16 C bytes) of every row:
// while step t is multiplied, step t + 1 travels into the other one, one barrier per step.  DIRECT: operands whose vectors are aligned travel
// global -> LDS without registers (a partial last step goes through registers, zero-filled); otherwise through registers, requested before
// the products and stored behind them.  TWO: the row operand's two parts (LinParts), the sum run over twice, the lower part first.
// Bound: the matrix pipe for long sums (bf16 16384 x 4096 x 8192 with gelu_tanh 880 us = 1250 TFLOP/s, a library product alone 824; the two gradients
// of 8192 x 2048 x 8192 with two parts each 492 and 502 us = 1095 - 1117; fp32 17408 x 768 x 256 64 us = 107 TFLOP/s of 136: 4.25 tiles per CU take the
// time of 5).  Short sums: products, epilogue and stores of a tile follow each other, only the CU's other workgroups overlap them (bf16 17408 x
// 512 x 2048 54 us, with gelu 63.5: vector pipe 43 % of the time, matrix pipe 23 %, waves wait 39 % of theirs for memory and barriers).
// (steps of 64 bytes: 128 registers, so that four workgroups share a CU; with three 131072 x 256 x 512 57 us against 51, with five it spills)
template <int DT, int BM, int BN, int WM, int WN, bool AMC, bool BMC, bool DIRECT, int C, bool TWO>
__global__ __launch_bounds__(64 * WM * WN, C == 4 ? 4 : 1) void k_lin_gemm(const LinArgs g)
{
    constexpr int V = LinT<DT>::V, BK = C * V, NT = 64 * WM * WN, ES = 16 / V;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int NA = BN * C / NT, NB = BM * C / NT;       // vectors per thread and step
    constexpr int IMG = (BM + BN) * C;
    extern __shared__ uint4 lin_lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
    // consecutive workgroups go to the 8 XCDs in turn, each with an L2 of its own: an XCD takes one run of the work (slice by slice, tile by tile),
    // so what its workgroups share is fetched into that L2 once.  Inside a slice tiles go in bands of 8 tile rows
    const unsigned all = gridDim.x, xcd = blockIdx.x & 7u, id = xcd * (all >> 3) + (xcd < (all & 7u) ? xcd : all & 7u) + (blockIdx.x >> 3);
    const unsigned slice = id / (g.tiles_m * g.tiles_n), tile = id - slice * (g.tiles_m * g.tiles_n);
    const unsigned band = 8 * g.tiles_n, b0 = tile / band, in = tile % band;
    const unsigned rows_in_band = g.tiles_m - b0 * 8 < 8 ? g.tiles_m - b0 * 8 : 8;
    const int m0 = (int)(b0 * 8 + in % rows_in_band) * BM, n0 = (int)(in / rows_in_band) * BN;
    const int kbeg = (int)slice * g.kspan, kend = g.K - kbeg < g.kspan ? g.K : kbeg + g.kspan;

    LinOperand rows = g.b;      // (TWO: of the part in hand)

    uint4 ra[NA], rb[NB];
    auto fetch = [&](int k0) {
        int t = tid;
        if constexpr (TWO) asm("" : "+v"(t), "+s"(k0));      // (each part forms its own addresses: kept from part to part they cost a workgroup per CU)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int v = t + NT * i;
            if constexpr (AMC) ra[i] = lin_fetch<DT, true>(g.a, g.N, kend, n0 + v % (BN / V) * V, k0 + v / (BN / V));
            else ra[i] = lin_fetch<DT, false>(g.a, g.N, kend, n0 + v / C, k0 + v % C * V);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int v = t + NT * i;
            if constexpr (BMC) rb[i] = lin_fetch<DT, true>(rows, g.M, kend, m0 + v % (BM / V) * V, k0 + v / (BM / V));
            else rb[i] = lin_fetch<DT, false>(rows, g.M, kend, m0 + v / C, k0 + v % C * V);
        }
    };
    auto stage = [&](uint4 *img) {
#pragma unroll
        for (int i = 0; i < NA; ++i) img[lin_place<DT, AMC, BN, C>(tid + NT * i)] = ra[i];
        img += BN * C;
#pragma unroll
        for (int i = 0; i < NB; ++i) img[lin_place<DT, BMC, BM, C>(tid + NT * i)] = rb[i];
    };
    // direct copies: byte offsets of this lane's sources from the tile's corner of the step.  Rows behind the matrix take its last row
    // (vector) -- their sums are never stored.  The exchange of an image is its own inverse: the vector that belongs at place v is lin_place(v)
    unsigned oa[NA], ob[NB];
    const char *pa = nullptr, *pb = nullptr;
    const size_t stepa = AMC ? (size_t)BK * g.a.ld * ES : 16 * C, stepb = BMC ? (size_t)BK * g.b.ld * ES : 16 * C;
    if constexpr (DIRECT) {
        pa = (const char *)g.a.p + ((AMC ? (size_t)kbeg * g.a.ld + n0 : (size_t)n0 * g.a.ld + kbeg)) * ES;
        pb = (const char *)g.b.p + ((BMC ? (size_t)kbeg * g.b.ld + m0 : (size_t)m0 * g.b.ld + kbeg)) * ES;
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int v = lin_place<DT, AMC, BN, C>(tid + NT * i);
            if constexpr (AMC) {
                const int k = v / (BN / V), c = v % (BN / V), n = n0 + c * V + V <= g.a.run ? c * V : g.a.run - V - n0;
                oa[i] = (unsigned)((long long)k * g.a.ld + n) * ES;
            } else {
                const int row = n0 + v / C < g.N ? v / C : g.N - 1 - n0;
                oa[i] = (unsigned)((long long)row * g.a.ld) * ES + (unsigned)(v % C) * 16;
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int v = lin_place<DT, BMC, BM, C>(tid + NT * i);
            if constexpr (BMC) {
                const int k = v / (BM / V), c = v % (BM / V), m = m0 + c * V + V <= g.b.run ? c * V : g.b.run - V - m0;
                ob[i] = (unsigned)((long long)k * g.b.ld + m) * ES;
            } else {
                const int row = m0 + v / C < g.M ? v / C : g.M - 1 - m0;
                ob[i] = (unsigned)((long long)row * g.b.ld) * ES + (unsigned)(v % C) * 16;
            }
        }
    }
    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char *)lin_lds + wave * 1024;
    auto copy = [&](int img) {      // the next step's operands into image `img`
        lin_copy16<NA, NT * 16>(pa, oa, lds0 + img * IMG * 16);
        lin_copy16<NB, NT * 16>(pb, ob, lds0 + (img * IMG + BN * C) * 16);
        pa += stepa;
        pb += stepb;
    };

    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const uint4 *ia) {
        const uint4 *ib = ia + BN * C;
#pragma unroll
        for (int ks = 0; ks < C / 4; ++ks) {
            uint4 fa[FN], fb[FM];
#pragma unroll
            for (int i = 0; i < FN; ++i) fa[i] = lin_frag<DT, AMC, BN, C>(ia, wn * (BN / WN) + 16 * i, ks, lane);
#pragma unroll
            for (int j = 0; j < FM; ++j) fb[j] = lin_frag<DT, BMC, BM, C>(ib, wm * (BM / WM) + 16 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j) lin_mma<DT>(acc[i][j], fa[i], fb[j]);
        }
    };

    int img = 0;        // (images in turn, also from part to part: the one that is written was last read before the previous barrier)
    auto sum = [&]() {
        if constexpr (DIRECT) {
            const int full = (kend - kbeg) / BK;
            if (full > 0) copy(img);
            for (int t = 0; t < full; ++t) {
                lin_meet();
                if (t + 1 < full) copy(img ^ 1);
                multiply(lin_lds + img * IMG);
                img ^= 1;
            }
            if (kbeg + full * BK < kend) {
                fetch(kbeg + full * BK);
                stage(lin_lds + img * IMG);
                __syncthreads();
                multiply(lin_lds + img * IMG);
                img ^= 1;
            }
        } else {
            fetch(kbeg);
            stage(lin_lds + img * IMG);
            __syncthreads();
            for (int k0 = kbeg; k0 < kend; k0 += BK) {
                const bool more = k0 + BK < kend;
                if (more) fetch(k0 + BK);
                multiply(lin_lds + img * IMG);
                if (more) stage(lin_lds + (img ^ 1) * IMG);
                __syncthreads();
                img ^= 1;
            }
        }
    };
    if constexpr (!TWO) sum();
    else
#pragma nounroll
        for (int part = 1; part >= 0; --part) {
            const size_t lo = part ? g.b_lo : 0;
            rows.p = (const char *)g.b.p + lo;
            if constexpr (DIRECT) {
                pa = (const char *)g.a.p + ((AMC ? (size_t)kbeg * g.a.ld + n0 : (size_t)n0 * g.a.ld + kbeg)) * ES;
                pb = (const char *)rows.p + ((BMC ? (size_t)kbeg * g.b.ld + m0 : (size_t)m0 * g.b.ld + kbeg)) * ES;
            }
            sum();
            // (an infinity or NaN among the operands is the upper part's to answer for: what is left of dz may be 0 or of the other sign)
            const float f = part ? 1.f / LinParts<DT>::LO : 1.f / LinParts<DT>::PRE;
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = part && !__builtin_isfinite(acc[i][j][e]) ? 0.f : acc[i][j][e] * f;
        }

    // the sums meet their epilogue through the LDS: a wave lays RH rows of them (16-byte vector c of row r at c ^ (r & its mask)) into its own
    // part of the images and takes them back row by row, so that every access to memory is a whole 16-byte vector
    constexpr int CW = BN / WN, CPR = CW / 4, FIT = 2 * IMG / (WM * WN * CPR);       // columns of a wave, vectors per row, rows that fit
    constexpr int RH = BM / WM <= FIT && BM / WM <= 64 ? BM / WM : FIT >= 64 ? 64 : FIT >= 32 ? 32 : 16;
    static_assert(FIT >= 16 && (CPR & (CPR - 1)) == 0 && CPR <= 16 && BM / WM % RH == 0, "the images hold the waves' sums");
    constexpr int PER_ROW = CW / V, RPI = 64 / PER_ROW;         // lanes per row, rows per round
    constexpr int AHEAD = RH / RPI < 4 ? RH / RPI : 4;          // rounds whose residuals are requested together
    uint4 *own = lin_lds + wave * (RH * CPR);
    const int n = n0 + wn * CW + (lane % PER_ROW) * V;
    float bias[V];
    lin_bias<DT>(bias, g.ep, g.N, n);
    lin_meet();         // all waves have read the last step
#pragma unroll
    for (int h = 0; h < BM / WM / RH; ++h) {        // (the part is the wave's own and its LDS accesses stay in order: no barrier)
#pragma unroll
        for (int j = 0; j < RH / 16; ++j)
#pragma unroll
            for (int i = 0; i < FN; ++i) own[(16 * j + (lane & 15)) * CPR + ((4 * i + (lane >> 4)) ^ (lane & (CPR - 1)))] = __builtin_bit_cast(uint4, acc[i][RH / 16 * h + j]);
        __builtin_amdgcn_wave_barrier();
        for (int r0 = lane / PER_ROW; r0 < RH; r0 += AHEAD * RPI) {
            float res[AHEAD][V];
            const int mb = m0 + wm * (BM / WM) + RH * h;
            if (g.ep.res && !g.part)
#pragma unroll
                for (int q = 0; q < AHEAD; ++q)
                    if (mb + r0 + q * RPI < g.M && n < g.N) lin_residual<DT>(res[q], g.ep, g.N, mb + r0 + q * RPI, n);
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int r = r0 + q * RPI, m = mb + r;
                if (m >= g.M || n >= g.N) continue;
                float v[V];
#pragma unroll
                for (int p = 0; p < V / 4; ++p) {
                    const f32x4 f = __builtin_bit_cast(f32x4, own[r * CPR + (((lane % PER_ROW) * (V / 4) + p) ^ (r & (CPR - 1)))]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * p + e] = f[e];
                }
                if (g.part) lin_save<float, V>(g.part + ((size_t)slice * g.M + m) * g.N + n, v, g.N - n);
                else lin_epilogue<DT>(g.ep, g.N, m, n, v, bias, res[q]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// sums of the slices, then the epilogue.  A workgroup takes 64 x 16 bytes of outputs, four waves a quarter of the slices each; the quarters are
// added in their order (run-to-run identical)
template <int DT> __global__ __launch_bounds__(256) void k_lin_join(const float *part, int slices, int M, int N, LinEpi ep)
{
    constexpr int W = LinT<DT>::V;
    __shared__ float red[3][W][64];
    const unsigned units = ((unsigned)N + W - 1) / W;
    const size_t id = (size_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const size_t m = id / units;
    const int n = (int)(id % units) * W, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const bool live = m < (size_t)M;
    float v[W];
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = 0.f;
    if (live) {
        const int s1 = slices * (wave + 1) / 4;
#pragma unroll 4
        for (int s = slices * wave / 4; s < s1; ++s) {
            float t[W];
            lin_load<float, W>(t, part + ((size_t)s * M + m) * N + n, N - n);
#pragma unroll
            for (int e = 0; e < W; ++e) v[e] += t[e];
        }
        if (wave)
#pragma unroll
            for (int e = 0; e < W; ++e) red[wave - 1][e][lane] = v[e];
    }
    __syncthreads();
    if (wave || !live) return;
    float b[W], r[W];
    lin_bias<DT>(b, ep, N, n);
    if (ep.res) lin_residual<DT>(r, ep, N, (int)m, n);
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = ((v[e] + red[0][e][lane]) + red[1][e][lane]) + red[2][e][lane];
    lin_epilogue<DT>(ep, N, (int)m, n, v, b, r);
}

// Few rows (a token, a handful of regions): bound by reading the weight once.  A workgroup takes 16 columns and all rows, its waves a share of the
// sum each (slices of 64 bytes per weight row, four at a time: 256 bytes in a row), straight from memory into the matrix instruction, four
// slices ahead; the waves' sums meet in the LDS in their order -- one launch, no partial sums in memory (1 x 4096 x 4096 bf16: 8.1 us = 4.1 TB/s, the
// tile kernel with 8 slices and their join 11.1).  MB x 16 rows
template <int DT, int MB, int NW> __global__ __launch_bounds__(64 * NW) void k_lin_few(const LinArgs g)
{
    constexpr int V = LinT<DT>::V, SL = 4 * V, UN = 4;          // summed indexes of a slice, slices at a time
    __shared__ f32x4 red[NW][MB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n0 = (int)blockIdx.x * 16, r = lane & 15, kl = (lane >> 4) * V;
    const int rounds = (g.K + SL * UN - 1) / (SL * UN);
    f32x4 acc[MB];
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint4 w[UN], x[UN][MB];
    auto ask = [&](int round) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int k = (round * UN + u) * SL + kl;
            w[u] = lin_fetch<DT, false>(g.a, g.N, g.K, n0 + r, k);
#pragma unroll
            for (int j = 0; j < MB; ++j) x[u][j] = lin_fetch<DT, false>(g.b, g.M, g.K, 16 * j + r, k);
        }
    };
    if (wave < rounds) ask(wave);
    for (int round = wave; round < rounds; round += NW) {
        uint4 wc[UN], xc[UN][MB];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            wc[u] = w[u];
#pragma unroll
            for (int j = 0; j < MB; ++j) xc[u][j] = x[u][j];
        }
        if (round + NW < rounds) ask(round + NW);
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int j = 0; j < MB; ++j) lin_mma<DT>(acc[j], wc[u], xc[u][j]);
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) red[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave >= MB) return;
    f32x4 s = red[0][wave][lane];
    for (int q = 1; q < NW; ++q) s += red[q][wave][lane];
    const int m = 16 * wave + r, n = n0 + 4 * (lane >> 4);
    if (m >= g.M || n >= g.N) return;
    float v[4] = {s[0], s[1], s[2], s[3]}, bias[4], res[4];
    lin_bias<DT, 4>(bias, g.ep, g.N, n);
    if (g.ep.res) lin_residual<DT, 4>(res, g.ep, g.N, m, n);
    lin_epilogue<DT, 4>(g.ep, g.N, m, n, v, bias, res);
}

// dz = dy * act'(z) (CURVED, 16 bits: its two parts) and the column sums of dz over a run of rows.  tpr threads (a power of two) take W columns each of a row.  Bound: memory, two
// reads and a write (fp16 131072 x 512 with gelu, 671 MB with z in fp32 and two parts of dz: 150 us = 4.5 TB/s)
struct DactArgs {
    const void *gy, *z;         // z NULL: no activation, dz = gy
    void *dz, *lo;              // NULL: not stored; lo: the lower part (CURVED in 16 bits)
    float *part;                // [gridDim.y][N] (one run of rows: not used, the sums go to db)
    void *db;                   // NULL: no sums asked for
    long long ldg, ldz;         // ldz: elements between the rows of dz
    int M, N, span, act, tpr_log, db_f32;
};

template <int DT, bool CURVED> __global__ __launch_bounds__(256) void k_lin_dact(const DactArgs a)
{
    typedef typename LinT<DT>::S S;
    typedef std::conditional_t<CURVED, float, S> Z;
    constexpr int W = LinT<DT>::V;
    __shared__ float red[256 * W];
    const int tpr = 1 << a.tpr_log, tid = threadIdx.x, c = tid & (tpr - 1), r = tid >> a.tpr_log, rows = 256 >> a.tpr_log;
    const int n = ((int)blockIdx.x * tpr + c) * W, cnt = a.N - n;
    const int m1 = a.M - (int)blockIdx.y * a.span < a.span ? a.M : ((int)blockIdx.y + 1) * a.span;
    float sum[W];
#pragma unroll
    for (int e = 0; e < W; ++e) sum[e] = 0.f;
    if (n < a.N)
#pragma unroll 4
        for (int m = (int)blockIdx.y * a.span + r; m < m1; m += rows) {
            float d[W], z[W];
            lin_load<S, W>(d, (const S *)a.gy + (size_t)m * a.ldg + n, cnt);
            if (a.z) {
                lin_load<Z, W>(z, (const Z *)a.z + (size_t)m * a.N + n, cnt);
                lin_dacts<DT, W>(d, z, a.act);
            }
#pragma unroll
            for (int e = 0; e < W; ++e) sum[e] += d[e];
            if (!a.dz) continue;
            const size_t at = (size_t)m * a.ldz + n;
            if constexpr (CURVED && DT != DT_F32) {
                float lo[W];
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    d[e] *= LinParts<DT>::PRE;
                    const float hi = (float)(S)d[e];
                    lo[e] = __builtin_isfinite(hi) ? (d[e] - hi) * LinParts<DT>::LO : 0.f;
                }
                lin_save<S, W>((S *)a.lo + at, lo, cnt);
            }
            lin_save<S, W>((S *)a.dz + at, d, cnt);
        }
    if (!a.db) return;
#pragma unroll
    for (int e = 0; e < W; ++e) red[e * 256 + tid] = sum[e];
    __syncthreads();
    if (r == 0 && n < a.N)
#pragma unroll
        for (int e = 0; e < W; ++e) {
            float s = 0.f;
            for (int q = 0; q < rows; ++q) s += red[e * 256 + (q << a.tpr_log) + c];
            if (e >= cnt) continue;
            if (gridDim.y > 1) a.part[(size_t)blockIdx.y * a.N + n + e] = s;
            else if (a.db_f32) ((float *)a.db)[n + e] = s;
            else ((S *)a.db)[n + e] = (S)s;
        }
}

// rows of any start and width -> rows that start on 16 bytes (ldo elements apart, a multiple of a vector; the columns behind the row's end are
// zeros): two elements per thread, whole 4-byte words written
template <int DT> __global__ __launch_bounds__(256) void k_lin_pack(void *out, const void *in, long long ld, int rows, int len, int ldo)
{
    typedef typename LinT<DT>::S S;
    typedef S S2 __attribute__((ext_vector_type(2)));
    const unsigned pairs = (unsigned)ldo / 2;
    for (size_t id = (size_t)blockIdx.x * 256 + threadIdx.x; id < (size_t)rows * pairs; id += (size_t)gridDim.x * 256) {
        const unsigned row = (unsigned)(id / pairs), c = (unsigned)(id - (size_t)row * pairs) * 2;
        const S *p = (const S *)in + (size_t)row * ld + c;
        S2 v;
        v[0] = c < (unsigned)len ? p[0] : (S)0.f;
        v[1] = c + 1 < (unsigned)len ? p[1] : (S)0.f;
        *(S2 *)((S *)out + (size_t)row * ldo + c) = v;
    }
}

// 16 columns x 16 runs of partial sums per workgroup, joined in order
template <int DT> __global__ __launch_bounds__(256) void k_lin_colsum(void *db, int db_f32, const float *part, int P, int N)
{
    typedef typename LinT<DT>::S S;
    __shared__ float red[256];
    const int n = (int)blockIdx.x * 16 + (threadIdx.x & 15), run = threadIdx.x >> 4;
    float s = 0.f;
    if (n < N)
#pragma unroll 8
        for (int p = run; p < P; p += 16) s += part[(size_t)p * N + n];
    red[threadIdx.x] = s;
    __syncthreads();
    if (run || n >= N) return;
    s = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += red[16 * r + threadIdx.x];
    if (db_f32) ((float *)db)[n] = s;
    else ((S *)db)[n] = (S)s;
}

// ------------------------------------------------------------------------------------------------------------------ host side
constexpr int LIN_CUS = 256;

struct LinPlan { int slices, kspan, edge; unsigned tm, tn; };

inline int lin_bk(int dtype) { return dtype == DT_F32 ? 32 : 64; }
inline long long lin_round(long long v, long long to) { return (v + to - 1) / to * to; }
inline long long lin_min(long long a, long long b) { return a < b ? a : b; }
inline long long lin_tiles(long long M, long long N, int edge) { return ((M + edge - 1) / edge) * ((N + edge - 1) / edge); }

LinPlan lin_plan(int dtype, long long M, long long N, long long K)
{
    LinPlan p;
    const int bk = lin_bk(dtype);
    const long long steps = (K + bk - 1) / bk, t64 = lin_tiles(M, N, 64), t128 = lin_tiles(M, N, 128), t256 = lin_tiles(M, N, 256);
    long long s;
    if (dtype == DT_F32) {
        // 64 (the matrix instructions take so long that a small tile's operands arrive in time: 17408 x 768 x 256 and 1024^3 in 0.7 of the time that
        // 128 takes).  Slices until every CU has a tile, of 2 steps at least (128 x 512 x 512 8 slices 8.2 us, one 12.9), or two or three, of 24
        // steps at least (256 x 768 x 17408 16 slices 62 us, 8: 80; but 512 x 1024 x 1024 2 slices 17 us, 4: 19; 256 x 4096 x 1024 4: 28, 5: 35)
        p.edge = 64;
        s = lin_min(LIN_CUS / t64, steps / 2);
        for (int per_cu = 2; per_cu <= 3; ++per_cu)
            if (per_cu * LIN_CUS / t64 <= steps / 24) s = per_cu * LIN_CUS / t64;
    } else {
        // 256 once that fills the chip's rounds and the sum is long enough to pay for an epilogue that nothing overlaps
        // (16384 x 4096 x 8192: 845 us, 128: 970, 64: 1512; 8192 x 2048 x 8192: 225, 250, 345; 8192 x 768 x 4096: 54, 61, 76 -- but 17408 x 512 x 2048: 73,
        // 53, 66; rounds filled: 7 tenths pay from 1024 summed indexes on, 9 below: 16384 x 640 x 2560 in 2.5 rounds 92 us, 128: 81; 32768 x 768 x 768
        // in 1.5 67, 57), else 128 while that, with a long sum in slices of at least 16 steps, gives every CU one (2048 x 512 x 17408 in 8 slices 47 us,
        // 64: 66; 256 x 4096 x 4096 in 4: 23.2, 8: 25.3; but 512 x 4096 x 1024 in 8 of 8 steps 21 us, 64: 15.7), else 64 (1024^3 11 us against 17),
        // in slices of at least 8 steps of a sum of more than 16 (64 x 4096 x 4096 8 slices 12.9 us, 16: 16; 100 x 1024 x 4096 one 6.7, 4: 10.3), 64
        // slices at most (256 x 64 x 65536 64: 18.8, 128: 22.5)
        const long long rounds = (t256 + LIN_CUS - 1) / LIN_CUS, s128 = t128 >= LIN_CUS ? 1 : lin_min(2 * LIN_CUS / t128, steps / 16);
        const bool full = t256 >= LIN_CUS && 10 * t256 >= (K < 1024 ? 9 : 7) * rounds * LIN_CUS;
        p.edge = K > 512 && full ? 256 : t128 * (s128 > 1 ? s128 : 1) >= LIN_CUS ? 128 : 64;
        s = p.edge == 256 ? 1 : p.edge == 128 ? s128 : t64 >= LIN_CUS || steps <= 16 ? 1 : lin_min(lin_min(2 * LIN_CUS / t64, 64), steps / 8);
    }
    p.tm = (unsigned)((M + p.edge - 1) / p.edge);
    p.tn = (unsigned)((N + p.edge - 1) / p.edge);
    if (s < 1) s = 1;
    const long long per = (steps + s - 1) / s;
    p.kspan = (int)(per * bk);
    p.slices = (int)((steps + per - 1) / per);
    if (p.slices < 1) p.slices = 1;
    return p;
}

inline long long lin_part_bytes(const LinPlan &p, long long M, long long N) { return p.slices > 1 ? lin_round(4ll * p.slices * M * N, 256) : 0; }
inline int lin_esize(int dtype) { return dtype == DT_F32 ? 4 : 2; }

// may an operand travel global -> LDS directly: aligned 16-byte vectors that never straddle a row's end, offsets inside a tile below 2^31
inline bool lin_direct(const LinOperand &o, bool mc, int dtype)
{
    const int e = lin_esize(dtype), v = 16 / e;
    return (uintptr_t)o.p % 16 == 0 && o.ld % v == 0 && (!mc || o.run % v == 0) && o.ld * e * 256 < 0x7fffffffll;
}

template <int DT, int BM, int BN, int WM, int WN, bool AMC, bool BMC, bool DIRECT, int C, bool TWO> int lin_run(LinArgs &g, const LinPlan &p, hipStream_t st)
{
    const size_t lds = (size_t)2 * (BM + BN) * C * sizeof(uint4);
    if (lds > 64 * 1024) {      // (asked for once per device)
        static std::atomic<unsigned long long> asked{0};
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        if (e == hipSuccess && !(asked.load() >> (dev & 63) & 1)) {
            e = hipFuncSetAttribute((const void *)k_lin_gemm<DT, BM, BN, WM, WN, AMC, BMC, DIRECT, C, TWO>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e == hipSuccess) asked.fetch_or(1ull << (dev & 63));
        }
        if (e != hipSuccess) return (int)e;
    }
    k_lin_gemm<DT, BM, BN, WM, WN, AMC, BMC, DIRECT, C, TWO><<<p.tm * p.tn * (unsigned)p.slices, 64 * WM * WN, lds, st>>>(g);
    return lin_status();
}

template <int DT, bool AMC, bool BMC, bool TWO> int lin_pick(LinArgs &g, LinPlan p, void *ws, hipStream_t st)
{
    g.part = p.slices > 1 ? (float *)ws : nullptr;
    const bool direct = lin_direct(g.a, AMC, DT) && lin_direct(g.b, BMC, DT);
    if (!direct && p.edge == 256) {     // (the register route has no large tile)
        p.edge = 128;
        p.tm = (unsigned)(((long long)g.M + 127) / 128);
        p.tn = (unsigned)(((long long)g.N + 127) / 128);
    }
    g.kspan = p.kspan;
    g.tiles_m = p.tm;
    g.tiles_n = p.tn;
    int r = BC_OK;
    if (p.edge == 64) r = direct ? lin_run<DT, 64, 64, 2, 2, AMC, BMC, true, 8, TWO>(g, p, st) : lin_run<DT, 64, 64, 2, 2, AMC, BMC, false, 8, TWO>(g, p, st);
    else if constexpr (DT != DT_F32) {
        // (a short sum: steps of 64 bytes halve the images, four workgroups share a CU and one's epilogue runs beside the others' products:
        //  131072 x 256 x 512 52 us against 63; a long one: 128 bytes, half the barriers: 8192 x 768 x 4096 61 us against 65)
        if (!direct) r = lin_run<DT, 128, 128, 2, 2, AMC, BMC, false, 8, TWO>(g, p, st);
        else if (p.edge == 256) r = lin_run<DT, 256, 256, 2, 4, AMC, BMC, true, 8, TWO>(g, p, st);
        else if (g.K <= 512) r = lin_run<DT, 128, 128, 2, 2, AMC, BMC, true, 4, TWO>(g, p, st);
        // (one workgroup per CU, or up to two with a whole sum each and operands along it: eight waves hide each other's waits, 4096 x 1024 x 1024
        //  13.5 us against 16.3, 2048^3 24.7 against 27.4, 3000 x 768 x 2304 16.6 against 18.1; else four waves, whose larger tiles read less from
        //  the LDS, 2048 x 512 x 17408 45 against 51, the data gradient of 2048 x 4096 x 4096 60 against 66)
        else if (p.tm * p.tn * (unsigned)p.slices <= LIN_CUS || (!AMC && !BMC && p.slices == 1 && p.tm * p.tn <= 2 * LIN_CUS)) r = lin_run<DT, 128, 128, 2, 4, AMC, BMC, true, 8, TWO>(g, p, st);
        else r = lin_run<DT, 128, 128, 2, 2, AMC, BMC, true, 8, TWO>(g, p, st);
    }
    if (r != BC_OK || p.slices == 1) return r;
    const long long units = (long long)g.M * ((g.N + LinT<DT>::V - 1) / LinT<DT>::V);
    k_lin_join<DT><<<(unsigned)((units + 63) / 64), 256, 0, st>>>(g.part, p.slices, g.M, g.N, g.ep);
    return lin_status();
}

template <bool AMC, bool BMC> int lin_product(int dtype, LinArgs &g, const LinPlan &p, void *ws, hipStream_t st)
{
    switch (dtype) {
    case DT_F32: return lin_pick<DT_F32, AMC, BMC, false>(g, p, ws, st);
    case DT_F16:
        if constexpr (AMC)      // (dz is the row operand of both gradients, whose other operand runs across the summed index)
            if (g.b_lo) return lin_pick<DT_F16, AMC, BMC, true>(g, p, ws, st);
        return lin_pick<DT_F16, AMC, BMC, false>(g, p, ws, st);
    default:
        if constexpr (AMC)
            if (g.b_lo) return lin_pick<DT_BF16, AMC, BMC, true>(g, p, ws, st);
        return lin_pick<DT_BF16, AMC, BMC, false>(g, p, ws, st);
    }
}

template <int DT> int lin_few(const LinArgs &g, hipStream_t st)
{
    const unsigned wgs = ((unsigned)g.N + 15) / 16;
    if (g.M <= 16) {        // 16 waves where there are too few columns to fill the chip with 8
        if (wgs < LIN_CUS) k_lin_few<DT, 1, 16><<<wgs, 1024, 0, st>>>(g);
        else k_lin_few<DT, 1, 8><<<wgs, 512, 0, st>>>(g);
    } else
        k_lin_few<DT, 2, 8><<<wgs, 512, 0, st>>>(g);
    return lin_status();
}

inline bool lin_aligned(const void *p, int dtype) { return (uintptr_t)p % lin_esize(dtype) == 0; }
inline bool lin_z_aligned(const void *z, int act, int dtype) { return (uintptr_t)z % (lin_curved(act) ? 4 : lin_esize(dtype)) == 0; }
inline bool lin_two_parts(int act, int dtype) { return dtype != DT_F32 && lin_curved(act); }

int lin_sizes(long long M, int N, int K, int dtype)
{
    if (dtype < 0 || dtype > 2) return BC_ERR_ELEM;
    if (M < 0 || N < 1 || K < 1) return BC_ERR_SHAPE;
    if (M > 0x7fffff00ll || N > 0x7fffff00 || K > 0x7fffff00) return BC_ERR_RANGE;
    const long long m = (M + 63) / 64, n = ((long long)N + 63) / 64, k = ((long long)K + 63) / 64, most = 0xffffff;      // (tiles x 256 threads of a launch)
    if (m > most / n || m > most / k || n > most / k) return BC_ERR_RANGE;
    return BC_OK;
}

// Is it worth bringing operands whose rows do not start on 16 bytes into order first?  The register route takes about twice the direct one's time
// (16 bits: 4.3 GFLOP 22 us against 11, 69 GFLOP 104 against 58, its weight gradient 272 against 110; fp32: 4.2 GFLOP 65 against 42), the copy two
// passes over the operands and a launch: worth it from about 2 GFLOP on, unless one side is so short that the copy outweighs the products
inline bool lin_worth(long long M, long long N, long long K) { return (double)M * (double)N * (double)K >= 1e9 && M * N >= 200 * (M + N); }
inline int lin_padded(long long len, int dtype) { return (int)lin_round(len, 16 / lin_esize(dtype)); }
inline long long lin_pack_bytes(long long rows, long long len, int dtype) { return lin_round(rows * lin_padded(len, dtype) * lin_esize(dtype), 256); }

// the operand in order, in the workspace at *ws (moved on)
LinOperand lin_pack(const LinOperand &o, long long rows, char **ws, int dtype, hipStream_t st)
{
    const LinOperand r = {*ws, lin_padded(o.run, dtype), lin_padded(o.run, dtype)};
    const long long words = rows * r.ld / 2;
    const unsigned grid = (unsigned)((words + 1023) / 1024 < 4096 ? (words + 1023) / 1024 : 4096);
    switch (dtype) {
    case DT_F32: k_lin_pack<DT_F32><<<grid, 256, 0, st>>>(*ws, o.p, o.ld, (int)rows, o.run, (int)r.ld); break;
    case DT_F16: k_lin_pack<DT_F16><<<grid, 256, 0, st>>>(*ws, o.p, o.ld, (int)rows, o.run, (int)r.ld); break;
    default: k_lin_pack<DT_BF16><<<grid, 256, 0, st>>>(*ws, o.p, o.ld, (int)rows, o.run, (int)r.ld);
    }
    *ws += lin_pack_bytes(rows, o.run, dtype);
    return r;
}

struct DactPlan { int tpr_log, span; unsigned gx, gy; };

DactPlan lin_dact_plan(long long M, int N, int dtype)
{
    DactPlan p;
    const int W = 16 / lin_esize(dtype), units = (int)(((long long)N + W - 1) / W);
    p.tpr_log = 0;
    while (p.tpr_log < 8 && (1 << p.tpr_log) < units) ++p.tpr_log;
    const int rows = 256 >> p.tpr_log;
    p.gx = (unsigned)((units + (1 << p.tpr_log) - 1) >> p.tpr_log);
    long long chunks = 4 * LIN_CUS / p.gx > 0 ? 4 * LIN_CUS / p.gx : 1;
    const long long most = (M + 4 * rows - 1) / (4 * rows);
    if (chunks > most) chunks = most;
    if (chunks < 1) chunks = 1;
    p.span = (int)((M + chunks - 1) / chunks);
    if (p.span < 1) p.span = 1;
    p.gy = (unsigned)((M + p.span - 1) / p.span);
    return p;
}

template <int DT> int lin_dact_run(const DactArgs &a0, const DactPlan &p, hipStream_t st)
{
    DactArgs a = a0;
    a.span = p.span;
    a.tpr_log = p.tpr_log;
    if (a.z && lin_curved(a.act)) k_lin_dact<DT, true><<<dim3(p.gx, p.gy), 256, 0, st>>>(a);
    else k_lin_dact<DT, false><<<dim3(p.gx, p.gy), 256, 0, st>>>(a);
    if (a.db && p.gy > 1) k_lin_colsum<DT><<<(a.N + 15) / 16, 256, 0, st>>>(a.db, a.db_f32, a.part, (int)p.gy, a.N);
    return lin_status();
}

}  // namespace

// does the forward product take k_lin_few: few rows, and enough columns to fill part of the chip or a short sum (8 x 8192 x 128 13 us there, 7 as
// tiles); 16-bit rows must start on 4 bytes (13 x 2047 x 1001: 13 us against 8, 13 x 2046 x 1001: 5.8).  Beyond 16 rows only short sums
// (32 x 1024 x 1024 4.8 us against 6.0, 32 x 4096 x 4096 14 against 11)
static bool lin_takes_few(const void *x, const void *w, long long M, int N, int K, long long ldx, long long ldw, int dtype)
{
    if (M > 32 || (M > 16 && K > 1024) || (N < 1024 && K > 2048) || N > 16 * 0x3fffff) return false;       // (the launch: below 2^32 threads)
    return dtype == DT_F32 || ((uintptr_t)x % 4 == 0 && (uintptr_t)w % 4 == 0 && ldx % 2 == 0 && ldw % 2 == 0);
}

BC_EXPORT long long bc_linear_fwd_workspace(long long M, int N, int K, int dtype)
{
    if (lin_sizes(M, N, K, dtype) != BC_OK || M == 0) return 0;
    const long long pack = K % (16 / lin_esize(dtype)) && lin_worth(M, N, K) ? lin_pack_bytes(M, K, dtype) + lin_pack_bytes(N, K, dtype) : 0;
    return lin_part_bytes(lin_plan(dtype, M, N, K), M, N) + pack;
}

BC_EXPORT int bc_linear_fwd(void *y, void *z, const void *x, const void *w, const void *bias, const void *residual, long long M, int N, int K, long long ldx,
                            long long ldw, long long ldr, int act, int dtype, int bias_f32, void *workspace, long long workspace_bytes, void *stream)
{
    const int rc = lin_sizes(M, N, K, dtype);
    if (rc != BC_OK) return rc;
    if (act < 0 || act >= ACT_COUNT || ldx < K || ldw < K || (residual && ldr < N)) return BC_ERR_SHAPE;
    if (M == 0) return BC_OK;
    if (!y || !x || !w) return BC_ERR_NULL;
    if (!lin_aligned(x, dtype) || !lin_aligned(w, dtype) || !lin_aligned(y, dtype) || !lin_z_aligned(z, act, dtype) || !lin_aligned(residual, dtype)) return BC_ERR_ALIGN;
    if (bias && (uintptr_t)bias % (bias_f32 ? 4 : lin_esize(dtype))) return BC_ERR_ALIGN;
    const long long need = bc_linear_fwd_workspace(M, N, K, dtype);
    if (need > 0 && !workspace) return BC_ERR_NULL;
    if (workspace_bytes < need) return BC_ERR_SHAPE;
    if (need > 0 && (uintptr_t)workspace % 256 != 0) return BC_ERR_ALIGN;
    hipStream_t st = (hipStream_t)stream;
    const LinPlan p = lin_plan(dtype, M, N, K);
    LinArgs g = {};
    g.a = {w, ldw, K};
    g.b = {x, ldx, K};
    g.M = (int)M;
    g.N = N;
    g.K = K;
    g.ep = {y, z, bias, residual, ldr, bias_f32, act};
    if (lin_takes_few(x, w, M, N, K, ldx, ldw, dtype))
        return dtype == DT_F32 ? lin_few<DT_F32>(g, st) : dtype == DT_F16 ? lin_few<DT_F16>(g, st) : lin_few<DT_BF16>(g, st);
    char *free_ws = (char *)workspace + lin_part_bytes(p, M, N);
    if (K % (16 / lin_esize(dtype)) && lin_worth(M, N, K)) {
        if (!lin_direct(g.a, false, dtype)) g.a = lin_pack(g.a, N, &free_ws, dtype, st);
        if (!lin_direct(g.b, false, dtype)) g.b = lin_pack(g.b, M, &free_ws, dtype, st);
    }
    return lin_product<false, false>(dtype, g, p, workspace, st);
}

// the workspace of a backward pass: dz (with an activation, or where gy is brought into order), the column sums' partials, the slices of one
// product at a time, and x and w in order.  What is brought into order goes by the sizes alone, here and in the call
struct LinBwdSpace { long long dz, part, slices, pack; bool order_n, order_k; };
static LinBwdSpace lin_bwd_space(long long M, int N, int K, int act, int dtype)
{
    LinBwdSpace s;
    const int v = 16 / lin_esize(dtype);
    const bool worth = lin_worth(M, N, K);
    s.order_n = N % v && worth;
    s.order_k = K % v && worth;
    s.dz = act != ACT_NONE || s.order_n ? lin_pack_bytes(M, N, dtype) * (lin_two_parts(act, dtype) ? 2 : 1) : 0;
    s.part = lin_round(4ll * N * lin_dact_plan(M, N, dtype).gy, 256);
    const long long x = lin_part_bytes(lin_plan(dtype, M, K, N), M, K), w = lin_part_bytes(lin_plan(dtype, N, K, M), N, K);
    s.slices = x > w ? x : w;
    s.pack = s.order_k ? lin_pack_bytes(M, K, dtype) + lin_pack_bytes(N, K, dtype) : 0;
    return s;
}

BC_EXPORT long long bc_linear_bwd_workspace(long long M, int N, int K, int act, int dtype)
{
    if (lin_sizes(M, N, K, dtype) != BC_OK || M == 0 || act < 0 || act >= ACT_COUNT) return 0;
    const LinBwdSpace s = lin_bwd_space(M, N, K, act, dtype);
    return s.dz + s.part + s.slices + s.pack;
}

BC_EXPORT int bc_linear_bwd(void *dx, void *dw, void *db, const void *gy, const void *z, const void *x, const void *w, long long M, int N, int K, long long ldg,
                            long long ldx, long long ldw, int act, int dtype, int bias_f32, void *workspace, long long workspace_bytes, void *stream)
{
    const int rc = lin_sizes(M, N, K, dtype);
    if (rc != BC_OK) return rc;
    if (act < 0 || act >= ACT_COUNT || ldg < N || (dw && ldx < K) || (dx && ldw < K)) return BC_ERR_SHAPE;
    if (M == 0) return BC_ERR_SHAPE;        // (no rows: the caller's gradients are zeros, nothing to launch)
    if (!gy || (act != ACT_NONE && !z) || (dx && !w) || (dw && !x)) return BC_ERR_NULL;
    if (!lin_aligned(gy, dtype) || !lin_z_aligned(z, act, dtype) || !lin_aligned(x, dtype) || !lin_aligned(w, dtype) || !lin_aligned(dx, dtype) || !lin_aligned(dw, dtype))
        return BC_ERR_ALIGN;
    if (db && (uintptr_t)db % (bias_f32 ? 4 : lin_esize(dtype))) return BC_ERR_ALIGN;
    const LinBwdSpace s = lin_bwd_space(M, N, K, act, dtype);
    if (!workspace) return BC_ERR_NULL;
    if (workspace_bytes < s.dz + s.part + s.slices + s.pack) return BC_ERR_SHAPE;
    if ((uintptr_t)workspace % 256 != 0) return BC_ERR_ALIGN;
    hipStream_t st = (hipStream_t)stream;
    char *wsp = (char *)workspace, *pack = wsp + s.dz + s.part + s.slices;
    void *slices = wsp + s.dz + s.part;
    LinOperand dz = {gy, ldg, N};
    const size_t lo = lin_two_parts(act, dtype) ? (size_t)lin_pack_bytes(M, N, dtype) : 0;
    const bool store = (dx || dw) && (act != ACT_NONE || s.order_n);
    if (store || db) {
        const DactPlan p = lin_dact_plan(M, N, dtype);
        DactArgs a = {};
        a.gy = gy;
        a.z = act != ACT_NONE ? z : nullptr;
        a.dz = store ? wsp : nullptr;
        a.lo = store && lo ? wsp + lo : nullptr;
        a.part = (float *)(wsp + s.dz);
        a.db = db;
        a.db_f32 = bias_f32;
        a.ldg = ldg;
        a.ldz = lin_padded(N, dtype);       // (what lies behind a row's end is never part of a stored sum)
        a.M = (int)M;
        a.N = N;
        a.act = act;
        const int r = dtype == DT_F32 ? lin_dact_run<DT_F32>(a, p, st) : dtype == DT_F16 ? lin_dact_run<DT_F16>(a, p, st) : lin_dact_run<DT_BF16>(a, p, st);
        if (r != BC_OK) return r;
        if (store) dz = {wsp, a.ldz, (int)a.ldz};
    }
    if (dx) {       // dx[m][k] = sum_n dz[m][n] w[n][k]: the weight runs across the summed index
        LinArgs g = {};
        g.a = {w, ldw, K};
        if (s.order_k) g.a = lin_pack(g.a, N, &pack, dtype, st);
        g.b = {dz.p, dz.ld, N};
        g.b_lo = lo;
        g.M = (int)M;
        g.N = K;
        g.K = N;
        g.ep = {dx, nullptr, nullptr, nullptr, 0, 0, ACT_NONE};
        const int r = lin_product<true, false>(dtype, g, lin_plan(dtype, M, K, N), slices, st);
        if (r != BC_OK) return r;
    }
    if (dw) {       // dw[n][k] = sum_m dz[m][n] x[m][k]: both run across it
        LinArgs g = {};
        g.a = {x, ldx, K};
        if (s.order_k) g.a = lin_pack(g.a, M, &pack, dtype, st);
        g.b = dz;
        g.b_lo = lo;
        g.M = N;
        g.N = K;
        g.K = (int)M;
        g.ep = {dw, nullptr, nullptr, nullptr, 0, 0, ACT_NONE};
        const int r = lin_product<true, true>(dtype, g, lin_plan(dtype, N, K, M), slices, st);
        if (r != BC_OK) return r;
    }
    return BC_OK;
}
