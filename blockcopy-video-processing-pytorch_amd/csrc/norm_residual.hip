// norm_residual.hip -- what stands between two blocks of a residual network, in one pass over the rows, and its gradient.  Part of
// libblockcopy_hip.so.
//
//   t  = N_out(y) * wo + bo                 the norm after a block (or y itself)
//   h' = residual_scale * h + gate * t      the block's gate (per channel, or per sample and channel) and the residual stream
//   u  = N_in(h') * wi + bi                 the norm before the next block (or nothing)
//   N(x) = x / sqrt(mean(x^2) + eps)  (rms)   or   (x - mean(x)) / sqrt(mean((x - mean(x))^2) + eps)  (layer), over the C channels of a row
//
// A row is one pixel of a channels-last map (or one token).  All statistics and sums are fp32 and centred (a second pass over registers);
// u is formed from the unrounded h'.  Bound: memory -- forward reads h, y and writes h', u; backward reads h, y and the two gradients and
// writes dh, dy.  It forms h' again out of h and y (the same bytes as reading it back, without its rounding).
// Decomposition: a lane owns E channels of a row (16-byte vectors) and a row G lanes -- part of a wave, or up to 16 waves that exchange
// their sums through the LDS.  Backward: a lane keeps the same channels for every row of its workgroup, so what the column sums (gate, norm
// weights and biases) need stays in registers, and goes to a workspace once per workgroup; a second launch adds them in a fixed order.
// Measured (a large copy reaches 5.2 TB/s), layer norm after and rms norm before the block, with gate and parameters, 128 MB per tensor:
//   bf16   131072 x 512 forward 108 us (5.0 TB/s), backward 180 (4.5)    32768 x 2048 106 (5.1), 193 (4.2)    16384 x 4096 109 (4.9), 203 (4.0)
//          8192 x 8192 126 (4.3), 218 (3.7)    4096 x 16384 142 (3.8), 448 (1.8: the column sums' second pass)
//   fp32   65536 x 512 102 (5.3), 175 (4.6)    8192 x 4096 104 (5.2), 178 (4.5)    4096 x 8192 117 (4.6), 198 (4.1)
//   rows that start anywhere, bf16: 65154 x 1030 168 (3.2), 300 (2.7)    16368 x 4100 158 (3.4), 471 (1.7)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/blockcopy_hip.h"

#define BC_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

enum { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };
enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };

template <int DT> struct NrT { typedef float S; static constexpr int V = 4; };
template <> struct NrT<DT_F16> { typedef _Float16 S; static constexpr int V = 8; };
template <> struct NrT<DT_BF16> { typedef __bf16 S; static constexpr int V = 8; };

inline int nr_status()
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BC_OK : (int)e;
}

struct NormArgs {
    const void *h, *y;                          // (M, C), rows ldh / ldy apart; y NULL: no block, h' = h (not stored)
    const void *wo, *bo, *gate, *wi, *bi;       // NULL: ones / zeros; fp32 or the tensors' type (pf32)
    void *ho, *u;
    float *stats;                               // [M][4]: mean, 1 / deviation of y; mean, 1 / deviation of h' (backward)
    const void *gh, *gu;                        // gradients of h' and u (NULL: zeros)
    void *dh, *dy;
    float *part;                                // [workgroups][5][C]: column sums of gate, wo, bo, wi, bi
    float *means;                               // [M][2]: mean(p n), mean(p) of the inner norm's backward (column sums in a second pass)
    long long ldh, ldy, ldgh, ldgu;
    int M, C, g_log, rows_per_gate, span, chunks;
    int out_kind, in_kind, pf32, need_dh, need_dy;
    float alpha, eps;
    void *d_gate;                               // the gate's gradient where k_norm_cols writes it itself
    int gate_every;                             // backward: rows per gate where a workgroup's rows have several (rows_per_gate is 0 then)
};

// ---- sums over the G lanes of a row; every lane of the row gets the same bits
template <int CTRL> __device__ __forceinline__ float nr_dpp(float v)
{
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

typedef unsigned nr_pair __attribute__((ext_vector_type(2)));

// v + the v of the lane 16 / 32 away, without the LDS
__device__ __forceinline__ float nr_swap16(float v)
{
    const nr_pair p = __builtin_bit_cast(nr_pair, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

__device__ __forceinline__ float nr_swap32(float v)
{
    const nr_pair p = __builtin_bit_cast(nr_pair, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

__device__ __forceinline__ float nr_wave_sum(float v, int g_log)
{
    if (g_log > 0) v = nr_dpp<0xB1>(v);         // quad_perm 1 0 3 2
    if (g_log > 1) v = nr_dpp<0x4E>(v);         // quad_perm 2 3 0 1
    if (g_log > 2) v = nr_dpp<0x141>(v);        // row_half_mirror
    if (g_log > 3) v = nr_dpp<0x140>(v);        // row_mirror
    if (g_log > 4) v = nr_swap16(v);
    if (g_log > 5) v = nr_swap32(v);
    return v;
}

// WPR waves share a row: the waves' sums meet in `red` (two halves used in turn, so one barrier per exchange is enough; entries of waves that
// were not launched stay zeros).  Lane l reads wave l % WPR's and the lanes add up by exchange
template <int WPR, int NW> struct NrSum {
    static constexpr int LOG = WPR == 16 ? 4 : WPR == 8 ? 3 : WPR == 4 ? 2 : WPR == 2 ? 1 : 0;
    float2 *red;            // [2][NW]
    int turn, wave, g_log;
    float n, inv_n;         // channels of wave lane % WPR, and their reciprocal (0: none)
    __device__ __forceinline__ float2 exchange(float a, float b)
    {
        float2 *r = red + turn * NW;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) r[wave] = float2{a, b};
        __syncthreads();
        return r[wave / WPR * WPR + (threadIdx.x & (WPR - 1))];
    }
    __device__ __forceinline__ void operator()(float &a, float &b, bool two)
    {
        a = nr_wave_sum(a, g_log);
        if (two) b = nr_wave_sum(b, g_log);
        if constexpr (WPR > 1) {
            const float2 t = exchange(a, b);
            a = nr_wave_sum(t.x, LOG);
            if (two) b = nr_wave_sum(t.y, LOG);
        }
    }
};

template <int WPR, int NW, int V, int NV> __device__ __forceinline__ NrSum<WPR, NW> nr_sum(float2 *red, int wave, int g_log, int G, int C)
{
    NrSum<WPR, NW> s = {red, 0, wave, g_log, 0.f, 0.f};
    if constexpr (WPR > 1) {
        if (threadIdx.x < 2 * NW) red[threadIdx.x] = float2{0.f, 0.f};
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) n += min(max(C - (i * G + 64 * (int)(threadIdx.x & (WPR - 1))) * V, 0), min(64, max(G - 64 * (int)(threadIdx.x & (WPR - 1)), 0)) * V);
        s.n = (float)n;
        s.inv_n = n ? 1.f / s.n : 0.f;
        __syncthreads();
    }
    return s;
}

// `cnt` of V elements (all of them or none unless ODD) at column `at` of row `base` (in elements).  With the base in scalar registers (whole
// waves share a row) a lane's address is one 32-bit offset.  Rows of any width and start: the 16-byte accesses ask for the alignment of an
// element only (the hardware takes unaligned vectors).
template <typename S, int V> struct NrVec { typedef S T __attribute__((ext_vector_type(V), aligned(sizeof(S)))); };

template <bool ODD, int V> __device__ __forceinline__ bool nr_has(int cnt, int e) { return ODD ? e < cnt : cnt > 0; }

template <typename S, int V, bool ODD> __device__ __forceinline__ typename NrVec<S, V>::T nr_raw(const void *q, size_t base, unsigned at, int cnt)
{
    typedef typename NrVec<S, V>::T SV;
    const S *p = (const S *)q + base + at;
    SV v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (S)0.f;
    if (cnt <= 0) return v;         // (lanes without channels: one branch, nothing else)
    if (!ODD || cnt >= V) return *(const SV *)p;
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < cnt) v[e] = p[e];
    return v;
}

template <typename S, int V, bool ODD> __device__ __forceinline__ void nr_load(float *f, const void *q, size_t base, unsigned at, int cnt)
{
    const typename NrVec<S, V>::T v = nr_raw<S, V, ODD>(q, base, at, cnt);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (float)v[e];
}

template <typename S, int V, bool ODD> __device__ __forceinline__ void nr_store(void *q, size_t base, unsigned at, int cnt, const float *f)
{
    typedef typename NrVec<S, V>::T SV;
    if (cnt <= 0) return;
    S *p = (S *)q + base + at;
    SV v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (S)f[e];
    if (!ODD || cnt >= V) *(SV *)p = v;
    else {              // the end of a row in pieces of 4, 2 and 1
        if constexpr (V == 8)
            if (cnt & 4) {
                *(typename NrVec<S, 4>::T *)p = __builtin_shufflevector(v, v, 0, 1, 2, 3);
                p += 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = v[e + 4];
            }
        if (cnt & 2) {
            *(typename NrVec<S, 2>::T *)p = __builtin_shufflevector(v, v, 0, 1);
            p += 2;
            v[0] = v[2];
        }
        if (cnt & 1) *p = v[0];
    }
}

// per-channel parameters; `none` where the pointer is NULL
template <typename S, int V, bool ODD> __device__ __forceinline__ void nr_param(float *f, const void *p, int pf32, size_t base, unsigned at, int cnt, float none)
{
    if (!p) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = none;
    } else if (pf32) {
        if constexpr (V == 8) {
            nr_load<float, 4, ODD>(f, p, base, at, cnt);
            nr_load<float, 4, ODD>(f + 4, p, base, at + 4, ODD ? cnt - 4 : cnt);
        } else
            nr_load<float, V, ODD>(f, p, base, at, cnt);
    } else
        nr_load<S, V, ODD>(f, p, base, at, cnt);
}

// one row of a tensor as a lane holds it before its turn: NV vectors as they come from memory (requested a row ahead, so that the latency of
// memory lies behind the row in hand).  ODD: the last vector of a row is read as the row's last V elements and moved down at its turn by
// those that belong to the vector before -- one load like all others; element by element its 16-bit pieces are put together as they arrive,
// in front of everything behind them
template <typename S, int V, int NV, bool ODD> struct NrRow {
    typename NrVec<S, V>::T v[NV];
    static __device__ __forceinline__ bool last(unsigned col, int cnt) { return ODD && cnt > 0 && cnt < V && (int)col + cnt >= V; }
    __device__ __forceinline__ void ask(const void *q, size_t base, const unsigned *col, const int *cnt, bool live)
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!q || !live)
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = (S)0.f;
            else {
                const bool l = last(col[i], cnt[i]);
                v[i] = nr_raw<S, V, ODD>(q, base, l ? col[i] + cnt[i] - V : col[i], l ? V : cnt[i]);
            }
        }
    }
    __device__ __forceinline__ void settle(const unsigned *col, const int *cnt)
    {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (last(col[i], cnt[i])) v[i] = __builtin_bit_cast(typename NrVec<S, V>::T, __builtin_bit_cast(unsigned __int128, v[i]) >> ((V - cnt[i]) * (128 / V)));
    }
    __device__ __forceinline__ float at(int k) const { return (float)v[k / V][k % V]; }
};

// a parameter's channels of this lane, in registers for all its rows
template <typename S, int V, int NV, bool ODD> __device__ __forceinline__ void nr_params(float *f, const void *p, int pf32, size_t base, const unsigned *col, const int *cnt, float none)
{
#pragma unroll
    for (int i = 0; i < NV; ++i) nr_param<S, V, ODD>(f + i * V, p, pf32, base, col[i], cnt[i], none);
}

// x[E] -> normalised in place (0 behind the row's end); mean and 1 / deviation returned.  E = NV vectors of V.  Variances are sums of squared
// distances from the mean.  Of the row where a wave or less holds it; where waves share it, each takes the distances from its own mean, and
// sum (x - mean)^2 = sum over waves of [sum (x - mean_w)^2 + n_w (mean_w - mean)^2]: one exchange instead of two
template <int V, int NV, bool ODD, int WPR, int NW>
__device__ __forceinline__ void nr_normalise(float *x, int kind, const int *cnt, float inv_c, float eps, float own_inv_n, NrSum<WPR, NW> &sum, float &mean, float &rstd)
{
    float q = 0.f, none = 0.f;
    mean = 0.f;
    if (kind == NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV * V; ++i) s += x[i];
        s = nr_wave_sum(s, sum.g_log);
        mean = s * (WPR > 1 ? own_inv_n : inv_c);
        if constexpr (WPR > 1) {
#pragma unroll
            for (int i = 0; i < NV * V; ++i) {
                const float d = nr_has<ODD, V>(cnt[i / V], i % V) ? x[i] - mean : 0.f;
                q += d * d;
            }
            const float2 t = sum.exchange(s, nr_wave_sum(q, sum.g_log));
            mean = nr_wave_sum(t.x, sum.LOG) * inv_c;
            const float d = t.x * sum.inv_n - mean;
            q = nr_wave_sum(t.y + sum.n * d * d, sum.LOG);
        }
#pragma unroll
        for (int i = 0; i < NV * V; ++i) x[i] = nr_has<ODD, V>(cnt[i / V], i % V) ? x[i] - mean : 0.f;
    }
    if (WPR == 1 || kind != NORM_LAYER) {
#pragma unroll
        for (int i = 0; i < NV * V; ++i) q += x[i] * x[i];
        sum(q, none, false);
    }
    rstd = 1.f / sqrtf(q * inv_c + eps);
#pragma unroll
    for (int i = 0; i < NV * V; ++i) x[i] *= rstd;
}

// Forward.  The next row is asked for before the sums of the row in hand (latency behind work), parameters stay in registers; rows of up to 512
// channels have no barrier at all.  From 4096 channels on a row's chain of exchanges shows as much as memory does
template <int DT, int V, int NV, int WPR, bool ODD>
__global__ __launch_bounds__(WPR > 4 ? 64 * WPR : 256) void k_norm_fwd(const NormArgs a)
{
    typedef typename NrT<DT>::S S;
    constexpr int NT = WPR > 4 ? 64 * WPR : 256, NW = NT / 64, E = V * NV;
    __shared__ float2 red[2 * NW];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // (rows of 4 waves and more have a workgroup of their own, of as many waves as hold channels)
    const int G = WPR > 2 ? (int)blockDim.x : WPR > 1 ? 128 : 1 << a.g_log, lr = tid & (WPR > 2 ? 1023 : G - 1), RPB = WPR > 2 ? 1 : 256 / G;
    const int slot = WPR > 2 ? 0 : WPR > 1 ? wave >> 1 : tid >> a.g_log;       // (a scalar where whole waves share a row)
    const float inv_c = 1.f / (float)a.C;
    NrSum<WPR, NW> sum = nr_sum<WPR, NW, V, NV>(red, wave, a.g_log, G, a.C);
    unsigned col[NV];
    int cnt[NV];        // how many of a vector's channels exist
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        col[i] = (i * G + lr) * V;
        cnt[i] = a.C - (int)col[i];
    }
    const float own_inv_n = WPR > 1 ? __shfl(sum.inv_n, wave % WPR) : 0.f;
    constexpr bool KEEP = WPR < 16 || (E == 8 && DT != DT_F32);     // parameters and the next row stay in registers (16 waves leave a lane 128 of them: else asked for at their turn)
    const bool outer = a.y != nullptr && a.out_kind != NORM_NONE, inner = a.in_kind != NORM_NONE;
    float wo[E], bo[E], gate[E], wi[E], bi[E];
    if constexpr (KEEP) {
        nr_params<S, V, NV, ODD>(wo, a.wo, a.pf32, 0, col, cnt, 1.f);
        nr_params<S, V, NV, ODD>(bo, a.bo, a.pf32, 0, col, cnt, 0.f);
        nr_params<S, V, NV, ODD>(wi, a.wi, a.pf32, 0, col, cnt, 1.f);
        nr_params<S, V, NV, ODD>(bi, a.bi, a.pf32, 0, col, cnt, 0.f);
        if (!a.rows_per_gate) nr_params<S, V, NV, ODD>(gate, a.gate, a.pf32, 0, col, cnt, 1.f);
    }
    const long long hop = (long long)gridDim.x * RPB;
    NrRow<S, V, NV, ODD> ry, rh;
    long long row = (long long)blockIdx.x * RPB + slot;
    if constexpr (KEEP) {
        ry.ask(a.y, (size_t)row * a.ldy, col, cnt, row < a.M);
        rh.ask(a.h, (size_t)row * a.ldh, col, cnt, row < a.M);
    }
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.M; r0 += hop) {      // (uniform: every wave meets every barrier)
        const bool live = row < a.M;
        float x[E], mean_y = 0.f, rstd_y = 0.f, mean_h = 0.f, rstd_h = 0.f, h[E];
        if constexpr (!KEEP) {
            ry.ask(a.y, (size_t)row * a.ldy, col, cnt, live);
            rh.ask(a.h, (size_t)row * a.ldh, col, cnt, live);
        }
        ry.settle(col, cnt);
        rh.settle(col, cnt);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] = ry.at(i);
            h[i] = rh.at(i);
        }
        const long long next = row + hop;
        if (KEEP && r0 + hop < a.M) {
            ry.ask(a.y, (size_t)next * a.ldy, col, cnt, next < a.M);
            rh.ask(a.h, (size_t)next * a.ldh, col, cnt, next < a.M);
        }
        if (a.y) {
            if (!KEEP || a.rows_per_gate) nr_params<S, V, NV, ODD>(gate, live ? a.gate : nullptr, a.pf32, live && a.rows_per_gate ? (size_t)(row / a.rows_per_gate) * a.C : 0, col, cnt, 1.f);
            if (outer) {
                nr_normalise<V, NV, ODD>(x, a.out_kind, cnt, inv_c, a.eps, own_inv_n, sum, mean_y, rstd_y);
                if constexpr (!KEEP) {
                    nr_params<S, V, NV, ODD>(wo, a.wo, a.pf32, 0, col, cnt, 1.f);
                    nr_params<S, V, NV, ODD>(bo, a.bo, a.pf32, 0, col, cnt, 0.f);
                }
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = x[i] * wo[i] + bo[i];
            }
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = nr_has<ODD, V>(cnt[i / V], i % V) ? a.alpha * h[i] + gate[i] * x[i] : 0.f;
            if (live)
#pragma unroll
                for (int i = 0; i < NV; ++i) nr_store<S, V, ODD>(a.ho, (size_t)row * a.C, col[i], cnt[i], x + i * V);
        } else
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = h[i];
        if (inner) {
            nr_normalise<V, NV, ODD>(x, a.in_kind, cnt, inv_c, a.eps, own_inv_n, sum, mean_h, rstd_h);
            if constexpr (!KEEP) {
                nr_params<S, V, NV, ODD>(wi, a.wi, a.pf32, 0, col, cnt, 1.f);
                nr_params<S, V, NV, ODD>(bi, a.bi, a.pf32, 0, col, cnt, 0.f);
            }
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = x[i] * wi[i] + bi[i];
            if (live)
#pragma unroll
                for (int i = 0; i < NV; ++i) nr_store<S, V, ODD>(a.u, (size_t)row * a.C, col[i], cnt[i], x + i * V);
        }
        if (a.stats && live && lr == 0) *(float4 *)(a.stats + 4 * row) = float4{mean_y, rstd_y, mean_h, rstd_h};
        row = next;
    }
}

// the five column sums of a workgroup: lanes of a wave that hold the same channels of different rows add up by exchange, the waves' sums meet
// in the LDS in the order of the waves
template <int V, int NV, bool ODD, int WPR, int NW> __device__ __forceinline__ void nr_put_sums(float *lds, float *dst, float *acc, const unsigned *col, const int *cnt, int wave, int lr, int g_log)
{
    constexpr int E = V * NV, ROWS = WPR > 4 ? 1 : 4 / WPR;       // groups of waves with rows of their own
    if constexpr (WPR == 1)
#pragma unroll
        for (int i = 0; i < E; ++i)
            for (int m = 1 << g_log; m < 64; m <<= 1) acc[i] += __shfl_xor(acc[i], m);
    if constexpr (ROWS > 1) {
        const int lane = threadIdx.x & 63;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < E; ++i) lds[i * 256 + threadIdx.x] = acc[i];
        __syncthreads();
        if (wave >= WPR || (WPR == 1 && lane >> g_log)) return;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float t = 0.f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) t += lds[i * 256 + r * 64 * WPR + lr];
            acc[i] = t;
        }
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (nr_has<ODD, V>(cnt[i / V], i % V)) dst[col[i / V] + i % V] = acc[i];
}

// Backward, p = du * wi, n and n' the normalised y and h':
//   g = dh' + (p - mean(p) - n' mean(p n')) / dev'   (rms: without mean(p))     dh = scale * g     q = g * gate * wo
//   dy = (q - mean(q) - n mean(q n)) / dev           d gate = sum g (n wo + bo)   d wo = gate sum g n   d bo = gate sum g   d wi = sum du n'   d bi = sum du
// (rows of more than 8192 channels, 16 per lane: four sums of each would not fit the 128 registers of a lane; they go to k_norm_cols, and what is left
// still spills 184 - 356 bytes per lane, rows of any width of 4097 .. 8192 channels 44 - 116: their rates in the table above are those of spilling code.  GATES: so do
// those of many gates, and a row takes its own)
template <int DT, int V, int NV, int WPR, bool ODD, bool GATES>
__global__ __launch_bounds__(WPR > 4 ? 64 * WPR : 256, DT == DT_F32 || WPR > 4 || ODD ? 1 : 3) void k_norm_bwd(const NormArgs a)
{
    typedef typename NrT<DT>::S S;
    constexpr int NT = WPR > 4 ? 64 * WPR : 256, NW = NT / 64, E = V * NV;
    __shared__ float2 red[2 * NW];
    __shared__ float meet[WPR > 2 ? 1 : 256 * E];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // (rows of 4 waves and more have a workgroup of their own, of as many waves as hold channels)
    const int G = WPR > 2 ? (int)blockDim.x : WPR > 1 ? 128 : 1 << a.g_log, lr = tid & (WPR > 2 ? 1023 : G - 1), RPB = WPR > 2 ? 1 : 256 / G;
    const int slot = WPR > 2 ? 0 : WPR > 1 ? wave >> 1 : tid >> a.g_log;       // (a scalar where whole waves share a row)
    const float inv_c = 1.f / (float)a.C;
    NrSum<WPR, NW> sum = nr_sum<WPR, NW, V, NV>(red, wave, a.g_log, G, a.C);
    unsigned col[NV];
    int cnt[NV];        // how many of a vector's channels exist
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        col[i] = (i * G + lr) * V;
        cnt[i] = a.C - (int)col[i];
    }
    // workgroup b: chunk b % chunks of the rows of gate group b / chunks
    const int group = (int)blockIdx.x / a.chunks, chunk = (int)blockIdx.x % a.chunks;
    const int per_group = a.rows_per_gate ? a.rows_per_gate : a.M;
    const long long base = (long long)group * per_group;
    const int first = chunk * a.span, last = per_group - first < a.span ? per_group : first + a.span;
    size_t gate_at = a.rows_per_gate ? (size_t)group * a.C : 0;

    constexpr bool SUMS = E == 8 && !GATES;
    float s_g[E], s_gn[E], s_wi[E], s_bi[E];        // sums of g and g n (a workgroup's rows share their gate: three of the five sums follow), p n', p
#pragma unroll
    for (int i = 0; i < E; ++i) s_g[i] = s_gn[i] = s_wi[i] = s_bi[i] = 0.f;
    constexpr bool KEEP = WPR < 16;     // (as in k_norm_fwd)
    float wo[E], bo[E], gate[E], wi[E];
    auto outer = [&]() {
        nr_params<S, V, NV, ODD>(wo, a.wo, a.pf32, 0, col, cnt, 1.f);
        nr_params<S, V, NV, ODD>(bo, a.bo, a.pf32, 0, col, cnt, 0.f);
        nr_params<S, V, NV, ODD>(gate, a.gate, a.pf32, gate_at, col, cnt, 1.f);
    };
    if constexpr (KEEP) {
        outer();
        nr_params<S, V, NV, ODD>(wi, a.wi, a.pf32, 0, col, cnt, 1.f);
    }

    NrRow<S, V, NV, ODD> rgh, ry, rh, rgu;
    float4 rst;
    auto own_gate = [&](int r) {        // of a row (a gate of its own, or of few rows)
        gate_at = (size_t)((unsigned)(r < last ? r : last - 1) / (unsigned)a.gate_every) * a.C;
        if constexpr (KEEP) nr_params<S, V, NV, ODD>(gate, a.gate, a.pf32, gate_at, col, cnt, 1.f);
    };
    auto ask = [&](int r) {
        const bool live = r < last;
        const long long row = base + r;
        rst = live ? *(const float4 *)(a.stats + 4 * row) : float4{0.f, 0.f, 0.f, 0.f};
        ry.ask(a.y, (size_t)row * a.ldy, col, cnt, live);
        rh.ask(a.in_kind != NORM_NONE ? a.h : nullptr, (size_t)row * a.ldh, col, cnt, live);
        rgu.ask(a.gu, (size_t)row * a.ldgu, col, cnt, live);
        rgh.ask(a.gh, (size_t)row * a.ldgh, col, cnt, live);
    };
    if constexpr (KEEP) ask(first + slot);
    for (int r0 = first; r0 < last; r0 += RPB) {
        const bool live = r0 + slot < last;
        const size_t out = (size_t)(base + r0 + slot) * a.C;
        if constexpr (GATES) own_gate(r0 + slot);
        if constexpr (!KEEP) ask(r0 + slot);
        float n[E], g[E], p[E], hn[E];      // normalised y; gradient of h'; working row; normalised h'
        const float4 st = rst;
        ry.settle(col, cnt);
        rh.settle(col, cnt);
        rgu.settle(col, cnt);
        rgh.settle(col, cnt);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            n[i] = ry.at(i);
            g[i] = rgh.at(i);
            hn[i] = rh.at(i);
            p[i] = rgu.at(i);
        }
        if (KEEP && r0 + RPB < last) ask(r0 + RPB + slot);
        // (rows and channels that do not exist are zeros from here on: gradients zero, normalised values forced to zero)
        if (a.out_kind != NORM_NONE)
#pragma unroll
            for (int i = 0; i < E; ++i) n[i] = nr_has<ODD, V>(cnt[i / V], i % V) ? (n[i] - st.x) * st.y : 0.f;
        if (a.in_kind != NORM_NONE) {
            float m1 = 0.f, m2 = 0.f;
            if constexpr (!KEEP) {
                outer();
                nr_params<S, V, NV, ODD>(wi, a.wi, a.pf32, 0, col, cnt, 1.f);
            }
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if (a.y) hn[i] = a.alpha * hn[i] + gate[i] * (n[i] * wo[i] + bo[i]);
                hn[i] = nr_has<ODD, V>(cnt[i / V], i % V) ? (hn[i] - st.z) * st.w : 0.f;
                if constexpr (SUMS) {
                    s_wi[i] += p[i] * hn[i];
                    s_bi[i] += p[i];
                }
                p[i] *= wi[i];
                m1 += p[i] * hn[i];
                m2 += p[i];
            }
            sum(m1, m2, a.in_kind == NORM_LAYER);
            m1 *= inv_c;
            m2 = a.in_kind == NORM_LAYER ? m2 * inv_c : 0.f;
            if (!SUMS && a.means && live && lr == 0) *(float2 *)(a.means + 2 * (base + r0 + slot)) = float2{m1, m2};
#pragma unroll
            for (int i = 0; i < E; ++i) g[i] += st.w * (p[i] - m2 - hn[i] * m1);
        }
        if (a.need_dh && live)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float d[V];
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] = a.alpha * g[i * V + e];
                nr_store<S, V, ODD>(a.dh, out, col[i], cnt[i], d);
            }
        if (!a.y) continue;
        if constexpr (!KEEP) outer();
        float m1 = 0.f, m2 = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (!(live && nr_has<ODD, V>(cnt[i / V], i % V))) g[i] = 0.f;
            if constexpr (SUMS) {
                s_g[i] += g[i];
                s_gn[i] += g[i] * n[i];
            }
            p[i] = g[i] * gate[i] * wo[i];
            m1 += p[i] * n[i];
            m2 += p[i];
        }
        if (a.out_kind != NORM_NONE) {
            sum(m1, m2, a.out_kind == NORM_LAYER);
            m1 *= inv_c;
            m2 = a.out_kind == NORM_LAYER ? m2 * inv_c : 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) p[i] = st.y * (p[i] - m2 - n[i] * m1);
        }
        if (a.need_dy && live)
#pragma unroll
            for (int i = 0; i < NV; ++i) nr_store<S, V, ODD>(a.dy, out, col[i], cnt[i], p + i * V);
    }
    if (!SUMS || !a.part) return;
    float *dst = a.part + (size_t)blockIdx.x * 5 * a.C;
    if (a.y) {
        if constexpr (!KEEP) outer();
        float t[E];
        auto put = [&](int which) { nr_put_sums<V, NV, ODD, WPR, NW>(meet, dst + which * (size_t)a.C, t, col, cnt, wave, lr, a.g_log); };
#pragma unroll
        for (int i = 0; i < E; ++i) t[i] = wo[i] * s_gn[i] + bo[i] * s_g[i];
        put(0);
#pragma unroll
        for (int i = 0; i < E; ++i) t[i] = gate[i] * s_gn[i];
        put(1);
#pragma unroll
        for (int i = 0; i < E; ++i) t[i] = gate[i] * s_g[i];
        put(2);
    }
    nr_put_sums<V, NV, ODD, WPR, NW>(meet, dst + 3 * (size_t)a.C, s_wi, col, cnt, wave, lr, a.g_log);
    nr_put_sums<V, NV, ODD, WPR, NW>(meet, dst + 4 * (size_t)a.C, s_bi, col, cnt, wave, lr, a.g_log);
}

// the column sums of wide rows, or of many gates, in a second pass: with the rows' statistics and means known everything is element by element.
// A lane takes V channels, a workgroup a strip of 64 V of them and a run of rows, its four waves every fourth.  GATES: a run of gates (whole groups of
// rows), a wave a quarter of it: a gate's gradient is complete where its rows end, the four other sums go on
template <int DT, bool GATES> __global__ __launch_bounds__(256) void k_norm_cols(const NormArgs a)
{
    typedef typename NrT<DT>::S S;
    constexpr int V = NrT<DT>::V;
    __shared__ float meet[3][5 * V][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const unsigned col[1] = {(blockIdx.x * 64 + lane) * V};
    const int cnt[1] = {a.C - (int)col[0]};
    float wo[V], bo[V], gate[V], wi[V], s[5 * V];
    nr_params<S, V, 1, true>(wo, a.wo, a.pf32, 0, col, cnt, 1.f);
    nr_params<S, V, 1, true>(bo, a.bo, a.pf32, 0, col, cnt, 0.f);
    nr_params<S, V, 1, true>(wi, a.wi, a.pf32, 0, col, cnt, 1.f);
#pragma unroll
    for (int i = 0; i < 5 * V; ++i) s[i] = 0.f;
    auto add = [&](long long row) {
        const float4 st = *(const float4 *)(a.stats + 4 * row);
        const float2 mean = a.in_kind != NORM_NONE ? *(const float2 *)(a.means + 2 * row) : float2{0.f, 0.f};
        NrRow<S, V, 1, true> ry, rh, rgu, rgh;
        ry.ask(a.y, (size_t)row * a.ldy, col, cnt, true);
        rh.ask(a.in_kind != NORM_NONE ? a.h : nullptr, (size_t)row * a.ldh, col, cnt, true);
        rgu.ask(a.gu, (size_t)row * a.ldgu, col, cnt, true);
        rgh.ask(a.gh, (size_t)row * a.ldgh, col, cnt, true);
        ry.settle(col, cnt);
        rh.settle(col, cnt);
        rgu.settle(col, cnt);
        rgh.settle(col, cnt);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float n = a.out_kind != NORM_NONE ? (ry.at(e) - st.x) * st.y : ry.at(e);
            float g = rgh.at(e);
            if (a.in_kind != NORM_NONE) {
                const float h = a.y ? a.alpha * rh.at(e) + gate[e] * (n * wo[e] + bo[e]) : rh.at(e);
                const float hn = (h - st.z) * st.w, u = rgu.at(e);
                s[3 * V + e] += u * hn;
                s[4 * V + e] += u;
                g += st.w * (u * wi[e] - mean.y - hn * mean.x);
            }
            s[e] += g * (n * wo[e] + bo[e]);
            s[V + e] += g * gate[e] * n;
            s[2 * V + e] += g * gate[e];
        }
    };
    if constexpr (GATES) {
        const int groups = a.M / a.gate_every, g0 = ((int)blockIdx.y * 4 + wave) * a.span;
        const int g1 = groups - g0 < a.span ? groups : g0 + a.span;
        if (cnt[0] > 0)
            for (int group = g0; group < g1; ++group) {
                const size_t at = (size_t)group * a.C;
                nr_params<S, V, 1, true>(gate, a.gate, a.pf32, at, col, cnt, 1.f);
                for (int r = 0; r < a.gate_every; ++r) add((long long)group * a.gate_every + r);
                if (a.d_gate) {
                    if (a.pf32)
#pragma unroll
                        for (int p = 0; p < V; p += 4) nr_store<float, 4, true>(a.d_gate, at, col[0] + p, cnt[0] - p, s + p);
                    else nr_store<S, V, true>(a.d_gate, at, col[0], cnt[0], s);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] = 0.f;
            }
    } else {
        const int group = (int)blockIdx.y / a.chunks, chunk = (int)blockIdx.y % a.chunks, per_group = a.rows_per_gate ? a.rows_per_gate : a.M;
        const long long base = (long long)group * per_group;
        const int first = chunk * a.span, last = per_group - first < a.span ? per_group : first + a.span;
        nr_params<S, V, 1, true>(gate, a.gate, a.pf32, a.rows_per_gate ? (size_t)group * a.C : 0, col, cnt, 1.f);
        if (cnt[0] > 0)
#pragma unroll 2
            for (int r = first + wave; r < last; r += 4) add(base + r);
    }
    if (wave)
#pragma unroll
        for (int i = 0; i < 5 * V; ++i) meet[wave - 1][i][lane] = s[i];
    __syncthreads();
    if (wave) return;
    float *dst = a.part + (size_t)blockIdx.y * 5 * a.C + col[0];
#pragma unroll
    for (int i = 0; i < 5 * V; ++i) {
        const float t = ((s[i] + meet[0][i][lane]) + meet[1][i][lane]) + meet[2][i][lane];
        if (i % V < cnt[0]) dst[(size_t)(i / V) * a.C + i % V] = t;
    }
}

// column sums of the workgroups: 16 columns x 16 runs of workgroups per launch block, joined in a fixed order.  blockIdx.x: which of the four that
// run over all workgroups, behind them the gate's, each over its own group's workgroups
struct NormJoin {
    const float *part;
    void *out[5];
    int C, blocks, chunks, groups, f32;
};

template <int DT> __global__ __launch_bounds__(256) void k_norm_join(const NormJoin a)
{
    typedef typename NrT<DT>::S S;
    __shared__ float red[256];
    const int which = blockIdx.x < 4 ? (int)blockIdx.x + 1 : 0, c = (int)blockIdx.y * 16 + (threadIdx.x & 15), run = threadIdx.x >> 4;
    if (!a.out[which]) return;
    const bool per_group = which == 0;
    const int group = per_group ? (int)blockIdx.x - 4 : 0, b0 = group * a.chunks, nb = per_group ? a.chunks : a.blocks;
    float s = 0.f;
    if (c < a.C)
#pragma unroll 8
        for (int b = run; b < nb; b += 16) s += a.part[((size_t)(b0 + b) * 5 + which) * a.C + c];
    red[threadIdx.x] = s;
    __syncthreads();
    if (run == 0 && c < a.C) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) t += red[16 * r + threadIdx.x];
        const size_t at = (size_t)group * a.C + c;
        if (a.f32) ((float *)a.out[which])[at] = t;
        else ((S *)a.out[which])[at] = (S)t;
    }
}

// ------------------------------------------------------------------------------------------------------------------ host side
constexpr int NR_MAX_C = 16384, NR_CUS = 256;

struct NormShape { int E, WPR, waves, g_log; bool odd; };      // waves: those of a row that have channels

// lanes per row so that a lane owns eight channels (sixteen beyond 8192)
NormShape nr_shape(int C, int dtype)
{
    NormShape s = {8, 1, 1, 0, C % (dtype == DT_F32 ? 4 : 8) != 0};
    while (s.WPR < 16 && 64 * s.WPR * s.E < C) s.WPR *= 2;
    if (64 * s.WPR * s.E < C) s.E = 16;
    while (s.g_log < 6 && (s.E << s.g_log) < C) ++s.g_log;
    s.waves = (C + 64 * s.E - 1) / (64 * s.E);
    return s;
}

inline int nr_rows_per_block(const NormShape &s) { return s.WPR > 1 ? (s.WPR > 4 ? 1 : 4 / s.WPR) : 256 >> s.g_log; }

template <int DT, int V, int NV> int nr_go(bool bwd, const NormArgs &a, const NormShape &s, unsigned grid, hipStream_t st)
{
#define NR_GO(W)                                                                                       \
    if (s.WPR == W) {                                                                                  \
        const int T = W > 2 ? 64 * s.waves : 256;                                                      \
        if (bwd && a.gate_every) k_norm_bwd<DT, V, NV, W, true, true><<<grid, T, 0, st>>>(a);          \
        else if (bwd && s.odd) k_norm_bwd<DT, V, NV, W, true, false><<<grid, T, 0, st>>>(a);           \
        else if (bwd) k_norm_bwd<DT, V, NV, W, false, false><<<grid, T, 0, st>>>(a);                   \
        else if (s.odd) k_norm_fwd<DT, V, NV, W, true><<<grid, T, 0, st>>>(a);                         \
        else k_norm_fwd<DT, V, NV, W, false><<<grid, T, 0, st>>>(a);                                   \
        return nr_status();                                                                            \
    }
    if constexpr (V * NV == 8) {
        NR_GO(1)
        NR_GO(2)
        NR_GO(4)
        NR_GO(8)
    }
    NR_GO(16)
#undef NR_GO
    return BC_ERR_SHAPE;
}

template <int DT> int nr_launch(bool bwd, const NormArgs &a, const NormShape &s, unsigned grid, hipStream_t st)
{
    constexpr int V = NrT<DT>::V;
    return s.E == 8 ? nr_go<DT, V, 8 / V>(bwd, a, s, grid, st) : nr_go<DT, V, 16 / V>(bwd, a, s, grid, st);
}

int nr_dispatch(int dtype, bool bwd, const NormArgs &a, const NormShape &s, unsigned grid, hipStream_t st)
{
    switch (dtype) {
    case DT_F32: return nr_launch<DT_F32>(bwd, a, s, grid, st);
    case DT_F16: return nr_launch<DT_F16>(bwd, a, s, grid, st);
    default: return nr_launch<DT_BF16>(bwd, a, s, grid, st);
    }
}

inline int nr_esize(int dtype) { return dtype == DT_F32 ? 4 : 2; }

int nr_check(long long M, int C, int dtype, int out_kind, int in_kind, long long rows_per_gate, const void *gate, const void *y)
{
    if (dtype < 0 || dtype > 2) return BC_ERR_ELEM;
    if (M < 0 || C < 1 || C > NR_MAX_C || out_kind < 0 || out_kind > 2 || in_kind < 0 || in_kind > 2) return BC_ERR_SHAPE;
    if (M > 0x7fffffffll) return BC_ERR_RANGE;
    if (rows_per_gate < 0 || (rows_per_gate && (!gate || M % rows_per_gate))) return BC_ERR_SHAPE;
    if (rows_per_gate && M / rows_per_gate > 65535) return BC_ERR_RANGE;       // (a launch dimension)
    if (!y && (out_kind != NORM_NONE || gate || in_kind == NORM_NONE)) return BC_ERR_SHAPE;
    return BC_OK;
}

// the rows of a gate group divided evenly among whole workgroups (chunks)
struct NormChunks { int chunks, span, groups; };
NormChunks nr_split(long long M, long long rows_per_gate, int want, int rows_per_block)
{
    NormChunks c;
    const long long per = rows_per_gate ? rows_per_gate : M;
    c.groups = (int)(M / per);
    long long n = (want + c.groups - 1) / c.groups;
    const long long most = (per + rows_per_block - 1) / rows_per_block;
    if (n > most) n = most;
    long long span = (per + n - 1) / n;
    span = (span + rows_per_block - 1) / rows_per_block * rows_per_block;
    c.span = (int)span;
    c.chunks = (int)((per + span - 1) / span);
    return c;
}

// workgroups of a launch: as many as run at once, so that each asks for its parameters and its first row once.  Forward, 128 MB per tensor, bf16:
// 16384 x 4096 107 us with two per CU, 129 with sixteen; 22369 x 3000 129 and 239; 8192 x 8192 126 with one, 160 with sixteen; 32768 x 2048 108 with
// four, 148 with two.  fp32 rows of whole vectors saturate memory with half as many (32768 x 2048 193 us with two, 211 with four; 65154 x 1030 349
// with two, 230 with four).  Backward (ratios of times as the rule was made): 16384 x 4096 one per CU 0.92 of three (1024 x 4096 0.70: fewer sums to join);
// 43690 x 1536 three 0.84 of two (fp32 0.93 -- but 65154 x 1030 1.30)
int nr_fill(const NormShape &s, int dtype, bool bwd)
{
    if (bwd) return NR_CUS * (s.waves > 4 ? 1 : s.waves == 3 && dtype != DT_F32 ? 3 : 2);
    if (s.waves > 4) return NR_CUS * (s.waves > 8 ? 1 : 2);
    return NR_CUS * (dtype == DT_F32 && !s.odd ? (s.waves == 3 ? 3 : 2) : (s.waves == 3 ? 5 : 4));
}

NormChunks nr_rows_split(long long M, long long rows_per_gate, int dtype, const NormShape &s)
{
    return nr_split(M, rows_per_gate, nr_fill(s, dtype, true), nr_rows_per_block(s));
}

inline unsigned nr_strips(int C, int dtype) { const int v = 64 * 16 / (dtype == DT_F32 ? 4 : 2); return (unsigned)((C + v - 1) / v); }

// the backward pass's plan.  A workgroup of the rows' kernel keeps the sums of one gate, and leaves five fp32 numbers per channel.  Gates of so few rows
// that this is more than a tensor of the call holds (and more than the L2s do) take their sums in the second pass instead, a run of gates per
// wave: backward of 65535 x 4096 bf16 with a gate per row 11 MB of workspace and 1.7 ms, sums per gate 5.4 GB and 21 ms; 65528 x 1024 with a gate per 8
// rows 11 MB and 398 us, 168 MB and 758
struct NormPlan {
    NormChunks rows, sums;      // the workgroups of the rows' kernel, and those that leave column sums (GATES: span counts gates, of a wave)
    bool second, gates;
};

NormPlan nr_plan(long long M, long long rows_per_gate, int C, int dtype, const NormShape &s)
{
    NormPlan p;
    const long long groups = rows_per_gate ? M / rows_per_gate : 1, left = 20ll * C * groups;
    p.gates = left > (16ll << 20) && left > M * C * (dtype == DT_F32 ? 4 : 2);
    p.second = p.gates || s.E != 8;
    p.rows = nr_rows_split(M, p.gates ? 0 : rows_per_gate, dtype, s);
    const int want = (int)(1024 / nr_strips(C, dtype));
    if (p.gates) {
        p.sums.span = (int)((groups + 4 * want - 1) / (4 * want));
        p.sums.chunks = (int)((groups + 4ll * p.sums.span - 1) / (4ll * p.sums.span));
        p.sums.groups = 1;
    } else
        p.sums = p.second ? nr_split(M, rows_per_gate, want, 4) : p.rows;
    return p;
}

// (the rows' means first: whatever the sums' size, they start on 256 bytes)
long long nr_bwd_space(long long M, int C, const NormPlan &p) { return (p.second ? (8 * M + 255) / 256 * 256 : 0) + 20ll * C * p.sums.chunks * p.sums.groups; }

template <int DT> void nr_cols(const NormArgs &a, bool gates, dim3 grid, hipStream_t st)
{
    if (gates) k_norm_cols<DT, true><<<grid, 256, 0, st>>>(a);
    else k_norm_cols<DT, false><<<grid, 256, 0, st>>>(a);
}

}  // namespace

BC_EXPORT int bc_norm_residual_fwd(void *h_out, void *u, float *stats, const void *h, const void *y, const void *out_weight, const void *out_bias, const void *gate,
                                   const void *in_weight, const void *in_bias, long long M, int C, long long ldh, long long ldy, long long rows_per_gate, float residual_scale,
                                   float eps, int out_kind, int in_kind, int dtype, int params_f32, void *stream)
{
    const int rc = nr_check(M, C, dtype, out_kind, in_kind, rows_per_gate, gate, y);
    if (rc != BC_OK) return rc;
    if (ldh < C || (y && ldy < C)) return BC_ERR_SHAPE;
    if (M == 0) return BC_OK;
    if (!h || (y && !h_out) || (in_kind != NORM_NONE && !u)) return BC_ERR_NULL;
    const int e = nr_esize(dtype), pe = params_f32 ? 4 : e;
    const void *ts[] = {h, y, h_out, u}, *ps[] = {out_weight, out_bias, gate, in_weight, in_bias};
    for (int i = 0; i < 4; ++i)
        if (ts[i] && (uintptr_t)ts[i] % e) return BC_ERR_ALIGN;
    for (int i = 0; i < 5; ++i)
        if (ps[i] && (uintptr_t)ps[i] % pe) return BC_ERR_ALIGN;
    if (stats && (uintptr_t)stats % 16) return BC_ERR_ALIGN;
    NormArgs a = {};
    a.h = h; a.y = y; a.wo = out_weight; a.bo = out_bias; a.gate = gate; a.wi = in_weight; a.bi = in_bias;
    a.ho = h_out; a.u = u; a.stats = stats;
    a.ldh = ldh; a.ldy = ldy; a.M = (int)M; a.C = C; a.rows_per_gate = (int)rows_per_gate;
    a.out_kind = out_kind; a.in_kind = in_kind; a.pf32 = params_f32; a.alpha = residual_scale; a.eps = eps;
    const NormShape s = nr_shape(C, dtype);
    a.g_log = s.g_log;
    const long long blocks = (M + nr_rows_per_block(s) - 1) / nr_rows_per_block(s);
    const int fill = nr_fill(s, dtype, false);
    return nr_dispatch(dtype, false, a, s, (unsigned)(blocks < fill ? blocks : fill), (hipStream_t)stream);
}

BC_EXPORT long long bc_norm_residual_bwd_workspace(long long M, int C, long long rows_per_gate, int dtype)
{
    if (M < 1 || C < 1 || C > NR_MAX_C || dtype < 0 || dtype > 2 || rows_per_gate < 0 || (rows_per_gate && M % rows_per_gate)) return 0;
    return nr_bwd_space(M, C, nr_plan(M, rows_per_gate, C, dtype, nr_shape(C, dtype)));
}

BC_EXPORT int bc_norm_residual_bwd(void *dh, void *dy, void *d_out_weight, void *d_out_bias, void *d_gate, void *d_in_weight, void *d_in_bias, const void *gh, const void *gu,
                                   const float *stats, const void *h, const void *y, const void *out_weight, const void *out_bias, const void *gate, const void *in_weight,
                                   long long M, int C, long long ldh, long long ldy, long long ldgh, long long ldgu, long long rows_per_gate, float residual_scale, int out_kind,
                                   int in_kind, int dtype, int params_f32, void *workspace, long long workspace_bytes, void *stream)
{
    const int rc = nr_check(M, C, dtype, out_kind, in_kind, rows_per_gate, gate, y);
    if (rc != BC_OK) return rc;
    if (ldh < C || (y && ldy < C) || (gh && ldgh < C) || (gu && ldgu < C) || M == 0) return BC_ERR_SHAPE;
    if (!h || !stats || (dy && !y)) return BC_ERR_NULL;
    const int e = nr_esize(dtype), pe = params_f32 ? 4 : e;
    const void *ts[] = {h, y, gh, gu, dh, dy}, *ps[] = {out_weight, out_bias, gate, in_weight, d_out_weight, d_out_bias, d_gate, d_in_weight, d_in_bias};
    for (int i = 0; i < 6; ++i)
        if (ts[i] && (uintptr_t)ts[i] % e) return BC_ERR_ALIGN;
    for (int i = 0; i < 9; ++i)
        if (ps[i] && (uintptr_t)ps[i] % pe) return BC_ERR_ALIGN;
    if ((uintptr_t)stats % 16) return BC_ERR_ALIGN;
    const NormShape s = nr_shape(C, dtype);
    const NormPlan p = nr_plan(M, rows_per_gate, C, dtype, s);
    const NormChunks &c = p.rows, &q = p.sums;
    const bool sums = d_out_weight || d_out_bias || d_gate || d_in_weight || d_in_bias;
    if (sums && !workspace) return BC_ERR_NULL;
    if (sums && workspace_bytes < nr_bwd_space(M, C, p)) return BC_ERR_SHAPE;
    if (sums && (uintptr_t)workspace % 256) return BC_ERR_ALIGN;
    NormArgs a = {};
    a.h = h; a.y = y; a.wo = out_weight; a.bo = out_bias; a.gate = gate; a.wi = in_weight;
    a.stats = (float *)stats; a.gh = gh; a.gu = gu; a.dh = dh; a.dy = dy;
    a.means = sums && p.second ? (float *)workspace : nullptr;
    float *part = sums ? (float *)((char *)workspace + nr_bwd_space(M, C, p) - 20ll * C * q.chunks * q.groups) : nullptr;
    a.part = p.second ? nullptr : part;
    a.ldh = ldh; a.ldy = ldy; a.ldgh = ldgh; a.ldgu = ldgu; a.M = (int)M; a.C = C;
    a.rows_per_gate = p.gates ? 0 : (int)rows_per_gate;
    a.gate_every = p.gates ? (int)rows_per_gate : 0;
    a.out_kind = out_kind; a.in_kind = in_kind; a.pf32 = params_f32; a.alpha = residual_scale;
    a.need_dh = dh != nullptr; a.need_dy = dy != nullptr;
    a.g_log = s.g_log; a.span = c.span; a.chunks = c.chunks;
    const hipStream_t st = (hipStream_t)stream;
    const int r = nr_dispatch(dtype, true, a, s, (unsigned)(c.chunks * c.groups), st);
    if (r != BC_OK || !sums) return r;
    if (p.second) {
        a.part = part;
        a.span = q.span;
        a.chunks = q.chunks;
        a.d_gate = d_gate;
        const dim3 grid(nr_strips(C, dtype), (unsigned)(q.chunks * q.groups));
        switch (dtype) {
        case DT_F32: nr_cols<DT_F32>(a, p.gates, grid, st); break;
        case DT_F16: nr_cols<DT_F16>(a, p.gates, grid, st); break;
        default: nr_cols<DT_BF16>(a, p.gates, grid, st);
        }
    }
    NormJoin j = {};
    j.part = part;
    j.out[0] = p.gates ? nullptr : d_gate; j.out[1] = d_out_weight; j.out[2] = d_out_bias; j.out[3] = d_in_weight; j.out[4] = d_in_bias;
    j.C = C; j.blocks = q.chunks * q.groups; j.chunks = q.chunks; j.groups = q.groups; j.f32 = params_f32;
    const dim3 grid(4 + (j.out[0] ? (unsigned)q.groups : 0), (unsigned)((C + 15) / 16));
    switch (dtype) {
    case DT_F32: k_norm_join<DT_F32><<<grid, 256, 0, st>>>(j); break;
    case DT_F16: k_norm_join<DT_F16><<<grid, 256, 0, st>>>(j); break;
    default: k_norm_join<DT_BF16><<<grid, 256, 0, st>>>(j);
    }
    return nr_status();
}
