// Norm of every query and key head and its rotation by the token's position (arcq_qk_norm_rotary), one launch between the
// qkv layer and the cache: every value is read once and written once.
//
//   x' = (x - mean?) / sqrt(mean(.^2) + eps) * weight + bias
//   (a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t),   t = positions[axis][token] * inv_freq[pair]
//
// The angle is taken in turns and in 64 bits: positions * inv_freq / (2 pi) less its nearest integer is exact to 2^-33 of a turn
// at position 2^20, where a 32-bit product is off by a tenth of a radian; the nearest quarter goes the same way, and sine and cosine
// of what is left (an eighth of a turn at most) are short polynomials in 32 bits.
//
// Bound by memory: 16 384 tokens of 40 heads of 128 (336 MB) 66.0 us, 5.1 TB/s, a copy's rate; a step of 64 tokens 5.6 us, a launch and
// one round trip.  The angles are not: in 64 bits they cost as much as the rest where every head computes its own (170 us), so a
// workgroup computes each token's once for all its heads.
#include "arcq_gemm.h"
#include "arcq_kv_pages.h"

#include <algorithm>

namespace arcq {
namespace {

constexpr int kMaxDim = 256;
constexpr double kInvTwoPi = 0.15915494309189533576888, kHalfPi = 1.57079632679489661923132;

struct RotaryArgs {
    const void *in[2];               // q, k
    void *out[2];
    const float *weight[2], *bias[2];
    int64_t in_token[2], in_head[2], out_token[2], out_head[2];
    const void *positions;
    int64_t axis_stride, tokens;
    const double *inv_freq;
    int heads[2], dim, pairs, ends[ARCQ_ROTARY_AXES];      // ends[a]: the first pair behind axis a
    float eps, magnitude, inv_dim;
    int positions_i64, block, per_row;                      // rows kernel: tokens of a workgroup, heads of a grid row
};

// magnitude * (cos, sin) of pair i at the token's position.
__device__ __forceinline__ void angle_of(const RotaryArgs &a, int64_t token, int pair, float &c, float &s)
{
    int axis = 0;
#pragma unroll
    for (int i = 0; i < ARCQ_ROTARY_AXES - 1; ++i) axis += pair >= a.ends[i] ? 1 : 0;
    const int64_t at = axis * a.axis_stride + token;
    const double p = a.positions_i64 ? static_cast<double>(static_cast<const int64_t *>(a.positions)[at])
                                     : static_cast<double>(static_cast<const int32_t *>(a.positions)[at]);
    const double turns = p * a.inv_freq[pair] * kInvTwoPi;
    const double quarters = 4.0 * (turns - __builtin_rint(turns));          // [-2, 2]
    const double k = __builtin_rint(quarters);
    const float x = static_cast<float>((quarters - k) * kHalfPi), z = x * x;    // [-pi / 4, pi / 4]
    // Taylor's series: the first terms left out are below 2^-29
    float sn = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
    sn = __builtin_fmaf(z, sn, 1.0f / 120.0f);
    sn = __builtin_fmaf(z, sn, -1.0f / 6.0f);
    sn = __builtin_fmaf(x * z, sn, x);
    float cs = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    cs = __builtin_fmaf(z, cs, -1.0f / 720.0f);
    cs = __builtin_fmaf(z, cs, 1.0f / 24.0f);
    cs = __builtin_fmaf(z, cs, -0.5f);
    cs = __builtin_fmaf(z, cs, 1.0f);
    const int q = static_cast<int>(k) & 3;
    const float u = (q & 1) ? sn : cs, w = (q & 1) ? cs : sn;
    c = a.magnitude * (((q + 1) & 2) ? -u : u);
    s = a.magnitude * ((q & 2) ? -w : w);
}

template <typename T> __device__ __forceinline__ float load1(const T *p) { return static_cast<float>(*p); }

// Any head_dim, rotation and alignment: a wave for each head, the normed head in LDS.
template <typename T, int NORM, bool INTER>
__global__ void __launch_bounds__(256) rotary_any_kernel(const RotaryArgs a)
{
    __shared__ float rows[4][kMaxDim];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int heads = a.heads[0] + a.heads[1];
    const int64_t job = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 4 + wave;
    if (job >= a.tokens * heads) return;               // (no barrier below: a wave keeps to its own row)
    const int64_t token = job / heads;
    int head = static_cast<int>(job - token * heads);
    const int which = head >= a.heads[0] ? 1 : 0;
    head -= which ? a.heads[0] : 0;
    const T *in = static_cast<const T *>(a.in[which]) + token * a.in_token[which] + head * a.in_head[which];
    T *out = static_cast<T *>(a.out[which]) + token * a.out_token[which] + head * a.out_head[which];
    float v[kMaxDim / 64];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) {
        const int d = lane + 64 * i;
        v[i] = d < a.dim ? load1(in + d) : 0.0f;
        sum += v[i];
    }
    if (NORM == ARCQ_NORM_LAYER) {
#pragma unroll
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        const float mean = sum * a.inv_dim;
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i)
            if (lane + 64 * i < a.dim) v[i] -= mean;
    }
    if (NORM != ARCQ_NORM_NONE) {
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i) sq = __builtin_fmaf(v[i], v[i], sq);
#pragma unroll
        for (int o = 32; o; o >>= 1) sq += __shfl_xor(sq, o);
        const float inv = 1.0f / sqrtf(__builtin_fmaf(sq, a.inv_dim, a.eps));
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i) v[i] *= inv;
    }
    const float *w = a.weight[which], *b = a.bias[which];
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) {
        const int d = lane + 64 * i;
        if (d >= a.dim) break;
        if (w) v[i] *= w[d];
        if (b) v[i] += b[d];
        rows[wave][d] = v[i];
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) {
        const int d = lane + 64 * i;
        if (d >= a.dim) break;
        float y = v[i];
        if (d < 2 * a.pairs) {
            const bool second = INTER ? (d & 1) != 0 : d >= a.pairs;
            const int pair = INTER ? d >> 1 : second ? d - a.pairs : d;
            const float other = rows[wave][INTER ? d ^ 1 : second ? d - a.pairs : d + a.pairs];
            float c, s;
            angle_of(a, token, pair, c, s);
            y = second ? __builtin_fmaf(other, s, y * c) : __builtin_fmaf(-other, s, y * c);
        }
        out[d] = static_cast<T>(y);
    }
}

template <typename T> constexpr int kPieces = 8 * static_cast<int>(sizeof(T)) / 16;      // 16-byte loads of 8 values
template <typename T>
__device__ __forceinline__ void widen8(const u32x4_t *w, float *v)
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4_t x = __builtin_bit_cast(float4_t, w[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = x[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack2(w[0][j], v[2 * j], v[2 * j + 1], T{});
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float *v)
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4_t w = {v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
            *reinterpret_cast<float4_t *>(p + 4 * i) = w;
        }
    } else {
        u32x4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], T{});
        *reinterpret_cast<u32x4_t *>(p) = w;
    }
}
// Eight consecutive floats in LDS.
__device__ __forceinline__ void read8(const float *p, float *v)
{
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float4_t x = *reinterpret_cast<const float4_t *>(p + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = x[j];
    }
}

// 16-byte rows, head_dim a multiple of 16.  A workgroup has `block` tokens and the heads [first, last) of grid row y.  It begins with the
// sines and cosines of its tokens, each once, and the weights in LDS; then a group of LANES lanes takes one head of one token at a
// time, the next one's values on their way.  A lane has two pieces of 8 values of each: two in a row for neighbours; for halves those
// that keep a pair's values in one lane (i and i + pairs / 8; of what does not turn two in a row) where pairs are a multiple of 8, else
// two in a row too, and a pair's other value comes through LDS (75 338 tokens of 12 heads of 32, 7 pairs: 35 us; by the kernel above 304).
enum : int { kHalves = 0, kNeighbours = 1, kHalvesAny = 2 };
template <typename T, int NORM, int HOW, int LANES>
__global__ void __launch_bounds__(256) rotary_rows_kernel(const RotaryArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float lds[];        // [q, k][weight, bias][dim], [block][cos, sin][pitch], [groups][row]
    constexpr int GROUPS = 256 / LANES;
    const int tid = threadIdx.x, lane = tid % LANES, group = tid / LANES;
    const int64_t token0 = static_cast<int64_t>(blockIdx.x) * a.block;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(a.block), a.tokens - token0));
    const int heads = a.heads[0] + a.heads[1];
    const int first = blockIdx.y * a.per_row, n = min(heads, first + a.per_row) - first;
    const bool busy = lane < a.dim / 16;                      // (LANES is a power of two)
    const int turned = a.pairs / 4;                           // pieces that turn (kHalves)
    const bool turns = HOW == kHalves && lane < turned / 2;
    int piece[2] = {turns ? lane : 2 * lane, turns ? lane + turned / 2 : 2 * lane + 1};
    if (!busy) piece[0] = piece[1] = 0;

    u32x4_t raw[2][kPieces<T>];
    int t = group / n, h = group - t * n;                     // the token and head at hand
    auto load = [&]() {
        const int head = first + h, which = head >= a.heads[0] ? 1 : 0;
        const T *src = static_cast<const T *>(which ? a.in[1] : a.in[0]) + (token0 + t) * (which ? a.in_token[1] : a.in_token[0]) +
                       (head - (which ? a.heads[0] : 0)) * (which ? a.in_head[1] : a.in_head[0]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < kPieces<T>; ++j) raw[i][j] = *reinterpret_cast<const u32x4_t *>(src + piece[i] * 8 + j * (16 / sizeof(T)));
    };
    if (t < tokens) load();
    float *trig = lds + 4 * a.dim;
    const bool weighted = a.weight[0] || a.weight[1], biased = a.bias[0] || a.bias[1];
    for (int i = tid; i < 4 * a.dim; i += 256) {
        const int what = i / a.dim, d = i - what * a.dim;
        const float *p = (what & 1) ? ((what & 2) ? a.bias[1] : a.bias[0]) : ((what & 2) ? a.weight[1] : a.weight[0]);
        lds[i] = p ? p[d] : (what & 1) ? 0.0f : 1.0f;
    }
    const int pitch = HOW == kNeighbours ? a.dim / 2 : (a.pairs + 3) / 4 * 4;       // (neighbours: behind the pairs, angles of zero)
    for (int i = tid; i < tokens * pitch; i += 256) {
        const int at = i / pitch, pair = i - at * pitch;
        float c = 1.0f, s = 0.0f;
        if (pair < a.pairs) angle_of(a, token0 + at, pair, c, s);
        trig[(2 * at) * pitch + pair] = c;
        trig[(2 * at + 1) * pitch + pair] = s;
    }
    float *row = trig + 2 * a.block * pitch + group * (a.dim + a.dim / 16);          // value d at d + d / 16: no two lanes' in one bank
    __syncthreads();
    while (t < tokens) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 2; ++i) widen8<T>(raw[i], v + 8 * i);
        const int head = first + h, which = head >= a.heads[0] ? 1 : 0;
        T *dst = static_cast<T *>(which ? a.out[1] : a.out[0]) + (token0 + t) * (which ? a.out_token[1] : a.out_token[0]) +
                 (head - (which ? a.heads[0] : 0)) * (which ? a.out_head[1] : a.out_head[0]);
        const float *cp = trig + 2 * t * pitch, *sp = cp + pitch;
        for (h += GROUPS; h >= n; h -= n) ++t;
        if (t < tokens) load();
        if (!busy)
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 0.0f;
        if (NORM == ARCQ_NORM_LAYER) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += v[i];
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) sum += __shfl_xor(sum, o);
            const float mean = busy ? sum * a.inv_dim : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] -= mean;
        }
        if (NORM != ARCQ_NORM_NONE) {
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sq = __builtin_fmaf(v[i], v[i], sq);
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) sq += __shfl_xor(sq, o);
            const float inv = 1.0f / sqrtf(__builtin_fmaf(sq, a.inv_dim, a.eps));
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= inv;
        }
        const float *wp = lds + 2 * which * a.dim;
        if (weighted) {
            float w[16];
#pragma unroll
            for (int i = 0; i < 2; ++i) read8(wp + piece[i] * 8, w + 8 * i);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= w[i];
        }
        if (biased) {
            float b[16];
#pragma unroll
            for (int i = 0; i < 2; ++i) read8(wp + a.dim + piece[i] * 8, b + 8 * i);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] += b[i];
        }
        float y[16];
        if constexpr (HOW == kHalvesAny) {
            if (busy)
#pragma unroll
                for (int i = 0; i < 16; ++i) row[17 * lane + i] = v[i];
            __builtin_amdgcn_wave_barrier();                   // (a group's lanes are in one wave, whose LDS accesses keep their order)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int d = 16 * lane + i;
                y[i] = v[i];
                if (d < 2 * a.pairs) {
                    const bool second = d >= a.pairs;
                    const int pair = second ? d - a.pairs : d, o = second ? d - a.pairs : d + a.pairs;
                    const float other = row[o + (o >> 4)], sn = sp[pair];
                    y[i] = __builtin_fmaf(second ? other : -other, sn, v[i] * cp[pair]);
                }
            }
            __builtin_amdgcn_wave_barrier();
        } else {
            float c[8], s[8];
            if (HOW == kNeighbours || turns) {
                read8(cp + (busy ? 8 * lane : 0), c);
                read8(sp + (busy ? 8 * lane : 0), s);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = 1.0f, s[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int p = HOW == kNeighbours ? 2 * i : i, q = HOW == kNeighbours ? 2 * i + 1 : 8 + i;
                y[p] = __builtin_fmaf(-v[q], s[i], v[p] * c[i]);
                y[q] = __builtin_fmaf(v[p], s[i], v[q] * c[i]);
            }
            // What does not turn is taken as it is: turned by an angle of zero an infinity would make its partner NaN, and -0 become 0.
            if (2 * a.pairs < a.dim) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int p = HOW == kNeighbours ? 2 * i : i, q = HOW == kNeighbours ? 2 * i + 1 : 8 + i;
                    const bool pair = HOW == kNeighbours ? 8 * lane + i < a.pairs : turns;
                    y[p] = pair ? y[p] : v[p];
                    y[q] = pair ? y[q] : v[q];
                }
            }
        }
        if (busy)
#pragma unroll
            for (int i = 0; i < 2; ++i) store8(dst + piece[i] * 8, y + 8 * i);
    }
}

template <typename T, int NORM, int HOW>
void launch_rows(RotaryArgs &a, hipStream_t st)
{
    const int heads = a.heads[0] + a.heads[1];
    const int lanes = a.dim <= 32 ? 2 : a.dim <= 64 ? 4 : a.dim <= 128 ? 8 : 16;
    // As many tokens as give every lane group one and a half heads, while the chip has four workgroups a compute unit: fewer leave the
    // beginning of a workgroup (positions, weights) uncovered, more leave a ragged end.  12 608 tokens of 12 heads of 64: 1, 4, 8, 12, 22
    // tokens 20.7, 12.1, 12.1, 13.1, 15.5 us; 16 384 of 40 of 128: 1, 2, 4, 8 tokens 71.2, 66.8, 68.7, 73.3.  Few tokens: the heads of one in
    // as many workgroups as leave every group one.
    const int groups = 256 / lanes;
    const int64_t fill = a.tokens / (4 * device_cus());
    a.block = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(3 * groups / 2 + heads - 1) / heads, fill, 4096 / (a.dim / 2)})));
    a.block = static_cast<int>(std::max<int64_t>(a.block, (a.tokens + (1 << 24) - 2) / ((1 << 24) - 1)));          // (a grid's axis: below 2^32 threads)
    const int most_y = a.block > 1 || heads <= groups ? 1 : static_cast<int>(std::min<int64_t>((heads + groups - 1) / groups, std::max<int64_t>(1, 2 * device_cus() / a.tokens)));
    a.per_row = (heads + most_y - 1) / most_y;
    const int rows_y = (heads + a.per_row - 1) / a.per_row;               // (no row without heads: 289 in 18 rows of 17 would leave the last one none)
    const dim3 grid(static_cast<uint32_t>((a.tokens + a.block - 1) / a.block), static_cast<uint32_t>(rows_y));
    const int pitch = HOW == kNeighbours ? a.dim / 2 : (a.pairs + 3) / 4 * 4;
    const int lds = 4 * (4 * a.dim + 2 * a.block * pitch + (HOW == kHalvesAny ? groups * (a.dim + a.dim / 16) : 0));      // (below 54 KB)
    switch (lanes) {
    case 2: hipLaunchKernelGGL((rotary_rows_kernel<T, NORM, HOW, 2>), grid, dim3(256), lds, st, a); break;
    case 4: hipLaunchKernelGGL((rotary_rows_kernel<T, NORM, HOW, 4>), grid, dim3(256), lds, st, a); break;
    case 8: hipLaunchKernelGGL((rotary_rows_kernel<T, NORM, HOW, 8>), grid, dim3(256), lds, st, a); break;
    default: hipLaunchKernelGGL((rotary_rows_kernel<T, NORM, HOW, 16>), grid, dim3(256), lds, st, a); break;
    }
}
template <typename T, int NORM, bool INTER>
void launch_rotary(RotaryArgs &a, bool rows, hipStream_t st)
{
    if (rows && INTER) return launch_rows<T, NORM, kNeighbours>(a, st);
    if (rows && a.pairs % 8 == 0) return launch_rows<T, NORM, kHalves>(a, st);
    if (rows) return launch_rows<T, NORM, kHalvesAny>(a, st);
    const int64_t groups = (a.tokens * (a.heads[0] + a.heads[1]) + 3) / 4, wide = std::min<int64_t>(groups, 1 << 20);     // (a grid's axis: below 2^32 threads)
    const dim3 grid(static_cast<uint32_t>(wide), static_cast<uint32_t>((groups + wide - 1) / wide));
    hipLaunchKernelGGL((rotary_any_kernel<T, NORM, INTER>), grid, dim3(256), 0, st, a);
}
template <typename T>
void launch_rotary_type(RotaryArgs &a, int norm, bool inter, bool rows, hipStream_t st)
{
    if (norm == ARCQ_NORM_NONE) inter ? launch_rotary<T, ARCQ_NORM_NONE, true>(a, rows, st) : launch_rotary<T, ARCQ_NORM_NONE, false>(a, rows, st);
    else if (norm == ARCQ_NORM_RMS) inter ? launch_rotary<T, ARCQ_NORM_RMS, true>(a, rows, st) : launch_rotary<T, ARCQ_NORM_RMS, false>(a, rows, st);
    else inter ? launch_rotary<T, ARCQ_NORM_LAYER, true>(a, rows, st) : launch_rotary<T, ARCQ_NORM_LAYER, false>(a, rows, st);
}

}  // namespace
}  // namespace arcq

using namespace arcq;

ARCQ_API int arcq_qk_norm_rotary(const arcq_qk_norm_rotary_args *p, void *stream)
{
    const char *fn = "arcq_qk_norm_rotary";
    if (!p) return fail(ARCQ_ERR_NULL, "%s: NULL arguments", fn);
    if (p->dtype != ARCQ_F16 && p->dtype != ARCQ_BF16 && p->dtype != ARCQ_F32)
        return fail(ARCQ_ERR_DTYPE, "%s: dtype must be ARCQ_F16, ARCQ_BF16 or ARCQ_F32", fn);
    if (p->norm < ARCQ_NORM_NONE || p->norm > ARCQ_NORM_LAYER) return fail(ARCQ_ERR_UNSUPPORTED, "%s: unknown norm %d", fn, p->norm);
    if (p->tokens < 0 || p->q_heads < 0 || p->k_heads < 0 || p->pairs < 0) return fail(ARCQ_ERR_SHAPE, "%s: negative size", fn);
    if (p->head_dim < 2 || p->head_dim > kMaxDim || p->head_dim % 2 != 0)
        return fail(ARCQ_ERR_UNSUPPORTED, "%s: head_dim must be even and at most %d (got %lld)", fn, kMaxDim, static_cast<long long>(p->head_dim));
    if (2 * p->pairs > p->head_dim) return fail(ARCQ_ERR_SHAPE, "%s: more pairs than head_dim / 2", fn);
    if (p->axes < 1 || p->axes > ARCQ_ROTARY_AXES) return fail(ARCQ_ERR_UNSUPPORTED, "%s: one to %d axes", fn, ARCQ_ROTARY_AXES);
    RotaryArgs a{};
    int64_t end = 0;
    for (int i = 0; i < ARCQ_ROTARY_AXES; ++i) {
        if (i < p->axes && p->sections[i] < 0) return fail(ARCQ_ERR_SHAPE, "%s: negative section", fn);
        end += i < p->axes ? p->sections[i] : 0;
        a.ends[i] = static_cast<int>(i < p->axes - 1 ? end : p->pairs);
    }
    if (end != p->pairs) return fail(ARCQ_ERR_SHAPE, "%s: the sections hold %lld pairs, not %lld", fn, static_cast<long long>(end), static_cast<long long>(p->pairs));
    if (!(p->eps >= 0.0f)) return fail(ARCQ_ERR_SHAPE, "%s: eps must not be negative", fn);
    // (values of a tensor: below 2^39, or the angles of a workgroup's tokens would not fit its LDS)
    const int64_t most = int64_t(1) << 32;
    if (p->q_heads > (1 << 20) || p->k_heads > (1 << 20) || p->tokens >= most || p->tokens * (p->q_heads + p->k_heads) >= most ||
        p->tokens * p->head_dim >= int64_t(1) << 37)
        return fail(ARCQ_ERR_SHAPE, "%s: tensor too large", fn);
    if (p->tokens * (p->q_heads + p->k_heads) == 0) return ARCQ_OK;
    if ((p->q_heads && (!p->q || !p->q_out)) || (p->k_heads && (!p->k || !p->k_out)) || (p->pairs && (!p->positions || !p->inv_freq)))
        return fail(ARCQ_ERR_NULL, "%s: NULL tensor pointer", fn);
    const int64_t strides[8] = {p->q_token_stride, p->q_head_stride, p->q_out_token_stride, p->q_out_head_stride,
                                p->k_token_stride, p->k_head_stride, p->k_out_token_stride, p->k_out_head_stride};
    const int size = p->dtype == ARCQ_F32 ? 4 : 2;
    bool rows = p->head_dim % 16 == 0;
    for (int i = 0; i < 8; ++i) {
        const int64_t heads = i < 4 ? p->q_heads : p->k_heads;           // (a dimension of one entry has any stride)
        rows = rows && (!heads || (i % 2 ? heads : p->tokens) == 1 || strides[i] * size % 16 == 0);
    }
    for (const void *q : {p->q, static_cast<const void *>(p->q_out)}) rows = rows && (!p->q_heads || aligned(q, 16));
    for (const void *k : {p->k, static_cast<const void *>(p->k_out)}) rows = rows && (!p->k_heads || aligned(k, 16));
    a.in[0] = p->q, a.in[1] = p->k, a.out[0] = p->q_out, a.out[1] = p->k_out;
    a.weight[0] = p->q_weight, a.weight[1] = p->k_weight, a.bias[0] = p->q_bias, a.bias[1] = p->k_bias;
    a.in_token[0] = p->q_token_stride, a.in_head[0] = p->q_head_stride, a.out_token[0] = p->q_out_token_stride, a.out_head[0] = p->q_out_head_stride;
    a.in_token[1] = p->k_token_stride, a.in_head[1] = p->k_head_stride, a.out_token[1] = p->k_out_token_stride, a.out_head[1] = p->k_out_head_stride;
    a.positions = p->positions, a.axis_stride = p->axis_stride, a.tokens = p->tokens, a.inv_freq = p->inv_freq;
    a.heads[0] = static_cast<int>(p->q_heads), a.heads[1] = static_cast<int>(p->k_heads);
    a.dim = static_cast<int>(p->head_dim), a.pairs = static_cast<int>(p->pairs), a.positions_i64 = p->positions_i64 ? 1 : 0;
    a.eps = p->eps, a.magnitude = p->magnitude, a.inv_dim = 1.0f / static_cast<float>(p->head_dim);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool inter = p->interleaved != 0;
    if (p->dtype == ARCQ_F32) launch_rotary_type<float>(a, p->norm, inter, rows, st);
    else if (p->dtype == ARCQ_BF16) launch_rotary_type<__bf16>(a, p->norm, inter, rows, st);
    else launch_rotary_type<_Float16>(a, p->norm, inter, rows, st);
    return launch_status(fn);
}
