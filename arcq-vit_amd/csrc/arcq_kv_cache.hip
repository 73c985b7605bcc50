// Keys and values into the pages of a cache and back (arcq_kv_cache_write, arcq_kv_cache_read): 16-bit pages hold the values as
// they are, FP8 pages y = E4M3(x / 2^e) with one exponent e for each token and head,
//   e = min { e : max |x| <= 448 * 2^e }   (448 the largest E4M3 value), read off the exponent and mantissa of max |x|.
// Scaling by a power of two is exact, so a value rounds the same way whatever computes it.
//
// Bound by memory: every value is read once and written once.  A page keeps values in 16-byte pieces of w tokens of one
// dim, so that attention reads its operand without a transpose; the write turns them in LDS.  A workgroup takes a run
// of rows of one head that begins where a piece does (rows that lie in consecutive slots, as those of a prompt), and stores whole
// pieces; tokens that do not fill one (a decoding step: one token a sequence) are stored value by value.  65 536 rows of 8 heads of 128 to
// FP8 pages and back: 808 MB, 181 us, 4.5 TB/s where a copy reaches 5.2; a step of 64 rows 4.4 us, a launch.  32 rows a workgroup (24 and 48:
// 188 and 184 us); stores past the caches: 198 to 216.
#include "arcq_gemm.h"
#include "arcq_kv_pages.h"

#include <algorithm>

namespace arcq {
namespace {

constexpr int kRows = 64;            // rows a workgroup can hold

struct CacheArgs {
    unsigned char *kp, *vp;
    int8_t *ke, *ve;
    unsigned char *k, *v;            // rows: read by the write, written by the read
    const int64_t *slots;
    int64_t rows, num_slots;
    int64_t k_row, k_head, v_row, v_head;        // bytes
    int heads, dim, page_shift, run;             // run: rows a workgroup begins after the last one's
};

// The first of the rows r .. r + W - 1 whose slot begins a piece, r if there is none: runs that follow one another begin and end at
// the same row, because their beginnings are at least W rows apart.
template <int W>
__device__ __forceinline__ int64_t run_start(const CacheArgs &a, int64_t r, int lane)
{
    if (r == 0) return 0;
    if (r >= a.rows) return a.rows;
    const int64_t at = r + (lane & (W - 1));
    const int64_t s = at < a.rows ? a.slots[at] : -1;
    const uint64_t hit = __ballot(s >= 0 && (s & (W - 1)) == 0) & ((uint64_t(1) << W) - 1);
    return hit ? r + __builtin_ctzll(hit) : r;
}

// The rows of the workgroup: their slots; the rows that begin a whole piece (W rows in its W slots); the rows that are not in one.
struct Rows {
    int64_t slot[kRows];          // -1: left out
    int begins[kRows / 8], alone[kRows];
    int n_begins, n_alone;
};
// By the first wave (kRows = 64: a lane a row).
template <int W>
__device__ __forceinline__ void classify(const CacheArgs &a, int64_t start, int n, Rows &rows, int tid)
{
    if (tid >= 64) return;
    int64_t s = tid < n ? a.slots[start + tid] : -1;
    if (s < 0 || s >= a.num_slots) s = -1;
    rows.slot[tid] = s;
    const int64_t before = __shfl_up(s, 1);
    const uint64_t follows = __ballot(tid > 0 && s >= 0 && s == before + 1);        // in the slot behind the row before
    const uint64_t rest = ((uint64_t(1) << (W - 1)) - 1) << 1;                       // the W - 1 rows behind this one
    const bool begins = s >= 0 && (s & (W - 1)) == 0 && tid + W <= kRows && ((follows >> tid) & rest) == rest;
    const uint64_t all = __ballot(begins);
    // (beginnings are at least W rows apart: a piece's rows follow one another)
    const uint64_t near = all & (((uint64_t(2) << tid) - 1) & ~((uint64_t(1) << max(tid - (W - 1), 0)) - 1));     // rows tid - (W - 1) .. tid
    const bool alone = s >= 0 && near == 0;
    const uint64_t loose = __ballot(alone), lower = (uint64_t(1) << tid) - 1;
    if (begins) rows.begins[__popcll(all & lower)] = tid;
    if (alone) rows.alone[__popcll(loose & lower)] = tid;
    if (tid == 0) rows.n_begins = __popcll(all), rows.n_alone = __popcll(loose);
}
// Four values of one row's bytes each -> the bytes of four rows' values: a 4 x 4 transpose.
__device__ __forceinline__ void transpose4(uint32_t (&x)[4])
{
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    x[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    x[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    x[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    x[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}
// A thread's four bytes of each of a piece's rows (dims 4 or 2 of them) -> its pieces, and back.
template <bool F8>
__device__ __forceinline__ void to_pieces(const uint32_t *row, u32x4_t *piece)          // 16 rows -> 4 pieces; 8 rows -> 2
{
    if constexpr (F8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t x[4] = {row[4 * i], row[4 * i + 1], row[4 * i + 2], row[4 * i + 3]};
            transpose4(x);
#pragma unroll
            for (int d = 0; d < 4; ++d) piece[d][i] = x[d];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            piece[0][i] = __builtin_amdgcn_perm(row[2 * i + 1], row[2 * i], 0x05040100u);
            piece[1][i] = __builtin_amdgcn_perm(row[2 * i + 1], row[2 * i], 0x07060302u);
        }
    }
}
template <bool F8>
__device__ __forceinline__ void to_rows(const u32x4_t *piece, uint32_t *row)
{
    if constexpr (F8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t x[4] = {piece[0][i], piece[1][i], piece[2][i], piece[3][i]};
            transpose4(x);
#pragma unroll
            for (int t = 0; t < 4; ++t) row[4 * i + t] = x[t];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            row[2 * i] = __builtin_amdgcn_perm(piece[1][i], piece[0][i], 0x05040100u);
            row[2 * i + 1] = __builtin_amdgcn_perm(piece[1][i], piece[0][i], 0x07060302u);
        }
    }
}

__device__ __forceinline__ bool finite(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7fffffffu) < 0x7f800000u; }

// Sixteen values of a row, whose other values are in the LANES lanes of the group: their exponent and FP8 form.
template <typename T, int LANES>
__device__ __forceinline__ int to_fp8_row(const u32x4_t (&in)[2], u32x4_t &out)
{
    float v[16];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) unpack2(in[i >> 2][i & 3], v[2 * i], v[2 * i + 1], T{});
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, finite(v[i]) ? fabsf(v[i]) : 0.0f);
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    const uint32_t bits = __builtin_bit_cast(uint32_t, most);
    int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
    e = min(max(e, ExponentRange<T>::lo), ExponentRange<T>::hi);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float y = __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(v[i], -e), -448.0f, 448.0f);
        v[i] = finite(v[i]) ? y : __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int w = 0;
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], w, true);
        out[i] = static_cast<uint32_t>(w);
    }
    return e;
}
// ... and back, rounded to T (exactly, where the row was written from T).
template <typename T>
__device__ __forceinline__ void from_fp8_row(const u32x4_t &in, int e, u32x4_t (&out)[2])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int w = static_cast<int>(in[i]);
        const float a = __builtin_amdgcn_ldexpf(__builtin_amdgcn_cvt_f32_fp8(w, 0), e), b = __builtin_amdgcn_ldexpf(__builtin_amdgcn_cvt_f32_fp8(w, 1), e);
        const float c = __builtin_amdgcn_ldexpf(__builtin_amdgcn_cvt_f32_fp8(w, 2), e), d = __builtin_amdgcn_ldexpf(__builtin_amdgcn_cvt_f32_fp8(w, 3), e);
        out[i >> 1][2 * (i & 1)] = pack2(a, b, T{});
        out[i >> 1][2 * (i & 1) + 1] = pack2(c, d, T{});
    }
}

// Bytes of a value; where the piece begins that has a slot's values of dim d.
template <bool F8> constexpr int kSize = F8 ? 1 : 2;
template <int W>
__device__ __forceinline__ int64_t value_piece(const CacheArgs &a, int64_t slot, int head, int d)
{
    const int64_t ph = (slot >> a.page_shift) * a.heads + head;
    const int off = static_cast<int>(slot) & ((1 << a.page_shift) - 1);
    return (((ph << a.page_shift) / W + off / W) * a.dim + d) * 16;
}

template <typename T, bool F8, int LANES>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheArgs a)
{
    constexpr int W = F8 ? 16 : 8, SZ = kSize<F8>;
    extern __shared__ __attribute__((aligned(16))) unsigned char tile[];       // [kRows][dim] values of v
    __shared__ Rows rows;
    const int tid = threadIdx.x, lane = tid & 63;
    const int head = blockIdx.y;
    const int64_t start = run_start<W>(a, static_cast<int64_t>(blockIdx.x) * a.run, lane);
    const int n = static_cast<int>(run_start<W>(a, static_cast<int64_t>(blockIdx.x + 1) * a.run, lane) - start);
    const int part = tid % LANES;
    const bool busy = part < a.dim / 16;
    u32x4_t kin[2], vin[2];
    auto load = [&](int r) {                        // (a row that is left out too: it is there)
#pragma unroll
        for (int i = 0; i < 2; ++i) kin[i] = vin[i] = u32x4_t{0u, 0u, 0u, 0u};
        if (!busy || r >= n) return;
        const unsigned char *ks = a.k + (start + r) * a.k_row + head * a.k_head + part * 32;
        const unsigned char *vs = a.v + (start + r) * a.v_row + head * a.v_head + part * 32;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            kin[i] = *reinterpret_cast<const u32x4_t *>(ks + 16 * i);
            vin[i] = *reinterpret_cast<const u32x4_t *>(vs + 16 * i);
        }
    };
    load(tid / LANES);
    classify<W>(a, start, n, rows, tid);
    __syncthreads();
    const int page_mask = (1 << a.page_shift) - 1;
    for (int r = tid / LANES; r < n; r += 256 / LANES) {
        if (r >= 256 / LANES) load(r);
        const int64_t s = rows.slot[r];
        const int64_t ph = (s >> a.page_shift) * a.heads + head;
        const int off = static_cast<int>(s) & page_mask;
        unsigned char *kd = a.kp + (((ph * (a.dim / W)) << a.page_shift) + off) * 16;          // + piece * page_size * 16
        unsigned char *vd = tile + (r * a.dim + part * 16) * SZ;
        if constexpr (F8) {
            u32x4_t ko, vo;
            const int ek = to_fp8_row<T, LANES>(kin, ko), ev = to_fp8_row<T, LANES>(vin, vo);
            if (s >= 0 && busy) {
                *reinterpret_cast<u32x4_t *>(kd + (static_cast<int64_t>(part) << a.page_shift) * 16) = ko;
                *reinterpret_cast<u32x4_t *>(vd) = vo;
                if (part == 0) {
                    a.ke[(ph << a.page_shift) + off] = static_cast<int8_t>(ek);
                    a.ve[(ph << a.page_shift) + off] = static_cast<int8_t>(ev);
                }
            }
        } else if (s >= 0 && busy) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                *reinterpret_cast<u32x4_t *>(kd + (static_cast<int64_t>(2 * part + i) << a.page_shift) * 16) = kin[i];
                *reinterpret_cast<u32x4_t *>(vd + 16 * i) = vin[i];
            }
        }
    }
    __syncthreads();
    // The values, four bytes of a row a thread: whole pieces, then the rows that fill none.
    constexpr int PER = 4 / SZ;                                       // dims of a thread
    const int units = a.dim / PER, unit = tid % units, group = tid / units, groups = 256 / units;
    if (group >= groups) return;
    const unsigned char *column = tile + unit * 4;
    for (int i = group; i < rows.n_begins; i += groups) {
        const int r = rows.begins[i];
        uint32_t x[W];
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = *reinterpret_cast<const uint32_t *>(column + (r + j) * a.dim * SZ);
        u32x4_t piece[PER];
        to_pieces<F8>(x, piece);
        const int64_t s = rows.slot[r];
        u32x4_t *dst = reinterpret_cast<u32x4_t *>(a.vp + value_piece<W>(a, s, head, unit * PER));
#pragma unroll
        for (int d = 0; d < PER; ++d) dst[d] = piece[d];
    }
    for (int i = group; i < rows.n_alone; i += groups) {
        const int r = rows.alone[i];
        const uint32_t x = *reinterpret_cast<const uint32_t *>(column + r * a.dim * SZ);
        const int64_t s = rows.slot[r];
        unsigned char *dst = a.vp + value_piece<W>(a, s, head, unit * PER) + (s & (W - 1)) * SZ;
#pragma unroll
        for (int d = 0; d < PER; ++d) {
            if constexpr (F8) dst[16 * d] = static_cast<unsigned char>(x >> (8 * d));
            else *reinterpret_cast<uint16_t *>(dst + 16 * d) = static_cast<uint16_t>(x >> (16 * d));
        }
    }
}

template <typename T, bool F8, int LANES>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheArgs a)
{
    constexpr int W = F8 ? 16 : 8, SZ = kSize<F8>;
    extern __shared__ __attribute__((aligned(16))) unsigned char tile[];       // [kRows][dim] values of v
    __shared__ Rows rows;
    const int tid = threadIdx.x, lane = tid & 63;
    const int head = blockIdx.y;
    const int64_t start = run_start<W>(a, static_cast<int64_t>(blockIdx.x) * a.run, lane);
    const int n = static_cast<int>(run_start<W>(a, static_cast<int64_t>(blockIdx.x + 1) * a.run, lane) - start);
    classify<W>(a, start, n, rows, tid);
    __syncthreads();
    const int page_mask = (1 << a.page_shift) - 1;
    constexpr int PER = 4 / SZ;                                       // dims of a thread
    const int units = a.dim / PER, unit = tid % units, group = tid / units, groups = 256 / units;
    unsigned char *column = tile + unit * 4;
    for (int i = group < groups ? group : kRows; i < rows.n_begins; i += groups) {
        const int r = rows.begins[i];
        const u32x4_t *src = reinterpret_cast<const u32x4_t *>(a.vp + value_piece<W>(a, rows.slot[r], head, unit * PER));
        u32x4_t piece[PER];
#pragma unroll
        for (int d = 0; d < PER; ++d) piece[d] = src[d];
        uint32_t x[W];
        to_rows<F8>(piece, x);
#pragma unroll
        for (int j = 0; j < W; ++j) *reinterpret_cast<uint32_t *>(column + (r + j) * a.dim * SZ) = x[j];
    }
    for (int i = group < groups ? group : kRows; i < rows.n_alone; i += groups) {
        const int r = rows.alone[i];
        const int64_t s = rows.slot[r];
        const unsigned char *src = a.vp + value_piece<W>(a, s, head, unit * PER) + (s & (W - 1)) * SZ;
        uint32_t x = 0;
#pragma unroll
        for (int d = 0; d < PER; ++d) {
            if constexpr (F8) x |= static_cast<uint32_t>(src[16 * d]) << (8 * d);
            else x |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(src + 16 * d)) << (16 * d);
        }
        *reinterpret_cast<uint32_t *>(column + r * a.dim * SZ) = x;
    }
    __syncthreads();
    const int part = tid % LANES;
    if (part >= a.dim / 16) return;
    for (int r = tid / LANES; r < n; r += 256 / LANES) {
        const int64_t s = rows.slot[r];
        u32x4_t ko[2], vo[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) ko[i] = vo[i] = u32x4_t{0u, 0u, 0u, 0u};
        if (s >= 0) {
            const int64_t ph = (s >> a.page_shift) * a.heads + head;
            const int off = static_cast<int>(s) & page_mask;
            const unsigned char *ks = a.kp + (((ph * (a.dim / W)) << a.page_shift) + off) * 16;
            const unsigned char *vs = tile + (r * a.dim + part * 16) * SZ;
            if constexpr (F8) {
                from_fp8_row<T>(*reinterpret_cast<const u32x4_t *>(ks + (static_cast<int64_t>(part) << a.page_shift) * 16),
                                a.ke[(ph << a.page_shift) + off], ko);
                from_fp8_row<T>(*reinterpret_cast<const u32x4_t *>(vs), a.ve[(ph << a.page_shift) + off], vo);
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    ko[i] = *reinterpret_cast<const u32x4_t *>(ks + (static_cast<int64_t>(2 * part + i) << a.page_shift) * 16);
                    vo[i] = *reinterpret_cast<const u32x4_t *>(vs + 16 * i);
                }
            }
        }
        unsigned char *kd = a.k + (start + r) * a.k_row + head * a.k_head + part * 32;
        unsigned char *vd = a.v + (start + r) * a.v_row + head * a.v_head + part * 32;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            *reinterpret_cast<u32x4_t *>(kd + 16 * i) = ko[i];
            *reinterpret_cast<u32x4_t *>(vd + 16 * i) = vo[i];
        }
    }
}

template <typename T, bool F8>
void launch_cache(const CacheArgs &a, bool write, hipStream_t st)
{
    const int lds = kRows * a.dim * kSize<F8>;
    const dim3 grid(static_cast<uint32_t>((a.rows + a.run - 1) / a.run), static_cast<uint32_t>(a.heads));
#define GO(L)                                                                                                             \
    if (write) hipLaunchKernelGGL((cache_write_kernel<T, F8, L>), grid, dim3(256), lds, st, a);                           \
    else hipLaunchKernelGGL((cache_read_kernel<T, F8, L>), grid, dim3(256), lds, st, a)
    if (a.dim <= 32) { GO(2); }
    else if (a.dim <= 64) { GO(4); }
    else if (a.dim <= 128) { GO(8); }
    else { GO(16); }
#undef GO
}

int cache_checked(const char *fn, const arcq_kv_cache_args *p, bool write, void *stream)
{
    if (!p) return fail(ARCQ_ERR_NULL, "%s: NULL arguments", fn);
    if (const int rc = check_pages(fn, p->pages, p->dtype)) return rc;
    if (p->rows < 0) return fail(ARCQ_ERR_SHAPE, "%s: negative size", fn);
    if (p->rows == 0 || p->pages.heads == 0) return ARCQ_OK;
    if (!p->k || !p->v || !p->slots) return fail(ARCQ_ERR_NULL, "%s: NULL tensor pointer", fn);
    if (const int rc = check_page_pointers(fn, p->pages)) return rc;
    if (!rows_aligned(p->k, p->rows, p->k_row_stride, p->pages.heads, p->k_head_stride) ||
        !rows_aligned(p->v, p->rows, p->v_row_stride, p->pages.heads, p->v_head_stride))
        return fail(ARCQ_ERR_ALIGN, "%s: every row of k and v must be 16-byte aligned", fn);
    // (a grid's axis holds fewer than 2^32 threads: at 32 rows a workgroup of 256 fewer than 2^24 workgroups)
    if (p->rows > ((int64_t(1) << 24) - 1) * 32) return fail(ARCQ_ERR_SHAPE, "%s: too many rows", fn);
    CacheArgs a{};
    a.kp = static_cast<unsigned char *>(p->pages.k), a.vp = static_cast<unsigned char *>(p->pages.v);
    a.ke = p->pages.k_exponents, a.ve = p->pages.v_exponents;
    a.k = static_cast<unsigned char *>(p->k), a.v = static_cast<unsigned char *>(p->v), a.slots = p->slots;
    a.rows = p->rows, a.num_slots = p->pages.num_pages * p->pages.page_size;
    a.k_row = 2 * p->k_row_stride, a.k_head = 2 * p->k_head_stride, a.v_row = 2 * p->v_row_stride, a.v_head = 2 * p->v_head_stride;
    a.heads = static_cast<int>(p->pages.heads), a.dim = static_cast<int>(p->pages.head_dim), a.page_shift = log2_of(p->pages.page_size);
    const bool f8 = p->pages.dtype == ARCQ_FP8;
    // Rows of a workgroup, and up to W - 1 more (at most kRows); few rows: fewer, so that more of the chip takes part.
    a.run = a.rows * a.heads >= int64_t(32) * 4 * device_cus() ? 32 : 16;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p->dtype == ARCQ_F16) f8 ? launch_cache<_Float16, true>(a, write, st) : launch_cache<_Float16, false>(a, write, st);
    else f8 ? launch_cache<__bf16, true>(a, write, st) : launch_cache<__bf16, false>(a, write, st);
    return launch_status(fn);
}

}  // namespace
}  // namespace arcq

using namespace arcq;

ARCQ_API int arcq_kv_cache_write(const arcq_kv_cache_args *a, void *stream) { return cache_checked("arcq_kv_cache_write", a, true, stream); }

ARCQ_API int arcq_kv_cache_read(const arcq_kv_cache_args *a, void *stream) { return cache_checked("arcq_kv_cache_read", a, false, stream); }
