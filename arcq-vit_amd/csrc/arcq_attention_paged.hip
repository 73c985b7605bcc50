// Attention of new tokens over the pages of a cache (arcq_attention_paged_fwd).
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q . k_j - m),   m the running maximum
//
// over the keys j that the token sees: those of its sequence up to its position (causal), the last `window` of them, or all.
//
// Rows.  The query heads that share a key head are the same keys' columns: a sequence's rows are its (token, head of the group)
// pairs, token first, and a tile is 32 or 128 consecutive rows.  The grid does not know the sequences' lengths (they are on the
// device): it has as many workgroups as there can be tiles and parts of their keys, and each finds its own from the lengths
// (find_item), which also say how long a part is: all blocks of all tiles over the workgroups that the chip takes at once.  A split by the
// table's width alone left short sequences' workgroups idle: 64 sequences of 1 to 8 192 keys, 8 key heads of 128: 276 us, so 187.
//
// Softmax.  One pass: the maximum m and the sum are per lane and row, in 32 bits, and the outputs are rescaled when m grows.
//
// Bounds.  Few rows (a step): the pages are read once at the rate at which memory is read: 6.0 TB/s, of which the 64 sequences
// above reach 5.4 (1 010 MB, 187 us, the join's launch of 5 us included), the FP8 pages of two of 130 000 keys 5.3 (537 MB, 101 us; 5.6 in
// the first launch alone).  Many rows: the matrix pipe.  A 32 x 32 x 16 instruction
// takes 32 clocks of its SIMD, the softmax between two products about as long in vector instructions, and what a wave leaves idle the other
// one of its SIMD fills only in part: a chunk of 2 048 tokens behind 6 000 keys (32 heads of 128, 8 key heads) 238 us, 990 TFLOP/s, the
// matrix pipe busy 46 % of all clocks; a library product of 8 192^3 reaches 1 210.
//
// Products.  As in the attention of an image: S^T = K Q^T with the keys as the matrix instruction's rows, so that a lane (row
// lane % 32 of the tile, half h = lane / 32) holds 16 of a block's 32 keys of its own row, and eight consecutive registers of
// them, rounded to 16 bits, are the second operand of O^T = V^T P^T.  Which token stands in which row of K is free: with
// token 16 (r / 8) + 8 h + r % 8 (FP8 pages: 16 h + r) behind register r of half h, the eight values of V^T that belong to the
// registers 8 i .. 8 i + 7 are one 16-byte piece of a page (eight bytes of one).  So are the eight values of a key row: a page's layout
// is that of the operands, both are loaded from memory into operand registers, 512 bytes of consecutive addresses for 32 lanes.
//
// FP8 pages: a key's exponent belongs to its row of K, one lane, and is applied as the values are widened (exact).  A value's belongs to a column
// of P^T.  With bf16 it is applied to the probabilities; fp16 has no room for that (2^-14 of a probability leaves its normal numbers at 2^-8 of
// the largest: 65 536 keys of values of 0.01 behind one of a score 12 higher were off by 24 %), so there every value is widened with
// its own exponent (exact), which is then no longer a part of the probabilities' range.
//
// Range.  Probabilities carry a factor 2^shift, FP8 values of bf16 another (Range below); both cancel in the end.  fp16: 2^8, so that many small
// probabilities behind one large stay above its subnormals for longer.  bf16: as small as keeps the sum of n keys finite in fp32 whatever
// finite values they have: the mean of values near the type's end is finite, its numerator need not be.  (What that takes from the other end: a term
// keeps all of fp32's bits while probability times value is above 2^-125 n 2^kSlack, 2^-106 for 8 192 keys.)
#include "arcq_gemm.h"
#include "arcq_kv_pages.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace arcq {
namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kNegInf = -__builtin_inff();
// A row's maximum: kNegInf if it sees no key (its result is zero), kLowest if it sees some and none has a score above minus infinity (0 / 0).
constexpr float kLowest = -3.402823466e38f;
__device__ __forceinline__ float row_maximum(float m, bool sees) { return sees ? fmaxf(m, kLowest) : m; }
// How far a score may be above the reference (in powers of two) before that follows, in the kernel of many rows.  (0: a chunk of 2 048 tokens 4 %
// slower; 16, which only bf16 probabilities have room for: no faster.)
constexpr int kSlack = 6;
constexpr int kShiftF16 = 8;

// Division of 0 .. 2^30 - 1 by a number known on the host: l = ceil(log2 d), m = ceil(2^(30 + l) / d) < 2^32; m d exceeds 2^(30 + l) by less
// than 2^l, n times that by less than 2^(30 + l), so the quotient is exact.
struct Divide {
    uint32_t m;
    int shift;
    Divide() = default;
    explicit Divide(int d)
    {
        int l = 0;
        while ((1 << l) < d) ++l;
        shift = 30 + l;
        m = static_cast<uint32_t>(((uint64_t(1) << shift) + d - 1) / d);
    }
    __device__ __forceinline__ int operator()(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> shift); }
};

// The factors of probabilities (2^shift) and of FP8 values whose exponents go to the probabilities (value_scale); back: the latter's inverse, for
// the result.  bf16, sums of up to 2^n keys, probabilities of up to 2^(shift + slack):
//   16-bit pages  2^n * 2^(shift + slack) * |v| < 2^128 / 2
//   FP8           P = p 2^e is a bf16 number at both ends of e, 2^(119 + 8) and 2^(-110 + 8 - slack) less 18 powers;
//                 2^n * 2^127 * 448 * value_scale < 2^128
struct Range {
    float shift, value_scale, back;
    Range(int dtype, bool f8, int64_t keys, int slack)
    {
        const int n = log2_of(std::max<int64_t>(keys, 1));
        const bool scaled = dtype == ARCQ_BF16 && f8;
        shift = static_cast<float>(dtype == ARCQ_F16 ? kShiftF16 : f8 ? 8 - slack : -(n + slack + 1));
        value_scale = scaled ? std::ldexp(1.0f, -(n + 9)) : 1.0f;
        back = scaled ? std::ldexp(1.0f, n + 9) : 1.0f;
    }
};

struct PagedArgs {
    const unsigned char *kp, *vp;
    const int8_t *ke, *ve;
    const unsigned char *q;
    unsigned char *out;
    const int32_t *table, *q_offsets, *kv_lengths;
    float *part_o;                   // [items * kv_heads * TILE][dim]: sums of a part's rows
    float2 *part_ml;                 // [items * kv_heads * TILE]: maximum (in powers of two) and sum of the probabilities
    int2 *part_at;                   // [tokens * q_heads]: the row of the first part above, and the number of parts, -1 if out is written already
    int64_t q_token, q_head, out_token, out_head, table_stride;      // q, out: bytes
    int64_t tokens, table_width, num_pages, part_rows;
    int q_heads, kv_heads, group, sequences, page_shift, window, causal;
    int slots, min_blocks;           // items that the chip takes at once for each key head (0: tiles are not split), and the least blocks of one
    float c2;                        // scale * log2(e)
    float shift, value_scale, back;  // Range
    Divide by_group, by_kv_heads, by_q_heads;
};

// A kernel's factors: constants for fp16, else read with its first arguments (where they are used first they cost short steps a round trip each:
// a step of four short sequences 7.44 us in place of 7.35).
template <typename T, bool F8>
struct Factors {
    float shift = kShiftF16, value_scale = 1.0f, back = 1.0f;
    __device__ __forceinline__ explicit Factors(const PagedArgs &a)
    {
        if constexpr (!std::is_same<T, _Float16>::value) {
            shift = a.shift;
            asm volatile("" : "+s"(shift));
            if constexpr (F8) {
                value_scale = a.value_scale, back = a.back;
                asm volatile("" : "+s"(value_scale), "+s"(back));
            }
        }
    }
};

__device__ __forceinline__ int offset_of(const PagedArgs &a, int b) { return min(max(a.q_offsets[b], 0), static_cast<int>(a.tokens)); }

// A sequence: its new tokens and keys, its tiles of TILE rows, and blocks of 2^SHIFT keys that one of them has about.
template <int TILE, int SHIFT>
struct Sequence {
    int begin, queries, len, tiles, blocks;
    __device__ __forceinline__ Sequence(const PagedArgs &a, int b, bool there)
    {
        const int at = min(b, a.sequences - 1);
        int first = a.q_offsets[at], behind = a.q_offsets[at + 1], keys = a.kv_lengths[at];
        asm volatile("" : "+v"(first), "+v"(behind), "+v"(keys));         // (one wait for the three: else they are loaded one by one, where they are used)
        begin = min(max(first, 0), static_cast<int>(a.tokens));
        queries = there ? max(min(max(behind, 0), static_cast<int>(a.tokens)) - begin, 0) : 0;
        len = min(max(keys, 0), static_cast<int>(a.table_width << a.page_shift));         // (below 2^30)
        tiles = (queries * a.group + TILE - 1) / TILE;
        blocks = (len + (1 << SHIFT) - 1) >> SHIFT;
        if (a.window) blocks = min(blocks, ((a.window + TILE / a.group) >> SHIFT) + 2);
    }
    // Parts of each tile, `per` blocks to one.
    __device__ __forceinline__ int parts(const PagedArgs &a, int per) const { return a.slots ? max(1, (blocks + per - 1) / per) : 1; }
};
// Sums of a lane and all before it, within 16 lanes, then with the last lane of the 16 and of the 32 before: no round trip through LDS.
template <int CONTROL, int ROWS> struct Step { static constexpr int control = CONTROL, rows = ROWS; };
template <typename T, typename Move>
__device__ __forceinline__ T sums(T s, Move move)
{
    s += move(s, Step<0x111, 0xf>{});
    s += move(s, Step<0x112, 0xf>{});
    s += move(s, Step<0x114, 0xf>{});
    s += move(s, Step<0x118, 0xf>{});
    s += move(s, Step<0x142, 0xa>{});
    s += move(s, Step<0x143, 0xc>{});
    return s;
}
// The sum over all lanes, the same register for them.
__device__ __forceinline__ double sum_all(double x)
{
    const uint64_t s = __builtin_bit_cast(uint64_t, sums(x, [](double v, auto step) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), step.control, step.rows, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), step.control, step.rows, 0xf, false);
        return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
    }));
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(s), 63), hi = __builtin_amdgcn_readlane(static_cast<int>(s >> 32), 63);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// The sum over the lanes before this one; of all, the same register for all lanes.
__device__ __forceinline__ int sum_before(int x, int &all)
{
    const int s = sums(x, [](int v, auto step) { return __builtin_amdgcn_update_dpp(0, v, step.control, step.rows, 0xf, false); });
    all = __builtin_amdgcn_readlane(s, 63);
    return s - x;
}

// What a workgroup does: one part of the keys of one tile of rows.
struct Item {
    int b, token0, queries, len;       // sequence: its first token, new tokens, keys
    int row0, rows;                    // first row of the tile within the sequence, rows of the sequence
    int lo, hi;                        // keys that some row of the tile sees
    int k0, k1;                        // blocks of the part
    int part, parts, first;            // first: the item of the tile's first part
};
// Item `item` of a key head, false if there are fewer.  The lengths are on the device, so the split is made there: all blocks of all
// tiles over `slots` are the blocks of a part, the items of a sequence are its tiles' parts.  64 sequences (or runs of sequences) at
// a time; up to 64 there is one round of loads.
template <int TILE, int SHIFT>
__device__ __forceinline__ bool find_item(const PagedArgs &a, int item, int lane, Item &it)
{
    typedef Sequence<TILE, SHIFT> Seq;
    const int run = (a.sequences + 63) / 64;
    int base = 0, n = a.sequences, rem = item, per = 1 << 30;
    const Seq own(a, lane * run, lane * run < a.sequences);          // (the only one of its lane up to 64 sequences)
    if (a.slots) {
        double all = static_cast<double>(own.tiles) * own.blocks;       // (exact: whole numbers below 2^53)
        for (int i = 1; i < run; ++i) {
            const int b = lane * run + i;
            const Seq s(a, b, b < a.sequences);
            all += static_cast<double>(s.tiles) * s.blocks;
        }
        all = sum_all(all);
        per = __builtin_amdgcn_readfirstlane(max(a.min_blocks, static_cast<int>(fmin(all / a.slots, 1e9)) + 1));
    }
    if (run > 1) {
        int mine = 0, all;
        for (int i = 0; i < run; ++i) {
            const int b = lane * run + i;
            const Seq s(a, b, b < a.sequences);
            mine += s.tiles * s.parts(a, per);
        }
        const int before = sum_before(mine, all);
        if (rem >= all) return false;
        const int l = __builtin_ctzll(__ballot(before + mine > rem));
        rem -= __builtin_amdgcn_readlane(before, l);
        base = l * run;
        n = min(run, a.sequences - base);
    }
    for (int w = 0; w < n; w += 64) {
        const Seq s = run == 1 ? own : Seq(a, base + w + lane, w + lane < n);
        int all;
        const int parts = s.parts(a, per), mine = s.tiles * parts, before = sum_before(mine, all);
        if (rem >= all) {
            rem -= all;
            continue;
        }
        const int l = __builtin_ctzll(__ballot(before + mine > rem));
        rem -= __builtin_amdgcn_readlane(before, l);
        it.b = base + w + l;
        it.token0 = __builtin_amdgcn_readlane(s.begin, l);
        it.queries = __builtin_amdgcn_readlane(s.queries, l);
        it.len = __builtin_amdgcn_readlane(s.len, l);
        it.parts = __builtin_amdgcn_readlane(parts, l);
        const int t = it.parts == 1 ? rem : rem / it.parts;                 // the last tile first: it has the most keys
        it.part = rem - t * it.parts;
        it.first = item - it.part;
        it.rows = it.queries * a.group;
        it.row0 = (__builtin_amdgcn_readlane(s.tiles, l) - 1 - t) * TILE;
        it.lo = 0;
        it.hi = it.len;
        if (a.causal) {
            const int first = a.by_group(it.row0), last = a.by_group(min(it.row0 + TILE, it.rows) - 1);
            it.hi = min(max(it.len - it.queries + last + 1, 0), it.len);
            if (a.window) it.lo = max(it.len - it.queries + first + 1 - a.window, 0);
        }
        const int b0 = it.lo >> SHIFT, blocks = it.hi > it.lo ? ((it.hi - 1) >> SHIFT) + 1 - b0 : 0;
        const int each = it.parts == 1 ? blocks : (blocks + it.parts - 1) / it.parts;
        it.k0 = __builtin_amdgcn_readfirstlane(b0 + min(blocks, it.part * each));      // (said to the compiler: one range for all lanes)
        it.k1 = __builtin_amdgcn_readfirstlane(b0 + min(blocks, (it.part + 1) * each));
        return true;
    }
    return false;
}

template <typename T> struct Vec8;
template <> struct Vec8<_Float16> { typedef half8_t type; };
template <> struct Vec8<__bf16> { typedef bf16x8_t type; };
__device__ __forceinline__ float16_t mfma(u32x4_t a, u32x4_t b, float16_t c, _Float16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ float16_t mfma(u32x4_t a, u32x4_t b, float16_t c, __bf16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// Eight FP8 values times a power of two.
__device__ __forceinline__ u32x4_t widen(uint32_t lo, uint32_t hi, float scale, _Float16)
{
    u32x4_t o;
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true));
    return o;
}
__device__ __forceinline__ u32x4_t widen(uint32_t lo, uint32_t hi, float scale, __bf16)
{
    u32x4_t o;
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return o;
}
// FP8 pages: the values' exponents are applied as they are widened, else to the probabilities.
template <typename T, bool F8> constexpr bool kScaleValues = false;
template <> constexpr bool kScaleValues<_Float16, true> = true;
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, static_cast<uint32_t>(127 + e) << 23); }

typedef short short2_t __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ int exponent_of(const u32x4_t &e, int i) { return __builtin_amdgcn_sbfe(static_cast<int>(e[i >> 2]), 8 * (i & 3), 8); }
// fp16: the powers of two of two tokens' values, times 2^8, so that those of fp16 rows (exponents -14 to 7) are normal numbers.  Pages that were
// written from another type: zero below -22, infinity above 7.  An exponent's byte goes to the top of 16 bits, then to fp16's field.
__device__ __forceinline__ half2_t scales_of(uint32_t e, bool upper)               // (of the upper two of four exponents)
{
    const uint32_t two = __builtin_amdgcn_perm(0u, e, upper ? 0x030c020cu : 0x010c000cu);
    const short2_t top = __builtin_elementwise_min(__builtin_elementwise_max(__builtin_bit_cast(short2_t, two), short2_t{-23 * 256, -23 * 256}),
                                                   short2_t{8 * 256, 8 * 256});
    return __builtin_bit_cast(half2_t, __builtin_bit_cast(ushort2_t, top) * ushort2_t{4, 4} + ushort2_t{23 << 10, 23 << 10});
}
// Eight FP8 values, each times its token's power of two: exact (2^-8 of an FP8 value is fp16's).
__device__ __forceinline__ u32x4_t widen_each(uint32_t lo, uint32_t hi, const half2_t *scale)
{
    u32x4_t o = widen(lo, hi, 1.0f / 256.0f, _Float16{});
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t two = o[i];                 // (a copy: a bit cast of a vector's element takes the first one)
        o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, two) * scale[i]);
    }
    return o;
}

// The token behind row m of a 32-key block of K.
template <bool F8>
__device__ __forceinline__ int token_of_row(int m)
{
    const int h = (m >> 2) & 1, r = 4 * (m >> 3) + (m & 3);
    return F8 ? 16 * h + r : 16 * (r >> 3) + 8 * h + (r & 7);
}
// The token behind register r of half h: half_token(h) + reg_token(r).
template <bool F8>
__device__ __forceinline__ int half_token(int h) { return F8 ? 16 * h : 8 * h; }
template <bool F8>
__device__ __forceinline__ constexpr int reg_token(int r) { return F8 ? r : 16 * (r >> 3) + (r & 7); }

// The keys [lo, hi) that a row sees, counted from the token of a block's first register.  (Opaque: else the compiler keeps a bound less
// each register's token in a register of its own through the whole loop.)
struct Seen {
    int lo, hi;
    __device__ __forceinline__ Seen(int row_lo, int row_hi, int first) : lo(row_lo - first), hi(row_hi - first)
    {
        asm volatile("" : "+v"(lo), "+v"(hi));
    }
    __device__ __forceinline__ bool operator()(int token) const { return token >= lo && token < hi; }
};
// Keeps the values of a 16-byte piece whose tokens first .. first + W - 1 are in [lo, hi).
template <bool F8>
__device__ __forceinline__ void keep_tokens(u32x4_t &v, int first, int lo, int hi)
{
    constexpr int PER = F8 ? 4 : 2, BITS = F8 ? 8 : 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t mask = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int t = first + PER * i + j;
            mask |= t >= lo && t < hi ? ((BITS == 8 ? 0xffu : 0xffffu) << (BITS * j)) : 0u;
        }
        v[i] &= mask;
    }
}

// Infinities and NaN among the values of a block that not all rows of the tile see whole: a probability of zero does not keep them out
// of a product.  Does a register of 16-bit values hold one?
template <typename T> constexpr uint32_t kExponent = 0x7c00u;
template <> constexpr uint32_t kExponent<__bf16> = 0x7f80u;
template <typename T>
__device__ __forceinline__ bool odd16(uint32_t w)
{
    constexpr uint32_t e = kExponent<T>;
    return (w & e) == e || (w & (e << 16)) == e << 16;
}
__device__ __forceinline__ bool odd8(uint32_t w)          // four FP8 values: NaN is 0x7f or 0xff
{
    return ((((w & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u) != 0;
}
// Where row r of part `part` of an item's tile lies among the parts.
template <int TILE>
__device__ __forceinline__ int64_t part_row(const PagedArgs &a, const Item &t, int kv, int part, int r)
{
    return (static_cast<int64_t>(t.first + part) * a.kv_heads + kv) * TILE + r;
}
template <int TILE>
__device__ __forceinline__ void say_parts(const PagedArgs &a, const Item &t, int kv, int r, int64_t at, float m, float l)
{
    if (!a.slots) return;
    if (t.part == 0) a.part_at[at] = make_int2(static_cast<int>(part_row<TILE>(a, t, kv, 0, r)), t.parts == 1 ? -1 : t.parts);
    if (t.parts > 1) a.part_ml[part_row<TILE>(a, t, kv, t.part, r)] = make_float2(m, l);
}
// A lane's half of its row: the result, or the part's sums.
template <typename T, int D, int TILE = 32>
__device__ __forceinline__ void store_rows(const PagedArgs &a, float back, const Item &t, int kv, int row, int lh, float m, float l, const float16_t (&o)[D / 32])
{
    const int tok = a.by_group(row), head = kv * a.group + row - tok * a.group;
    const int64_t token = static_cast<int64_t>(t.token0) + tok;
    if (t.parts == 1) {
        const float inv = m == kNegInf ? 0.0f : back / l;
        unsigned char *dst = a.out + token * a.out_token + head * a.out_head;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                u32x2_t w;
                w[0] = pack2(o[j][4 * r] * inv, o[j][4 * r + 1] * inv, T{});
                w[1] = pack2(o[j][4 * r + 2] * inv, o[j][4 * r + 3] * inv, T{});
                *reinterpret_cast<u32x2_t *>(dst + 2 * (32 * j + 8 * r + 4 * lh)) = w;
            }
    } else {
        float *dst = a.part_o + part_row<TILE>(a, t, kv, t.part, row - t.row0) * D;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4_t w = {o[j][4 * r], o[j][4 * r + 1], o[j][4 * r + 2], o[j][4 * r + 3]};
                *reinterpret_cast<float4_t *>(dst + 32 * j + 8 * r + 4 * lh) = w;
            }
    }
    if (lh == 0) say_parts<TILE>(a, t, kv, row - t.row0, token * a.q_heads + head, m, l);
}

// A tile by the definition, row by row and key by key: for one that has values which are not finite where some of its rows must not see
// them, or a page that does not exist.  A wave takes a row at a time, 64 keys' scores at once, a lane the dims lane + 64 i.  It is for tiles
// that hardly ever are, and slow: a chunk of 2 048 tokens behind 6 000 keys, 32 heads of 128, a NaN in its last value: 58 ms, without it 0.24.
template <typename T, bool F8, int D, int TILE, int SHIFT, int WAVES>
__device__ __forceinline__ void careful_tile(const PagedArgs &a, const Factors<T, F8> &f, const Item &t, int kv, int wave, int lane)
{
    constexpr int W = F8 ? 16 : 8, SZ = F8 ? 1 : 2, PER = (D + 63) / 64;
    const int32_t *table = a.table + t.b * a.table_stride;
    const int page_mask = (1 << a.page_shift) - 1;
    auto value = [&](const unsigned char *p, int e) -> float {
        if constexpr (F8) return __builtin_amdgcn_ldexpf(__builtin_amdgcn_cvt_f32_fp8(*p, 0), e);
        else return static_cast<float>(*reinterpret_cast<const T *>(p));
    };
    for (int r = wave; r < TILE && t.row0 + r < t.rows; r += WAVES) {
        const int row = t.row0 + r, tok = a.by_group(row), head = kv * a.group + row - tok * a.group;
        const int64_t token = static_cast<int64_t>(t.token0) + tok;
        int lo = 0, hi = t.len;
        if (a.causal) {
            hi = min(max(t.len - t.queries + tok + 1, 0), t.len);
            if (a.window) lo = max(t.len - t.queries + tok + 1 - a.window, 0);
        }
        const bool sees = hi > lo;
        lo = max(lo, t.k0 << SHIFT), hi = min(hi, t.k1 << SHIFT);
        const T *q = reinterpret_cast<const T *>(a.q + token * a.q_token + head * a.q_head);
        float m = kNegInf, l = 0.0f, o[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = 0.0f;
        for (int base = lo; base < hi; base += 64) {
            const int n = min(64, hi - base), key = base + min(lane, n - 1);
            const int page = table[key >> a.page_shift], off = key & page_mask;
            const bool there = page >= 0 && page < a.num_pages;
            const int64_t slot = ((static_cast<int64_t>(there ? page : 0) * a.kv_heads + kv) << a.page_shift) + off;
            const int ek = F8 ? a.ke[slot] : 0, ev = F8 ? a.ve[slot] : 0;
            const unsigned char *k = a.kp + (slot - off) * (D * SZ) + off * 16;
            float s = 0.0f;
            for (int d = 0; d < D; ++d)
                s = __builtin_fmaf(static_cast<float>(q[d]), value(k + (static_cast<int64_t>(d / W) << a.page_shift) * 16 + d % W * SZ, ek), s);
            s = !there ? __builtin_nanf("") : s * a.c2;
            float bm = lane < n ? s : kNegInf;
#pragma unroll
            for (int x = 32; x; x >>= 1) bm = fmaxf(bm, __shfl_xor(bm, x));
            const float m_new = fmaxf(m, bm), base2 = m_new == kNegInf ? 0.0f : m_new;
            const float alpha = __builtin_amdgcn_exp2f(m - base2);
            const float p = lane < n ? __builtin_amdgcn_exp2f(s - base2 + f.shift) : 0.0f;
            float sum = p;
#pragma unroll
            for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
            l = l * alpha + sum;
            m = m_new;
#pragma unroll
            for (int i = 0; i < PER; ++i) o[i] *= alpha;
            for (int j = 0; j < n; ++j) {
                const float pj = __shfl(p, j);
                const int64_t sj = __shfl(slot, j);
                const int oj = __shfl(off, j), ej = __shfl(ev, j);
                const unsigned char *v = a.vp + (sj - oj) * (D * SZ) + oj / W * D * 16 + oj % W * SZ;
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (lane + 64 * i < D) o[i] = __builtin_fmaf(pj, value(v + (lane + 64 * i) * 16, ej) * f.value_scale, o[i]);
            }
        }
        m = row_maximum(m, sees);
        const bool alone = t.parts == 1;
        const float inv = m == kNegInf ? 0.0f : f.back / l;
        T *dst = reinterpret_cast<T *>(a.out + token * a.out_token + head * a.out_head);
        const int64_t at = part_row<TILE>(a, t, kv, t.part, r) * D;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int d = lane + 64 * i;
            if (d >= D) break;
            if (alone) dst[d] = static_cast<T>(o[i] * inv);
            else a.part_o[at + d] = o[i];
        }
        if (lane == 0) say_parts<TILE>(a, t, kv, r, token * a.q_heads + head, m, l);
    }
}

// ---- few rows: a workgroup of WAVES waves has one tile of 32 rows and one part of its keys, the waves take the blocks of 32 keys in
// turn, straight from memory into operand registers, and are joined in LDS ----
//
// Every byte of a page is used once, so LDS would be a detour: a lane's 16-byte loads are its operands.  A block's keys are asked for as soon
// as the one before has been multiplied, its values after theirs, so that 16 KB (128 dims) a wave are on their way through the softmax; two
// waves a SIMD keep registers for that without spilling (four: 8 KB each and slower).  The page table would be a second round trip
// in front of every load, so a lane holds the page of one half of one of the next 32 blocks.
template <typename T, bool F8, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1)))
paged_rows_kernel(const PagedArgs a)
{
    constexpr int KF = D / 16;                     // operand registers (of 16 bytes) of 32 keys' K
    constexpr int NB = D / 32;                     // 32-dim blocks of the output
    constexpr int KL = F8 ? D / 32 : D / 16;       // 16-byte loads of K, and of V
    constexpr int W = F8 ? 16 : 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = WAVES == 1 ? 0 : tid >> 6;
    const int lr = lane & 31, lh = lane >> 5;
    const int place = a.by_kv_heads(blockIdx.x), kv = blockIdx.x - place * a.kv_heads;
    const Factors<T, F8> range(a);
    Item t;
    if (!find_item<32, 5>(a, place, lane, t)) return;
    const int k0 = t.k0, k1 = t.k1;

    // ---- this lane's row ----
    const int row = t.row0 + lr;
    const bool live = row < t.rows;
    const int tok = live ? a.by_group(row) : 0, gh = live ? row - tok * a.group : 0;
    const int head = kv * a.group + gh;
    int lo = t.lo, hi = t.hi;                       // (a lane without a row: the tile's)
    if (a.causal && live) {
        hi = min(max(t.len - t.queries + tok + 1, 0), t.len);
        if (a.window) lo = max(t.len - t.queries + tok + 1 - a.window, 0);
    }
    const uint64_t sees = __ballot(hi > lo);        // (a bit a lane: 36 sequences of 7 736 keys, 2 heads of 256, 152 us; by the bounds, kept in registers to the end, 155)
    u32x4_t qf[KF];
    {
        const unsigned char *src = a.q + static_cast<int64_t>(t.token0 + tok) * a.q_token + head * a.q_head;
#pragma unroll
        for (int i = 0; i < KF; ++i) {
            const int d = F8 ? 32 * (i >> 1) + 16 * lh + 8 * (i & 1) : 16 * i + 8 * lh;
            qf[i] = live ? *reinterpret_cast<const u32x4_t *>(src + 2 * d) : u32x4_t{0u, 0u, 0u, 0u};
        }
    }
    const int32_t *table = a.table + t.b * a.table_stride;
    const int page_mask = (1 << a.page_shift) - 1;
    const int last_key = t.hi - 1;
    const int ktok = token_of_row<F8>(lr);
    const int64_t page_bytes = (static_cast<int64_t>(D) << a.page_shift) * (F8 ? 1 : 2);

    // The pages of the wave's next 32 blocks, a lane for each 16 tokens (which lie in one page): a block's loads do not wait for the table.
    // What lies outside of the tile's keys is a place of the nearest page inside.
    auto pages_from = [&](int kb) -> int {
        const int at = (kb + WAVES * (lane >> 1)) * 32 + 16 * (lane & 1);
        return table[min(max(at, t.lo), last_key) >> a.page_shift];
    };
    int pages = 0, pages_next = 0;
    u32x4_t kreg[KL], vreg[KL];
    int kexp = 0;
    u32x4_t vexp = {0u, 0u, 0u, 0u};
    bool careful = false;                         // a page that does not exist, or a value that is not finite where not all rows see it
    // Page times heads, plus the head, of half a block; a page that does not exist is page 0.
    auto half_page = [&](int n, int half) -> int64_t {
        const int p = __builtin_amdgcn_readlane(pages, 2 * n + half);
        const bool bad = p < 0 || p >= a.num_pages;
        careful = careful || bad;
        return static_cast<int64_t>(bad ? 0 : p) * a.kv_heads + kv;
    };
    auto load_k = [&](int kb, int n) {            // n: the block's number in `pages`
        const int64_t ph0 = half_page(n, 0), ph1 = half_page(n, 1);
        const bool second = ktok >= 16;
        const int off = (kb * 32 + ktok) & page_mask;
        const unsigned char *src = (second ? a.kp + ph1 * page_bytes : a.kp + ph0 * page_bytes) + (static_cast<int64_t>(lh) << a.page_shift) * 16 + off * 16;
#pragma unroll
        for (int i = 0; i < KL; ++i) kreg[i] = *reinterpret_cast<const u32x4_t *>(src + (static_cast<int64_t>(2 * i) << a.page_shift) * 16);
        if (F8) kexp = (second ? a.ke + (ph1 << a.page_shift) : a.ke + (ph0 << a.page_shift))[off];
    };
    auto load_v = [&](int kb, int n) {
        const int64_t ph0 = half_page(n, 0), ph1 = half_page(n, 1);
        const int off0 = (kb * 32) & page_mask, off1 = (kb * 32 + 16) & page_mask;
        if constexpr (F8) {
            const int off = lh ? off1 : off0;
            const unsigned char *src = (lh ? a.vp + ph1 * page_bytes : a.vp + ph0 * page_bytes) + (off / W * D + lr) * 16;
#pragma unroll
            for (int i = 0; i < NB; ++i) vreg[i] = *reinterpret_cast<const u32x4_t *>(src + 32 * 16 * i);
            vexp = *reinterpret_cast<const u32x4_t *>((lh ? a.ve + (ph1 << a.page_shift) : a.ve + (ph0 << a.page_shift)) + off);
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const unsigned char *src = (s ? a.vp + ph1 * page_bytes : a.vp + ph0 * page_bytes) + (((s ? off1 : off0) / W + lh) * D + lr) * 16;
#pragma unroll
                for (int i = 0; i < NB; ++i) vreg[s * NB + i] = *reinterpret_cast<const u32x4_t *>(src + 32 * 16 * i);
            }
        }
    };

    float m = kNegInf, l = 0.0f;
    float16_t o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] = 0.0f;
    int kb = k0 + wave, n = 0;
    if (kb < k1) pages = pages_from(kb);
    if (kb + 32 * WAVES < k1) pages_next = pages_from(kb + 32 * WAVES);
    // The queries and pages have come, on every way to the loop: else the compiler waits for them in it, and with them for the values, which
    // are not needed before the softmax is done (1 to 3 % of steps; 256 dims, with one wave a SIMD, 232 -> 237 us: left as it was.  Loads
    // behind the last block too, so that the next keys stay on their way through the second product: nothing, and short steps 0.5 us more).
    if constexpr (D <= 128) {
#pragma unroll
        for (int i = 0; i < KF; ++i) asm volatile("" : "+v"(qf[i]));
        asm volatile("" : "+v"(pages), "+v"(pages_next));
    }
    if (kb < k1) {
        load_k(kb, 0);
        load_v(kb, 0);
    }
    for (; kb < k1; kb += WAVES) {
        float16_t s;
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 0.0f;
        const float kscale = power_of_two(kexp);
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            if constexpr (F8) {
                s = mfma(widen(kreg[i][0], kreg[i][1], kscale, T{}), qf[2 * i], s, T{});
                s = mfma(widen(kreg[i][2], kreg[i][3], kscale, T{}), qf[2 * i + 1], s, T{});
            } else {
                s = mfma(kreg[i], qf[i], s, T{});
            }
        }
        if (++n == 32) {
            n = 0;
            pages = pages_next;
            if (kb + 33 * WAVES < k1) pages_next = pages_from(kb + 33 * WAVES);
        }
        if (kb + WAVES < k1) load_k(kb + WAVES, n);
        const int base = kb * 32;
        const bool whole = __all(base >= lo && base + 32 <= hi);
        if (!whole) {
            bool odd = false;
            const Seen seen(lo, hi, base + half_token<F8>(lh));
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] = seen(reg_token<F8>(v)) ? s[v] : kNegInf;
            if constexpr (F8) {
#pragma unroll
                for (int i = 0; i < NB; ++i) keep_tokens<F8>(vreg[i], base + 16 * lh, t.lo, t.hi);
                if constexpr (kScaleValues<T, F8>) keep_tokens<F8>(vexp, base + 16 * lh, t.lo, t.hi);
            } else {
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) keep_tokens<F8>(vreg[i], base + 16 * (i / NB) + 8 * lh, t.lo, t.hi);
            }
#pragma unroll
            for (int i = 0; i < KL; ++i)
#pragma unroll
                for (int d = 0; d < 4; ++d) odd = odd || (F8 ? odd8(vreg[i][d]) : odd16<T>(vreg[i][d]));
            careful = careful || __any(odd);
        }
        float bm = s[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) bm = fmaxf(bm, s[v]);
        bm = fmaxf(bm, __shfl_xor(bm, 32));
        const float m_new = fmaxf(m, bm * a.c2);
        const float base2 = m_new == kNegInf ? 0.0f : m_new;         // (a row that has seen nothing yet)
        if (__any(m_new != m)) {
            const float alpha = __builtin_amdgcn_exp2f(m - base2);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[i][v] *= alpha;
            m = m_new;
        }
        const float shift = range.shift - base2;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], a.c2, shift));
            l += p;
            s[v] = F8 && !kScaleValues<T, F8> ? __builtin_amdgcn_ldexpf(p, exponent_of(vexp, v)) : p;
        }
        half2_t vscale[8];
        if constexpr (kScaleValues<T, F8>)
#pragma unroll
            for (int i = 0; i < 8; ++i) vscale[i] = scales_of(vexp[i >> 1], i & 1);
        u32x4_t pf[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) pf[i][e] = pack2(s[8 * i + 2 * e], s[8 * i + 2 * e + 1], T{});
        auto value = [&](int i, int j) {
            if constexpr (kScaleValues<T, F8>) return widen_each(vreg[j][2 * i], vreg[j][2 * i + 1], vscale + 4 * i);
            else if constexpr (F8) return widen(vreg[j][2 * i], vreg[j][2 * i + 1], range.value_scale, T{});
            else return vreg[i * NB + j];
        };
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) o[j] = mfma(value(i, j), pf[i], o[j], T{});
        if (kb + WAVES < k1) load_v(kb + WAVES, n);
    }
    l += __shfl_xor(l, 32);
    if (WAVES == 1 ? careful : __syncthreads_or(careful) != 0) {
        careful_tile<T, F8, D, 32, 5, WAVES>(a, range, t, kv, wave, lane);
        return;
    }

    m = row_maximum(m, (sees >> lane) & 1);
    if constexpr (WAVES == 1) {
        if (live) store_rows<T, D>(a, range.back, t, kv, row, lh, m, l, o);
        return;
    } else {
        // ---- the waves' maxima, sums and outputs ----
        constexpr int PITCH = D + 4;
        extern __shared__ __attribute__((aligned(16))) float joined[];       // [WAVES][32][PITCH]
        __shared__ float wave_m[WAVES][32], wave_l[WAVES][32];
        if (lh == 0) wave_m[wave][lr] = m, wave_l[wave][lr] = l;
        float *mine = joined + (wave * 32 + lr) * PITCH;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (!live) break;
                const float4_t w = {o[j][4 * r], o[j][4 * r + 1], o[j][4 * r + 2], o[j][4 * r + 3]};
                *reinterpret_cast<float4_t *>(mine + 32 * j + 8 * r + 4 * lh) = w;
            }
        __syncthreads();
        // 2 WAVES threads a row, pairs of dims
        const int r = tid / (2 * WAVES), part = tid % (2 * WAVES), rr = t.row0 + r;
        if (rr >= t.rows) return;
        float mm = wave_m[0][r];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, wave_m[w][r]);
        const float base2 = mm == kNegInf ? 0.0f : mm;
        float f[WAVES], total = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            f[w] = __builtin_amdgcn_exp2f(wave_m[w][r] - base2);
            total = __builtin_fmaf(wave_l[w][r], f[w], total);
        }
        const int rtok = a.by_group(rr), rhead = kv * a.group + rr - rtok * a.group;
        const int64_t token = static_cast<int64_t>(t.token0) + rtok;
        const bool alone = t.parts == 1;
        const float inv = alone ? (mm == kNegInf ? 0.0f : range.back / total) : 1.0f;
        const int64_t at = part_row<32>(a, t, kv, t.part, r);
        float *po = alone ? nullptr : a.part_o + at * D;
        unsigned char *dst = a.out + token * a.out_token + rhead * a.out_head;
#pragma unroll
        for (int i = 0; i < (D + 4 * WAVES - 1) / (4 * WAVES); ++i) {
            const int d = 4 * WAVES * i + 2 * part;
            if (D % (4 * WAVES) != 0 && d >= D) break;
            float y[2] = {0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float *src = joined + (w * 32 + r) * PITCH + d;
                y[0] = __builtin_fmaf(src[0], f[w], y[0]);
                y[1] = __builtin_fmaf(src[1], f[w], y[1]);
            }
            if (alone) *reinterpret_cast<uint32_t *>(dst + 2 * d) = pack2(y[0] * inv, y[1] * inv, T{});
            else *reinterpret_cast<float2 *>(po + d) = make_float2(y[0], y[1]);
        }
        if (part == 0) say_parts<32>(a, t, kv, r, token * a.q_heads + rhead, mm, total);
    }
}

// ---- many rows: a workgroup has kTileRows rows, 32 to a wave, and its waves share the keys: blocks of 64, two in LDS in turn, loaded there
// directly (a page's pieces are already in the operands' order) while the other one is multiplied ----
//
// 128 rows read a block from L2 once for four waves, 64 KB of LDS (128 dims) leave two workgroups a compute unit, and 256 registers a wave
// hold the queries, 64 keys' scores and the outputs: hence exactly two waves a SIMD (`amdgpu_waves_per_eu`; told "two at least" the
// compiler spilled to reach three).  Beside the products and the softmax a block's addresses count (at 64 dims as many instructions as
// either): a lane holds the place of one of the next 64 blocks, or of one of 16 tokens of the next 16, and a wave's loads share an
// address.  256 rows and eight waves: 269 us against 249 for the chunk of 2 048 tokens; the next block's scores
// begun before this one's softmax 266 against 259; row sums by dot products 256 against 249; three waves with one buffer each for
// keys and values: spills; the next block's loads behind the scores' products, or `s_setprio` around those: within 1 %.
constexpr int kTileRows = 128;

// 64 lanes' 16 bytes to LDS, lane by lane, N times: load i to the 1 KB from lds + 1024 i on, from 1024 i bytes behind its address (a
// load's constant offset counts for both).  One statement each, because of m0.  (The compiler does not count these loads: every wait for
// them is written out, and what it waits for itself can only be too much.)
#define LOAD(i, a, at) "\n\tglobal_load_lds_dwordx4 %" #i ", " a " offset:" #at
template <int N>
__device__ __forceinline__ void to_lds(const unsigned char *const (&p)[N], uint32_t lds)
{
    const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
    static_assert(N >= 1 && N <= 4, "");
    if constexpr (N == 1) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" LOAD(1, "off", 0) ::"s"(m), "v"(p[0]) : "memory", "m0");
    if constexpr (N == 2) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" LOAD(1, "off", 0) LOAD(2, "off", 0x400) ::"s"(m), "v"(p[0]), "v"(p[1]) : "memory", "m0");
    if constexpr (N == 3) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" LOAD(1, "off", 0) LOAD(2, "off", 0x400) LOAD(3, "off", 0x800) ::"s"(m), "v"(p[0]), "v"(p[1]), "v"(p[2]) : "memory", "m0");
    if constexpr (N == 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" LOAD(1, "off", 0) LOAD(2, "off", 0x400) LOAD(3, "off", 0x800) LOAD(4, "off", 0xc00) ::"s"(m), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void to_lds(const unsigned char *base, const uint32_t (&o)[N], uint32_t lds)      // base: the same in all lanes
{
    // (one value for all lanes already; said again, or the compiler may hold it in a vector register)
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const uint64_t b = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at))) |
                       static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32)))) << 32;
    const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
    static_assert(N >= 1 && N <= 4, "");
    if constexpr (N == 1) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" LOAD(2, "%1", 0) ::"s"(m), "s"(b), "v"(o[0]) : "memory", "m0");
    if constexpr (N == 2) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" LOAD(2, "%1", 0) LOAD(3, "%1", 0x400) ::"s"(m), "s"(b), "v"(o[0]), "v"(o[1]) : "memory", "m0");
    if constexpr (N == 3) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" LOAD(2, "%1", 0) LOAD(3, "%1", 0x400) LOAD(4, "%1", 0x800) ::"s"(m), "s"(b), "v"(o[0]), "v"(o[1]), "v"(o[2]) : "memory", "m0");
    if constexpr (N == 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" LOAD(2, "%1", 0) LOAD(3, "%1", 0x400) LOAD(4, "%1", 0x800) LOAD(5, "%1", 0xc00) ::"s"(m), "s"(b), "v"(o[0]), "v"(o[1]), "v"(o[2]), "v"(o[3]) : "memory", "m0");
}
#undef LOAD
// 64 lanes' 4 bytes to 256 bytes of LDS.
__device__ __forceinline__ void dword_to_lds(const void *src, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory", "m0");
}
// The larger of a lane's value and lane ^ 32's.
__device__ __forceinline__ float max_halves(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t lo = r[0], hi = r[1];
    return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

// A block's keys, its values, and (FP8) the exponents of both.  Two of them: three or four on their way changed no time by more than 2 %,
// the next one's loads take less than a block's products.
template <bool F8, int D>
struct Block {
    static constexpr int HALF = 64 * D * (F8 ? 1 : 2);             // bytes of a block's keys, and of its values
    static constexpr int SIZE = 2 * HALF + (F8 ? 256 : 0);
};
// Waves a SIMD that the compiler makes registers last for.  Up to 64 dims four, where that spills nothing (64 sequences of up to 512 new tokens
// and 4 096 keys, 16 heads: 64 dims 237 -> 221 us, 32 dims 186 -> 166, FP8 257 -> 222; FP8 pages of 64 dims would spill, 37.7 -> 38.6 us with
// a window of 1 000).
template <bool F8, int D> constexpr int kTileWaves = D <= 32 || (D <= 64 && !F8) ? 4 : D <= 128 ? 2 : 1;

template <typename T, bool F8, int D, bool ONE_PAGE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kTileWaves<F8, D>, kTileWaves<F8, D>)))
paged_tile_kernel(const PagedArgs a)
{
    constexpr int KF = D / 16, NB = D / 32, W = F8 ? 16 : 8, SZ = F8 ? 1 : 2;
    constexpr int HALF = Block<F8, D>::HALF, SIZE = Block<F8, D>::SIZE;
    constexpr int LOADS = HALF / 1024;             // 1 KB loads of each half
    constexpr int MINE = (LOADS + 3) / 4;          // a wave's (some are loaded twice where they do not divide)
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];      // [2][keys, values, exponents]
    __shared__ half2_t scales[kScaleValues<T, F8> ? 4 : 1][32];                 // each wave's, of a block's values
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lr = lane & 31, lh = lane >> 5;
    half2_t *wave_scales = scales[kScaleValues<T, F8> ? wave : 0];
    const int place = a.by_kv_heads(blockIdx.x), kv = blockIdx.x - place * a.kv_heads;
    const Factors<T, F8> range(a);
    Item t;
    if (!find_item<kTileRows, 6>(a, place, lane, t)) return;
    const int k0 = t.k0, k1 = t.k1;

    // ---- this lane's row, and the keys that the wave's rows see ----
    const int row = t.row0 + 32 * wave + lr;
    const bool live = row < t.rows;
    const int tok = live ? a.by_group(row) : 0, gh = live ? row - tok * a.group : 0;
    const int head = kv * a.group + gh;
    int lo = t.lo, hi = t.hi, wave_lo = t.lo, wave_hi = t.hi;
    int tile_lo = t.lo, tile_hi = t.hi;                       // keys that all rows of the tile see
    if (a.causal) {
        tile_hi = min(max(t.len - t.queries + a.by_group(t.row0) + 1, 0), t.len);
        if (a.window) tile_lo = max(t.len - t.queries + a.by_group(min(t.row0 + kTileRows, t.rows) - 1) + 1 - a.window, 0);
        const int first = a.by_group(t.row0 + 32 * wave), last = a.by_group(max(min(t.row0 + 32 * wave + 32, t.rows) - 1, 0));
        wave_hi = min(max(t.len - t.queries + last + 1, 0), t.len);
        if (a.window) wave_lo = max(t.len - t.queries + first + 1 - a.window, 0);
        if (live) {
            hi = min(max(t.len - t.queries + tok + 1, 0), t.len);
            if (a.window) lo = max(t.len - t.queries + tok + 1 - a.window, 0);
        }
    }
    if (t.row0 + 32 * wave >= t.rows) wave_hi = 0;                    // no rows: the wave only loads
    u32x4_t qf[KF];
    {
        const unsigned char *src = a.q + static_cast<int64_t>(t.token0 + tok) * a.q_token + head * a.q_head;
#pragma unroll
        for (int i = 0; i < KF; ++i) {
            const int d = F8 ? 32 * (i >> 1) + 16 * lh + 8 * (i & 1) : 16 * i + 8 * lh;
            qf[i] = live ? *reinterpret_cast<const u32x4_t *>(src + 2 * d) : u32x4_t{0u, 0u, 0u, 0u};
        }
    }
    const int32_t *table = a.table + t.b * a.table_stride;
    const int page_mask = (1 << a.page_shift) - 1;
    const int last_key = t.hi - 1;
    const int ktok = token_of_row<F8>(lr);
    const int64_t page_bytes = (static_cast<int64_t>(D) << a.page_shift) * SZ;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char *)smem)));
    constexpr bool one_page = ONE_PAGE;           // a block lies in one page (of 64 tokens or more)

    // Where the next blocks lie, a lane each (64 blocks), or a lane for each 16 tokens, which lie in one page (16 blocks): their pages as
    // they come from the table, and the first slot of page and head, once a page has come.
    constexpr int AHEAD = one_page ? 64 : 16;
    bool careful = false;                         // a page that does not exist, or a value that is not finite where not all rows see it
    auto pages_from = [&](int kb) -> int { return table[min(max(kb * 64 + lane * (one_page ? 64 : 16), t.lo), last_key) >> a.page_shift]; };
    int pages_next = 0, at_page = 0;
    uint32_t slot_lo = 0, slot_hi = 0;
    auto take_pages = [&](int pages) {
        const bool bad = pages < 0 || pages >= a.num_pages;
        careful = careful || __any(bad);
        const int64_t slot = (static_cast<int64_t>(bad ? 0 : pages) * a.kv_heads + kv) << a.page_shift;
        slot_lo = static_cast<uint32_t>(slot), slot_hi = static_cast<uint32_t>(slot >> 32);
    };
    auto slot_at = [&](int i) -> int64_t {         // of lane i, for all
        return static_cast<uint32_t>(__builtin_amdgcn_readlane(slot_lo, i)) | static_cast<int64_t>(__builtin_amdgcn_readlane(slot_hi, i)) << 32;
    };
    auto slot_of = [&](int i) -> int64_t {         // of each lane's i
        return static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * i, slot_lo)) | static_cast<int64_t>(__builtin_amdgcn_ds_bpermute(4 * i, slot_hi)) << 32;
    };
    // A wave's loads of keys and values: MINE from n0 on, in groups of up to four.
    constexpr int GROUP = MINE < 4 ? MINE : 4;
    static_assert(MINE % GROUP == 0, "");
    const int n0 = min(wave * MINE, LOADS - MINE);
    const int piece = 16 << a.page_shift;          // bytes from one piece of a token's keys to the next
    // A block's loads; blocks are asked for in their order.
    auto issue = [&](int kb, int buffer) {
        const uint32_t kl = lds0 + buffer * SIZE, vl = kl + HALF;
        if constexpr (one_page) {
            const int off = (kb * 64) & page_mask;
            const int64_t slot = slot_at(at_page);
            const unsigned char *ks = a.kp + slot * (D * SZ) + off * 16, *vs = a.vp + (slot + off) * (D * SZ);
#pragma unroll
            for (int g = 0; g < MINE; g += GROUP) {
                uint32_t ko[GROUP], vo[GROUP];
#pragma unroll
                for (int i = 0; i < GROUP; ++i) ko[i] = lane * 16 + (n0 + g + i) * piece - 1024 * i, vo[i] = lane * 16 + (n0 + g) * 1024;
                to_lds(ks, ko, kl + (n0 + g) * 1024);
                to_lds(vs, vo, vl + (n0 + g) * 1024);
            }
            if constexpr (F8) dword_to_lds(((lane & 16) ? a.ve : a.ke) + slot + off + 4 * (lane & 15), vl + HALF);
        } else {
            auto place = [&](int token) -> int { return (kb * 64 + token) & page_mask; };
            const unsigned char *ks = a.kp + slot_of(4 * at_page + (lane >> 4)) * (D * SZ) + place(lane) * 16;
#pragma unroll
            for (int g = 0; g < MINE; g += GROUP) {
                const unsigned char *kq[GROUP];
#pragma unroll
                for (int i = 0; i < GROUP; ++i) kq[i] = ks + ((n0 + g + i) * piece - 1024 * i);
                to_lds(kq, kl + (n0 + g) * 1024);
            }
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int n = n0 + i;
                if constexpr (D % 64 == 0) {                         // the pieces of a load: one run of tokens
                    const int token = n * 64 / D * W;
                    const uint32_t o[1] = {static_cast<uint32_t>(lane * 16)};
                    to_lds(a.vp + slot_at(4 * at_page + (token >> 4)) * (D * SZ) + (place(token) / W * D + n * 64 % D) * 16, o, vl + n * 1024);
                } else {
                    const int e = n * 64 + lane, token = e / D * W;
                    const unsigned char *p[1] = {a.vp + slot_of(4 * at_page + (token >> 4)) * (D * SZ) + (place(token) / W * D + e % D) * 16};
                    to_lds(p, vl + n * 1024);
                }
            }
            if constexpr (F8) {
                const int token = 4 * (lane & 15);
                dword_to_lds(((lane & 16) ? a.ve : a.ke) + slot_of(4 * at_page + (token >> 4)) + place(token), vl + HALF);
            }
        }
        if (++at_page == AHEAD) {
            at_page = 0;
            take_pages(pages_next);
            if (kb + 1 + AHEAD < k1) pages_next = pages_from(kb + 1 + AHEAD);
        }
    };

    float m = kNegInf, l = 0.0f;
    float16_t o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] = 0.0f;
    int pages = 0;
    if (k0 < k1) pages = pages_from(k0);
    if (k0 + AHEAD < k1) pages_next = pages_from(k0 + AHEAD);
    // (The queries and pages have come, on every way to the loop: else the compiler waits for them in it, and with them for all that is on
    // its way.)
#pragma unroll
    for (int i = 0; i < KF; ++i) asm volatile("" : "+v"(qf[i]));
    asm volatile("" : "+v"(pages), "+v"(pages_next));
    if (k0 < k1) {
        take_pages(pages);
        issue(k0, 0);
    }
    for (int kb = k0; kb < k1; ++kb) {
        // The block has landed, for this wave and after the barrier for all; everyone is done with the block before it.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int buffer = (kb - k0) & 1;
        const unsigned char *block = smem + buffer * SIZE;
        if (kb + 1 < k1) issue(kb + 1, buffer ^ 1);
        float kscale[2];
        u32x4_t vexp[2];
        if constexpr (F8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                kscale[h] = power_of_two(static_cast<int8_t>(block[2 * HALF + 32 * h + ktok]));
                if constexpr (!kScaleValues<T, F8>) vexp[h] = *reinterpret_cast<const u32x4_t *>(block + 2 * HALF + 64 + 32 * h + 16 * lh);
            }
        }
        const int base = kb * 64;
        if (base < tile_lo || base + 64 > tile_hi) {
            // A block that not every row of the tile sees whole: what lies outside of the tile's keys becomes zero.
            unsigned char *vb = const_cast<unsigned char *>(block) + HALF;
            bool odd = false;
            for (int e = tid; e < LOADS * 64; e += 256) {
                u32x4_t *at = reinterpret_cast<u32x4_t *>(vb + e * 16);
                u32x4_t w = *at;
                keep_tokens<F8>(w, base + e / D * W, t.lo, t.hi);
#pragma unroll
                for (int d = 0; d < 4; ++d) odd = odd || (F8 ? odd8(w[d]) : odd16<T>(w[d]));
                *at = w;
            }
            if (__syncthreads_or(odd)) {
                careful = true;
                break;
            }
        }
        if (careful) break;                       // (the same in all waves)
        if (base >= wave_hi || base + 64 <= wave_lo) continue;
        if constexpr (kScaleValues<T, F8>) {
            // A lane a pair of tokens, for all lanes of the wave: each lane for its own 32 took 41.8 us in place of 37.5 (ragged chunks, 64 dims,
            // a window of 1 000 keys), conversions of one value at a time with its own scale 49.6.
            // (What lies outside of the tile's keys, where an exponent may be anything: zero times zero.)
            const int first = base + 2 * lr;
            half2_t two = scales_of(*reinterpret_cast<const uint16_t *>(block + 2 * HALF + 64 + 2 * lr), false);
#pragma unroll
            for (int i = 0; i < 2; ++i) two[i] = first + i >= t.lo && first + i < t.hi ? two[i] : static_cast<_Float16>(0.0f);
            if (lh == 0) wave_scales[lr] = two;
            __builtin_amdgcn_wave_barrier();          // (the wave's own, and its LDS accesses keep their order)
        }
        const unsigned char *kt = block + (lh * 64 + ktok) * 16;
        const unsigned char *vt = block + HALF + lr * 16;
        float16_t s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int v = 0; v < 16; ++v) s[h][v] = 0.0f;
#pragma unroll
            for (int i = 0; i < LOADS / 2; ++i) {            // pieces 2 i + lh
                const u32x4_t k = *reinterpret_cast<const u32x4_t *>(kt + (2 * i * 64 + 32 * h) * 16);
                if constexpr (F8) {
                    s[h] = mfma(widen(k[0], k[1], kscale[h], T{}), qf[2 * i], s[h], T{});
                    s[h] = mfma(widen(k[2], k[3], kscale[h], T{}), qf[2 * i + 1], s[h], T{});
                } else {
                    s[h] = mfma(k, qf[i], s[h], T{});
                }
            }
        }
        const bool whole = __all(base >= lo && base + 64 <= hi);
        if (!whole) {
            const Seen seen(lo, hi, base + half_token<F8>(lh));
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int v = 0; v < 16; ++v) s[h][v] = seen(32 * h + reg_token<F8>(v)) ? s[h][v] : kNegInf;
        }
        float bm = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int v = 1; v < 16; ++v) bm = fmaxf(fmaxf(s[0][v], s[1][v]), bm);
        // The reference is left where it is while no score is more than kSlack above it: probabilities are relative, and `shift` leaves room for
        // 2^kSlack in theirs, their sums' and their products' types.
        if (__any(bm * a.c2 > m + static_cast<float>(kSlack))) {
            const float m_new = fmaxf(m, max_halves(bm) * a.c2);
            const float alpha = m_new == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[i][v] *= alpha;
            m = m_new;
        }
        const float shift = range.shift - (m == kNegInf ? 0.0f : m);       // (a row that has seen nothing yet)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4_t pf[2];
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][v], a.c2, shift));
                l += p;
                s[h][v] = F8 && !kScaleValues<T, F8> ? __builtin_amdgcn_ldexpf(p, exponent_of(vexp[h], v)) : p;
            }
            half2_t vscale[8];
            if constexpr (kScaleValues<T, F8>)
#pragma unroll
                for (int i = 0; i < 8; ++i) vscale[i] = wave_scales[16 * h + 8 * lh + i];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) pf[i][e] = pack2(s[h][8 * i + 2 * e], s[h][8 * i + 2 * e + 1], T{});
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if constexpr (F8) {
                    const u32x4_t w = *reinterpret_cast<const u32x4_t *>(vt + ((2 * h + lh) * D + 32 * j) * 16);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        u32x4_t v;
                        if constexpr (kScaleValues<T, F8>) v = widen_each(w[2 * i], w[2 * i + 1], vscale + 4 * i);
                        else v = widen(w[2 * i], w[2 * i + 1], range.value_scale, T{});
                        o[j] = mfma(v, pf[i], o[j], T{});
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        o[j] = mfma(*reinterpret_cast<const u32x4_t *>(vt + ((4 * h + 2 * i + lh) * D + 32 * j) * 16), pf[i], o[j], T{});
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (careful) {
        careful_tile<T, F8, D, kTileRows, 6, 4>(a, range, t, kv, wave, lane);
        return;
    }
    l += __shfl_xor(l, 32);
    if (live) store_rows<T, D, kTileRows>(a, range.back, t, kv, row, lh, row_maximum(m, hi > lo), l, o);
}

// ---- the parts of a row, joined: a workgroup has a row, groups of D / 4 threads take the parts in turn and are added in their order (the
// same bits every time; no atomics).  5 us, most of it the launch and one round trip: worth it from 2 048 keys on ----
template <typename T, int D, int TILE>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedArgs a)
{
    constexpr int PER = D / 4, GROUPS = 256 / PER;               // threads to a part; parts at a time (D = 96: 10, 16 threads idle)
    __shared__ float4_t sums[GROUPS][PER];
    __shared__ float totals[GROUPS];
    const int64_t at = blockIdx.x;
    const int token = a.by_q_heads(blockIdx.x);
    if (token < offset_of(a, 0) || token >= offset_of(a, a.sequences)) return;      // (nothing was written for it)
    const int n = a.part_at[at].y;
    const int64_t first = a.part_at[at].x, step = static_cast<int64_t>(a.kv_heads) * TILE;
    if (n <= 0 || first < 0 || first + (n - 1) * step >= a.part_rows) return;
    const int group = threadIdx.x / PER, d = threadIdx.x % PER;
    float mm = kNegInf;
    for (int p = threadIdx.x & 63; p < n; p += 64) mm = fmaxf(mm, a.part_ml[first + p * step].x);
#pragma unroll
    for (int o = 32; o; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
    const float base2 = mm == kNegInf ? 0.0f : mm;
    if (group < GROUPS) {
        float total = 0.0f;
        float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int p = group; p < n; p += GROUPS) {
            const float2 ml = a.part_ml[first + p * step];
            const float f = __builtin_amdgcn_exp2f(ml.x - base2);
            const float4_t o = *reinterpret_cast<const float4_t *>(a.part_o + (first + p * step) * D + 4 * d);
            total = __builtin_fmaf(ml.y, f, total);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(o[i], f, sum[i]);
        }
        sums[group][d] = sum;
        if (d == 0) totals[group] = total;
    }
    __syncthreads();
    if (threadIdx.x >= PER) return;
    float total = totals[0];
    float4_t sum = sums[0][d];
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) {
        total += totals[g];
        const float4_t o = sums[g][d];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += o[i];
    }
    const float inv = mm == kNegInf ? 0.0f : a.back / total;
    const int head = static_cast<int>(at - token * a.q_heads);
    u32x2_t w;
    w[0] = pack2(sum[0] * inv, sum[1] * inv, T{});
    w[1] = pack2(sum[2] * inv, sum[3] * inv, T{});
    *reinterpret_cast<u32x2_t *>(a.out + token * a.out_token + head * a.out_head + 8 * d) = w;
}

// ---- host ----
struct Plan {
    bool tile;           // the kernel of many rows
    int waves;           // of a workgroup of the other one
    int64_t items;       // bound, for each key head
    int slots, min_blocks;
    int64_t rows;        // of parts, bound
    int64_t o_bytes, ml_bytes, at_bytes;
};
Plan plan_of(const arcq_attention_paged_args *p)
{
    Plan r{};
    const int64_t heads = p->pages.heads, group = p->q_heads / heads, cus = device_cus();
    const int64_t most = p->table_width * p->pages.page_size;
    // Many rows: more than 64 a sequence (8 sequences of 4 000 keys, 8 heads of 128: 64 rows 38.2 us and 39.1 with 128 a workgroup, 96 rows
    // 56.3 and 42.0, 256 rows 88.2 and 67.4), but for few keys while the chip takes the tiles of 32 about at once (600 keys, 96 rows 13.2
    // and 22.2, 256 rows 17.5 and 23.2; 64 sequences of 1 000 keys, 96 rows 77.6 and 58.6).
    const int64_t tiles32 = p->tokens * group / 32 + p->sequences;            // (a ragged end for every sequence)
    r.tile = p->tokens * group > 64 * p->sequences && (most >= 2048 || tiles32 * heads > 3 * cus);
    const int rows = r.tile ? kTileRows : 32;
    const int64_t tiles = r.tile ? p->tokens * group / rows + p->sequences : tiles32;
    const int64_t window = std::min<int64_t>(p->window, 1 << 30);
    const int64_t keys = p->causal && window ? std::min<int64_t>(most, window + rows / group + 64) : most;           // of a tile
    const int64_t wide = p->pages.head_dim > 128 ? 1 : 2;                    // waves a SIMD has registers for
    int64_t slots, least;                                                    // in workgroups; keys of a part
    if (r.tile) {
        r.waves = 4;
        slots = 2 * tiles * heads > wide * cus ? 0 : wide * cus;
        least = 512;
    } else {
        // Few tiles: eight waves each (1 sequence of 6 heads and 1 000 keys 11.5 -> 10.0 us, 8 of 8 heads and 1 024 15.4 -> 13.3, 16 of them
        // 16.1 and 15.8, the 64 images of 6 heads and 197 keys 10.6 -> 15.8).  Few keys and many tiles: a wave each (256 sequences of
        // up to 512 keys, 8 heads: 62 us, with four waves 72); one or two blocks of keys: nothing to share.
        r.waves = keys <= (wide == 1 ? 256 : 64) || (keys < 1024 && tiles * heads >= 3 * wide * cus) ? 1 : 2 * tiles * heads <= cus && wide == 2 ? 8 : 4;
        // Parts: as many as the chip takes at once, or (many tiles, whose lengths differ) half as many again.  64 sequences of up to 8 192
        // keys, 8 key heads, 1, 1.5, 2 times: 199, 190, 193 us; 2 of 130 000 with FP8 pages 103, 123, 112; 16 of 4 096 55.5, 63.7, 59.9.
        slots = wide * cus * 4 / r.waves;
        if (r.waves == 4 && 2 * tiles * heads > slots) slots += slots / 2;
        least = r.waves == 8 ? 512 : 256;
    }
    const int64_t shift = r.tile ? 6 : 5;
    r.min_blocks = static_cast<int>(least >> shift);
    slots = std::min<int64_t>(slots / heads, tiles * (keys / least));
    // (from 2 048 keys on: a second launch joins the parts; 16 sequences of 1 024 keys 16.1 us in one part, 20.1 in more.  From 2^24 rows on
    // the tiles alone are many, and the join, a workgroup a row, would be more than a grid's axis holds.)
    r.slots = keys < 2048 || r.waves == 1 || p->tokens * p->q_heads >= (1 << 24) ? 0 : static_cast<int>(std::max<int64_t>(0, slots));
    r.items = tiles + r.slots;
    if (r.slots) {
        r.rows = r.items * heads * rows;
        r.o_bytes = r.rows * p->pages.head_dim * 4;
        r.ml_bytes = r.rows * 8;
        r.at_bytes = p->tokens * p->q_heads * 8;
    }
    return r;
}

template <typename T, bool F8, int D>
void launch_paged(const PagedArgs &a, const Plan &plan, hipStream_t st)
{
    const dim3 grid(static_cast<uint32_t>(plan.items * a.kv_heads));
    const dim3 join(static_cast<uint32_t>(a.tokens * a.q_heads));
    if (plan.tile) {
        constexpr int lds = 2 * Block<F8, D>::SIZE;
        if (a.page_shift >= 6) {
            if (lds > 65536) allow_dynamic_lds<paged_tile_kernel<T, F8, D, true>>(lds);
            hipLaunchKernelGGL((paged_tile_kernel<T, F8, D, true>), grid, dim3(256), lds, st, a);
        } else {
            if (lds > 65536) allow_dynamic_lds<paged_tile_kernel<T, F8, D, false>>(lds);
            hipLaunchKernelGGL((paged_tile_kernel<T, F8, D, false>), grid, dim3(256), lds, st, a);
        }
        if (plan.slots) hipLaunchKernelGGL((paged_join_kernel<T, D, kTileRows>), join, dim3(256), 0, st, a);
        return;
    }
    if (plan.waves == 1) {
        hipLaunchKernelGGL((paged_rows_kernel<T, F8, D, 1>), grid, dim3(64), 0, st, a);
    } else if (D <= 128 && plan.waves == 8) {
        constexpr int W = D <= 128 ? 8 : 4;                     // (256: its waves' outputs do not fit LDS)
        constexpr int lds = W * 32 * (D + 4) * 4;
        if (lds > 65536) allow_dynamic_lds<paged_rows_kernel<T, F8, D, W>>(lds);
        hipLaunchKernelGGL((paged_rows_kernel<T, F8, D, W>), grid, dim3(64 * W), lds, st, a);
    } else {
        constexpr int lds = 4 * 32 * (D + 4) * 4;
        if (lds > 65536) allow_dynamic_lds<paged_rows_kernel<T, F8, D, 4>>(lds);
        hipLaunchKernelGGL((paged_rows_kernel<T, F8, D, 4>), grid, dim3(256), lds, st, a);
    }
    if (plan.slots) hipLaunchKernelGGL((paged_join_kernel<T, D, 32>), join, dim3(256), 0, st, a);
}
template <typename T, bool F8>
void launch_paged_dim(const PagedArgs &a, const Plan &plan, int64_t dim, hipStream_t st)
{
    switch (dim) {
    case 32: launch_paged<T, F8, 32>(a, plan, st); break;
    case 64: launch_paged<T, F8, 64>(a, plan, st); break;
    case 96: launch_paged<T, F8, 96>(a, plan, st); break;
    case 128: launch_paged<T, F8, 128>(a, plan, st); break;
    default: launch_paged<T, F8, 256>(a, plan, st); break;
    }
}

// ARCQ_OK, or what is wrong with the sizes.
int check_sizes(const char *fn, const arcq_attention_paged_args *p)
{
    if (!p) return fail(ARCQ_ERR_NULL, "%s: NULL arguments", fn);
    if (const int rc = check_pages(fn, p->pages, p->dtype)) return rc;
    const int64_t d = p->pages.head_dim;
    if (d != 32 && d != 64 && d != 96 && d != 128 && d != 256)
        return fail(ARCQ_ERR_UNSUPPORTED, "%s: head_dim must be 32, 64, 96, 128 or 256 (got %lld)", fn, static_cast<long long>(d));
    if (p->tokens < 0 || p->q_heads < 0 || p->sequences < 0 || p->table_width < 0 || p->window < 0) return fail(ARCQ_ERR_SHAPE, "%s: negative size", fn);
    if (p->pages.heads < 1 || p->q_heads < 1 || p->q_heads % p->pages.heads != 0)
        return fail(ARCQ_ERR_SHAPE, "%s: %lld query heads do not divide by %lld key heads", fn, static_cast<long long>(p->q_heads), static_cast<long long>(p->pages.heads));
    if (p->window > 0 && !p->causal) return fail(ARCQ_ERR_UNSUPPORTED, "%s: a window needs causal", fn);
    if (!(p->scale > 0.0f) || !(p->scale < __builtin_inff())) return fail(ARCQ_ERR_UNSUPPORTED, "%s: scale must be positive", fn);
    if (p->table_width >= (int64_t(1) << 30) || p->table_width * p->pages.page_size >= (int64_t(1) << 30) || p->tokens >= (int64_t(1) << 30) ||
        p->q_heads > 65535 || p->tokens * p->q_heads >= (int64_t(1) << 30) || p->sequences >= (int64_t(1) << 24))
        return fail(ARCQ_ERR_SHAPE, "%s: tensor too large", fn);
    // (a grid's axis holds fewer than 2^32 threads; rows of parts: 32 bits)
    const Plan plan = plan_of(p);
    if (plan.items * p->pages.heads * 64 * plan.waves >= (int64_t(1) << 32) || plan.rows >= (int64_t(1) << 31))
        return fail(ARCQ_ERR_SHAPE, "%s: too many sequences", fn);
    return ARCQ_OK;
}

}  // namespace
}  // namespace arcq

using namespace arcq;

ARCQ_API int64_t arcq_attention_paged_workspace(const arcq_attention_paged_args *p)
{
    if (const int rc = check_sizes("arcq_attention_paged_workspace", p)) return rc;
    if (p->tokens == 0 || p->sequences == 0) return 0;
    const Plan plan = plan_of(p);
    return plan.o_bytes + plan.ml_bytes + plan.at_bytes;
}

ARCQ_API int arcq_attention_paged_fwd(const arcq_attention_paged_args *p, void *stream)
{
    const char *fn = "arcq_attention_paged_fwd";
    if (const int rc = check_sizes(fn, p)) return rc;
    if (p->tokens == 0 || p->sequences == 0) return ARCQ_OK;
    if (!p->q || !p->out || !p->q_offsets || !p->kv_lengths || (p->table_width && !p->page_table)) return fail(ARCQ_ERR_NULL, "%s: NULL tensor pointer", fn);
    if (const int rc = check_page_pointers(fn, p->pages)) return rc;
    if (p->pages.num_pages == 0 && p->table_width) return fail(ARCQ_ERR_SHAPE, "%s: a page table without pages", fn);
    if (!rows_aligned(p->q, p->tokens, p->q_token_stride, p->q_heads, p->q_head_stride) ||
        !rows_aligned(p->out, p->tokens, p->out_token_stride, p->q_heads, p->out_head_stride))
        return fail(ARCQ_ERR_ALIGN, "%s: every row of q and out must be 16-byte aligned", fn);
    const Plan plan = plan_of(p);
    if (plan.slots && (!p->workspace || !aligned(p->workspace, 16))) return fail(ARCQ_ERR_NULL, "%s: workspace missing or not 16-byte aligned", fn);
    PagedArgs a{};
    a.kp = static_cast<const unsigned char *>(p->pages.k), a.vp = static_cast<const unsigned char *>(p->pages.v);
    a.ke = p->pages.k_exponents, a.ve = p->pages.v_exponents;
    a.q = static_cast<const unsigned char *>(p->q), a.out = static_cast<unsigned char *>(p->out);
    a.table = p->page_table, a.q_offsets = p->q_offsets, a.kv_lengths = p->kv_lengths;
    if (plan.slots) {
        unsigned char *w = static_cast<unsigned char *>(p->workspace);
        a.part_o = reinterpret_cast<float *>(w);
        a.part_ml = reinterpret_cast<float2 *>(w + plan.o_bytes);
        a.part_at = reinterpret_cast<int2 *>(w + plan.o_bytes + plan.ml_bytes);
        a.part_rows = plan.rows;
    }
    a.q_token = 2 * p->q_token_stride, a.q_head = 2 * p->q_head_stride, a.out_token = 2 * p->out_token_stride, a.out_head = 2 * p->out_head_stride;
    a.table_stride = p->table_stride, a.tokens = p->tokens, a.table_width = p->table_width, a.num_pages = p->pages.num_pages;
    a.q_heads = static_cast<int>(p->q_heads), a.kv_heads = static_cast<int>(p->pages.heads), a.group = a.q_heads / a.kv_heads;
    a.sequences = static_cast<int>(p->sequences), a.page_shift = log2_of(p->pages.page_size);
    a.window = static_cast<int>(std::min<int64_t>(p->window, 1 << 30)), a.causal = p->causal ? 1 : 0, a.slots = plan.slots, a.min_blocks = plan.min_blocks;
    a.c2 = p->scale * kLog2e;
    const int64_t most = p->table_width * p->pages.page_size;
    const Range range(p->dtype, p->pages.dtype == ARCQ_FP8, p->window ? std::min(most, p->window) : most, plan.tile ? kSlack : 0);
    a.shift = range.shift, a.value_scale = range.value_scale, a.back = range.back;
    a.by_group = Divide(a.group), a.by_kv_heads = Divide(a.kv_heads), a.by_q_heads = Divide(a.q_heads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t dim = p->pages.head_dim;
    const bool f8 = p->pages.dtype == ARCQ_FP8;
    if (p->dtype == ARCQ_F16) f8 ? launch_paged_dim<_Float16, true>(a, plan, dim, st) : launch_paged_dim<_Float16, false>(a, plan, dim, st);
    else f8 ? launch_paged_dim<__bf16, true>(a, plan, dim, st) : launch_paged_dim<__bf16, false>(a, plan, dim, st);
    return launch_status(fn);
}
