// Kernels of the 4-bit key/value cache (format and semantics: include/homcomp_cache.h).
#include "homcomp_cache.hpp"

#include <math.h>

namespace hc {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

enum : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

// ---------------------------------------------------------------- numbers
__device__ __forceinline__ float bf16_to_f32(uint32_t bits) { return __builtin_bit_cast(float, bits << 16); }
__device__ __forceinline__ uint32_t f32_to_bf16(float x) { return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float f16_to_f32(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }
__device__ __forceinline__ uint32_t f32_to_f16(float x) { return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x); }

template <int TY>
__device__ __forceinline__ float load_number(const void *base, uint64_t at)
{
    if (TY == kBf16) return bf16_to_f32(((const uint16_t *)base)[at]);
    if (TY == kF16) return f16_to_f32(((const uint16_t *)base)[at]);
    return ((const float *)base)[at];
}
template <int TY>
__device__ __forceinline__ void store_number(void *base, uint64_t at, float x)
{
    if (TY == kBf16) ((uint16_t *)base)[at] = (uint16_t)f32_to_bf16(x);
    else if (TY == kF16) ((uint16_t *)base)[at] = (uint16_t)f32_to_f16(x);
    else ((float *)base)[at] = x;
}
// Eight adjacent numbers; 16-byte accesses where the address allows them.
template <int TY>
__device__ __forceinline__ void load8(const void *base, uint64_t at, float *x)
{
    const uint8_t *p = (const uint8_t *)base + at * (TY == kF32 ? 4 : 2);
    if (((uintptr_t)p & 15u) == 0) {
        if (TY == kF32) {
            const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 16);
            for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
        } else {
            const u32x4 w = *(const u32x4 *)p;
            for (int i = 0; i < 8; ++i) {
                const uint32_t bits = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
                x[i] = TY == kBf16 ? bf16_to_f32(bits) : f16_to_f32(bits);
            }
        }
    } else {
        for (int i = 0; i < 8; ++i) x[i] = load_number<TY>(base, at + (uint64_t)i);
    }
}
template <int TY>
__device__ __forceinline__ void store8(void *base, uint64_t at, const float *x)
{
    uint8_t *p = (uint8_t *)base + at * (TY == kF32 ? 4 : 2);
    if (((uintptr_t)p & 15u) == 0) {
        if (TY == kF32) {
            *(f32x4 *)p = f32x4{x[0], x[1], x[2], x[3]};
            *(f32x4 *)(p + 16) = f32x4{x[4], x[5], x[6], x[7]};
        } else {
            u32x4 w;
            for (int i = 0; i < 4; ++i) {
                w[i] = TY == kBf16 ? f32_to_bf16(x[2 * i]) | (f32_to_bf16(x[2 * i + 1]) << 16)
                                   : f32_to_f16(x[2 * i]) | (f32_to_f16(x[2 * i + 1]) << 16);
            }
            *(u32x4 *)p = w;
        }
    } else {
        for (int i = 0; i < 8; ++i) store_number<TY>(base, at + (uint64_t)i, x[i]);
    }
}

// ---------------------------------------------------------------- where things are
__device__ __forceinline__ int sequence_length(const CacheArgs &c, int s)
{
    const int n = c.lengths[s];
    return n < 0 ? 0 : (n > c.max_slots ? c.max_slots : n);
}
// Record of slot `slot` (0 <= slot < max_slots), null where the table names no page.
__device__ __forceinline__ uint8_t *record_of(const CacheArgs &c, const int32_t *table, uint32_t stride, int s, int h, int slot, int nb)
{
    const uint32_t page = (uint32_t)table[(uint64_t)s * stride + ((uint32_t)slot >> c.page_shift)];
    if (page >= c.n_pages) return nullptr;
    const uint32_t in_page = (uint32_t)slot & ((1u << c.page_shift) - 1u);
    const uint64_t record = (((uint64_t)page * (uint32_t)c.kv_heads + (uint32_t)h) << (c.page_shift - 5)) + (in_page >> 5);
    return c.pages + record * record_bytes(nb);
}
// Rows of a sequence: its first one and how many, inside 0 .. n_rows.
__device__ __forceinline__ void rows_of(const int32_t *starts, int s, int n_rows, int *first, int *count)
{
    int a = starts[s], b = starts[s + 1];
    a = a < 0 ? 0 : (a > n_rows ? n_rows : a);
    b = b < a ? a : (b > n_rows ? n_rows : b);
    *first = a;
    *count = b - a;
}
// The sequence that owns packed row `r`, -1 for padding: the last s with starts[s] <= r.
__device__ __forceinline__ int sequence_of(const int32_t *starts, int n_seqs, int r)
{
    if (r < starts[0] || r >= starts[n_seqs]) return -1;
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= r) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ---------------------------------------------------------------- the codec
struct Block8 {
    uint32_t code[8];   // of a lane's eight values
    uint32_t s, lo;     // f16 and bf16 bits, the same in the block's four lanes
};
// Four adjacent lanes hold a block, eight values each.  All decisions are those of exact arithmetic: the borders lo + (j + 1/2) s
// have at most 44 significant bits (s is at least a fifteenth of the range, lo at most 2^8 of its own last places), so 64-bit
// floats hold them; a 32-bit estimate that is off by at most one is put right against them.
__device__ __forceinline__ Block8 quantise(const float *x)
{
    float mn = x[0], mx = x[0];
    bool bad = false;
    for (int i = 0; i < 8; ++i) {
        mn = fminf(mn, x[i]);
        mx = fmaxf(mx, x[i]);
        bad = bad || !(fabsf(x[i]) <= 3.4028234663852886e38f);
    }
    for (int d = 1; d < 4; d <<= 1) {
        mn = fminf(mn, __shfl_xor(mn, d, 64));
        mx = fmaxf(mx, __shfl_xor(mx, d, 64));
    }
    int any = bad ? 1 : 0;
    any |= __shfl_xor(any, 1, 64);
    any |= __shfl_xor(any, 2, 64);
    Block8 r;
    // toward minus infinity: cutting the low bits moves toward zero, a negative number that loses some goes one further
    const uint32_t bits = __builtin_bit_cast(uint32_t, mn);
    r.lo = (bits >> 16) + (((bits >> 31) != 0 && (bits & 0xffffu) != 0) ? 1u : 0u);
    const double lo = (double)bf16_to_f32(r.lo), range = (double)mx - lo;
    r.s = f32_to_f16((float)(range / 15.0));
    if ((r.s & 0x7fffu) < 0x7c00u && 15.0 * (double)f16_to_f32(r.s) < range) ++r.s;
    if (any || !(range <= 1.0e38) || (r.s & 0x7fffu) >= 0x7c00u) {
        r.s = 0x7e00u;
        r.lo = 0;
        for (int i = 0; i < 8; ++i) r.code[i] = 0;
        return r;
    }
    const float sf = f16_to_f32(r.s), rs = sf > 0.0f ? 1.0f / sf : 0.0f, lof = (float)lo;
    const double s = (double)sf;
    for (int i = 0; i < 8; ++i) {
        const float guess = fminf(fmaxf(floorf((x[i] - lof) * rs + 0.5f), 0.0f), 15.0f);
        double c = (double)guess;
        const double v = (double)x[i];
        if (c < 15.0 && v >= fma(c + 0.5, s, lo)) c += 1.0;
        else if (c > 0.0 && v < fma(c - 0.5, s, lo)) c -= 1.0;
        r.code[i] = sf > 0.0f ? (uint32_t)(int)c : 0u;
    }
    return r;
}

// Offsets of the parts of a record, in units of nb bytes.
constexpr uint32_t kValueCodes = 512, kKeySteps = 1024, kValueSteps = 1088, kKeyLows = 1152, kValueLows = 1216;

// One row (32-bit numbers x[8] of a block in each four lanes): j is the lane's place in the block, t the slot in the record.
__device__ __forceinline__ void write_key_block(uint8_t *rec, int nb, int t, int b, int j, const Block8 &q)
{
    uint32_t w = 0;
    for (int i = 0; i < 8; ++i) w |= q.code[i] << (4 * (i >> 1) + 16 * (i & 1));
    *(uint32_t *)(rec + t * 16 * nb + j * 4 * nb + 4 * b) = w;
    if (j == 0) {
        *(uint16_t *)(rec + kKeySteps * nb + ((t >> 3) * nb + b) * 16 + (t & 7) * 2) = (uint16_t)q.s;
        *(uint16_t *)(rec + kKeyLows * nb + (t * nb + b) * 2) = (uint16_t)q.lo;
    }
}
// Values m and 16 + m of a block share a byte: lanes j and j ^ 2 exchange (all lanes of the wave take part), and lane j holds the bytes
// m = 8 (j & 1) + 4 (j >> 1) + i afterwards.
__device__ __forceinline__ void value_bytes(int j, const Block8 &q, uint32_t *bytes)
{
    for (int i = 0; i < 4; ++i) {
        const uint32_t give = j < 2 ? q.code[4 + i] : q.code[i];
        const uint32_t got = (uint32_t)__shfl_xor((int)give, 2, 64);
        bytes[i] = j < 2 ? q.code[i] | (got << 4) : got | (q.code[4 + i] << 4);
    }
}
__device__ __forceinline__ void write_value_block(uint8_t *rec, int nb, int t, int b, int j, const Block8 &q, const uint32_t *bytes)
{
    uint8_t *at = rec + kValueCodes * nb + (t >> 3) * 128 * nb + (t & 7) * 2 + (b & 1);
    for (int i = 0; i < 4; ++i) at[((b >> 1) * 16 + 8 * (j & 1) + 4 * (j >> 1) + i) * 16] = (uint8_t)bytes[i];
    if (j == 0) {
        *(uint16_t *)(rec + kValueSteps * nb + ((t >> 3) * nb + b) * 16 + (t & 7) * 2) = (uint16_t)q.s;
        *(uint16_t *)(rec + kValueLows * nb + ((t >> 3) * nb + b) * 16 + (t & 7) * 2) = (uint16_t)q.lo;
    }
}
__device__ __forceinline__ void read_key_block(const uint8_t *rec, int nb, int t, int b, int j, float *x)
{
    const uint32_t w = *(const uint32_t *)(rec + t * 16 * nb + j * 4 * nb + 4 * b);
    const float s = f16_to_f32(*(const uint16_t *)(rec + kKeySteps * nb + ((t >> 3) * nb + b) * 16 + (t & 7) * 2));
    const float lo = bf16_to_f32(*(const uint16_t *)(rec + kKeyLows * nb + (t * nb + b) * 2));
    for (int i = 0; i < 8; ++i) x[i] = fmaf(s, (float)((w >> (4 * (i >> 1) + 16 * (i & 1))) & 15u), lo);
}
__device__ __forceinline__ void read_value_block(const uint8_t *rec, int nb, int t, int b, int j, float *x)
{
    const uint8_t *at = rec + kValueCodes * nb + (t >> 3) * 128 * nb + (t & 7) * 2 + (b & 1);
    const float s = f16_to_f32(*(const uint16_t *)(rec + kValueSteps * nb + ((t >> 3) * nb + b) * 16 + (t & 7) * 2));
    const float lo = bf16_to_f32(*(const uint16_t *)(rec + kValueLows * nb + ((t >> 3) * nb + b) * 16 + (t & 7) * 2));
    for (int i = 0; i < 8; ++i) {
        const int m = 8 * (j & 1) + i;
        x[i] = fmaf(s, (float)((at[((b >> 1) * 16 + m) * 16] >> (4 * (j >> 1))) & 15u), lo);
    }
}

// Four lanes per block of 32 values of a row and head; every lane of a wave takes part in the exchanges, whether its row counts or not.
template <int NB, int TY, bool STORE>
__global__ __launch_bounds__(256) void k_cache_rows(CacheArgs c, RowsArgs a)
{
    const uint64_t unit = ((uint64_t)blockIdx.x * 256 + threadIdx.x) >> 2;   // (row, head, block)
    const int j = threadIdx.x & 3, b = (int)(unit % NB);
    const uint64_t head_row = unit / NB;
    const int h = (int)(head_row % (uint32_t)c.kv_heads);
    const uint64_t row = head_row / (uint32_t)c.kv_heads;
    int s = -1, slot = -1;
    if (row < (uint64_t)a.n_rows) {
        s = sequence_of(a.starts, c.n_seqs, (int)row);
        if (s >= 0) {
            const int n = sequence_length(c, s);
            slot = n - (a.starts[s + 1] - (int)row);
            if (slot < 0 || slot >= n) s = -1;
        }
    }
    uint8_t *rec = s >= 0 ? record_of(c, c.table, c.table_stride, s, h, slot, NB) : nullptr;
    const uint64_t at = row * a.row_stride + (uint64_t)h * a.head_stride + (uint64_t)(32 * b + 8 * j);
    float x[8];
    if (STORE) {
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
        if (rec) load8<TY>(a.k, at, x);
        const Block8 key = quantise(x);
        if (rec) {
            write_key_block(rec, NB, slot & 31, b, j, key);
            load8<TY>(a.v, at, x);
        }
        const Block8 value = quantise(x);
        uint32_t bytes[4];
        value_bytes(j, value, bytes);
        if (rec) write_value_block(rec, NB, slot & 31, b, j, value, bytes);
    } else if (s >= 0) {
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
        if (rec) read_key_block(rec, NB, slot & 31, b, j, x);
        store8<TY>(a.k, at, x);
        if (rec) read_value_block(rec, NB, slot & 31, b, j, x);
        store8<TY>(a.v, at, x);
    }
}

// ---------------------------------------------------------------- attention
//
// One workgroup takes 16 columns -- (row, head of the group) pairs of one sequence and key/value head -- over a part of the
// sequence's records; one wave takes one record (32 slots) at a time.
//
// Codes enter the matrix instructions as they are stored.  A nibble in the low bits of a 16-bit lane is a float16 or bfloat16 below
// the normal range: the float16 of bits c is c 2^-24 and that of 16 c is c 2^-20, the bfloat16 are c 2^-133 and c 2^-129, exactly, and the
// matrix unit takes them at their value.  So an AND (and one shift for every two) is all a pair of codes costs.
//   scores   S[slot, column] = sum_b s_b[slot] (sum_{j in b} c_j q_j) + sum_b lo_b[slot] (sum_{j in b} q_j)
//            one 16x16x32 product per block of 32 values with slots as rows; its result is scaled in 32 bits.  q is float16, scaled by a power
//            of two of its own row so that its largest value is near 2^14 (nothing that counts falls below float16's range), in three
//            parts where q is 32 bits wide.  The lo part is one more product over (block, part of the sums of q).
//   values   O[value, column] = sum_slots c[slot, value] (p s_b)[slot, column] + (sum_slots lo_b p)
//            p s_b is rounded to bfloat16 (two or three parts for outputs of 16 and 32 bits' precision); p carries 2^64 so that
//            products with codes of 2^-133 stay normal numbers.
// A wave's two products of 16 slots each take the slots so that what lane group g gets as scores (rows 4 g + r of both) is
// exactly what it owes the values' product as operand (slots 8 g .. 8 g + 7): nothing is exchanged between lanes.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -INFINITY;

template <int TY>
constexpr int query_parts() { return TY == kF32 ? 3 : 1; }
template <int TY>
constexpr int weight_parts() { return TY == kF32 ? 3 : (TY == kF16 ? 2 : 1); }

template <int NB, int NQ>
struct Queries {
    f16x8 q[NB][NQ];    // values 32 b + 8 g .. + 7 of the column's row, scaled; every other pair by 1/16 more
    bf16x8 sums;        // g-th part (of three) of the sums over each block, times 2^-24
    float factor;       // what turns a score into the exponent of a power of two
    int see_from, see_to;   // slots see_from <= j < see_to are seen
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { return f32_to_bf16(a) | (f32_to_bf16(b) << 16); }

// Eight numbers as NP bfloat16 vectors whose sum they are (to 8, 16 or 24 bits).
template <int NP>
__device__ __forceinline__ void split_bf16(const float *x, bf16x8 *out)
{
    float rest[8];
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
    for (int p = 0; p < NP; ++p) {
        u32x4 w;
        for (int i = 0; i < 4; ++i) {
            w[i] = pack_bf16(rest[2 * i], rest[2 * i + 1]);
            if (p + 1 < NP) {
                rest[2 * i] -= bf16_to_f32(w[i] & 0xffffu);
                rest[2 * i + 1] -= bf16_to_f32(w[i] >> 16);
            }
        }
        out[p] = __builtin_bit_cast(bf16x8, w);
    }
}

// column: row * group + head of the group, at or beyond `columns` none (it sees no slot).
template <int NB, int TY>
__device__ __forceinline__ void load_queries(const AttendArgs &a, int h, int first, int count, int length, int column, int g,
                                             Queries<NB, query_parts<TY>()> &r)
{
    constexpr int NQ = query_parts<TY>();
    const bool there = column < count * a.group;
    const int row = there ? column / a.group : 0, head = there ? column - row * a.group : 0;
    float x[NB][8];
    float top = 0.0f;
    for (int b = 0; b < NB; ++b) {
        for (int i = 0; i < 8; ++i) x[b][i] = 0.0f;
        if (there)
            load8<TY>(a.q, (uint64_t)(first + row) * a.q_row_stride + (uint64_t)(h * a.group + head) * a.q_head_stride + (uint64_t)(32 * b + 8 * g), x[b]);
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[b][i]));
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 126;   // top < 2^e
    if (e > 128) e = 0;                                             // an infinity stays one
    if (e < -100) e = -100;
    const float up = __builtin_bit_cast(float, (uint32_t)(127 + 14 - e) << 23);
    float sums[8];
    for (int b = 0; b < 8; ++b) sums[b] = 0.0f;
    for (int b = 0; b < NB; ++b) {
        float total = 0.0f;
        for (int i = 0; i < 8; ++i) total += x[b][i] * up;
        total += __shfl_xor(total, 16, 64);
        total += __shfl_xor(total, 32, 64);
        sums[b] = total * 0x1p-24f;
        float rest[8];
        for (int i = 0; i < 8; ++i) rest[i] = x[b][i] * up;
        for (int p = 0; p < NQ; ++p) {
            for (int i = 0; i < 8; ++i) {
                const _Float16 part = (_Float16)rest[i];
                rest[i] -= (float)part;
                r.q[b][p][i] = (i & 2) ? (_Float16)((float)part * 0.0625f) : part;
            }
        }
    }
    bf16x8 parts[3];
    split_bf16<3>(sums, parts);
    const bf16x8 none = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
    r.sums = g == 0 ? parts[0] : (g == 1 ? parts[1] : (g == 2 ? parts[2] : none));
    r.factor = ldexpf(a.scale * kLog2e, 10 + e);
    const int at = length - count + row;
    r.see_to = !there ? 0 : (a.causal ? (at + 1 < length ? at + 1 : length) : length);
    r.see_from = a.window > 0 && at + 1 - a.window > 0 ? at + 1 - a.window : 0;
}

// x[T][r]: the exponent (base 2) of slot 8 g + 4 T + r of the record for the lane's column.
template <int NB, int NQ>
__device__ __forceinline__ void record_scores(const uint8_t *rec, int lane, const Queries<NB, NQ> &q, float (&x)[2][4])
{
    const int m = lane & 15, g = lane >> 4;
    for (int T = 0; T < 2; ++T) {
        const int key = 8 * (m >> 2) + 4 * T + (m & 3);
        const uint8_t *codes = rec + key * 16 * NB + g * 4 * NB;
        const uint8_t *lows = rec + kKeyLows * NB + key * 2 * NB;
        u32x4 lo = {0, 0, 0, 0};
        uint32_t w[NB];
        for (int i = 0; i < NB / 2; ++i) lo[i] = ((const uint32_t *)lows)[i];
        for (int b = 0; b < NB; ++b) w[b] = ((const uint32_t *)codes)[b];
        f32x4 acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, lo), q.sums, f32x4{0, 0, 0, 0}, 0, 0, 0);
        for (int b = 0; b < NB; ++b) {
            const uint32_t high = w[b] >> 8;
            const f16x8 c = __builtin_bit_cast(f16x8, u32x4{w[b] & 0x000f000fu, w[b] & 0x00f000f0u, high & 0x000f000fu, high & 0x00f000f0u});
            f32x4 part = {0, 0, 0, 0};
            for (int p = 0; p < NQ; ++p) part = __builtin_amdgcn_mfma_f32_16x16x32_f16(c, q.q[b][p], part, 0, 0, 0);
            const f16x4 s = *(const f16x4 *)(rec + kKeySteps * NB + (g * NB + b) * 16 + 8 * T);
            for (int r = 0; r < 4; ++r) acc[r] = fmaf((float)s[r], part[r], acc[r]);
        }
        for (int r = 0; r < 4; ++r) x[T][r] = acc[r] * q.factor;
    }
}

// Records that a tile's columns can see at all: [*from, *to).
__device__ __forceinline__ void seen_records(const AttendArgs &a, int count, int length, int tile, int *from, int *to)
{
    const int first_row = tile * kColumns / a.group;
    int last_row = (tile * kColumns + kColumns - 1) / a.group;
    if (last_row >= count) last_row = count - 1;
    int end = length, begin = 0;
    if (a.causal && length - count + last_row + 1 < end) end = length - count + last_row + 1;
    if (a.window > 0 && length - count + first_row + 1 - a.window > 0) begin = length - count + first_row + 1 - a.window;
    if (end < 0) end = 0;
    *from = begin >> 5;
    *to = begin < end ? (end + 31) >> 5 : begin >> 5;
}

// One column's share of a workgroup's result: out rows of 16 columns, 16 threads each.
template <int NB, int TY>
__device__ __forceinline__ void write_result(const AttendArgs &a, int h, int first, int column, int part, float top, float total, const float *o)
{
    const int row = column / a.group, head = column - row * a.group;
    constexpr int N = 2 * NB;   // values of this thread: part * N ..
    float x[N];
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    for (int i = 0; i < N; ++i) x[i] = total == 0.0f ? 0.0f : o[i] * inv;
    const uint64_t at = (uint64_t)(first + row) * a.out_row_stride + (uint64_t)(h * a.group + head) * a.out_head_stride + (uint64_t)(part * N);
    for (int i = 0; i < N; ++i) store_number<TY>(a.out, at + (uint64_t)i, x[i]);
    if (a.lse && part == 0)
        a.lse[(uint64_t)(first + row) * ((uint64_t)a.c.kv_heads * a.group) + (uint64_t)(h * a.group + head)] =
            total == 0.0f ? kNegInf : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

template <int NB, int TY>
__global__ __launch_bounds__(256) void k_cache_attend(AttendArgs a)
{
    constexpr int NQ = query_parts<TY>(), NP = weight_parts<TY>(), D = 32 * NB;
    __shared__ float s_o[kAttendWaves][kColumns][D + 4];
    __shared__ float s_top[kAttendWaves][kColumns], s_total[kAttendWaves][kColumns];
    const int split = (int)(blockIdx.x % (unsigned)a.splits);
    const uint32_t unit = blockIdx.x / (unsigned)a.splits;    // (sequence, head, tile)
    const int tile = (int)(unit % (unsigned)a.tiles);
    const int h = (int)(unit / (unsigned)a.tiles % (unsigned)a.c.kv_heads);
    const int s = (int)(unit / (unsigned)a.tiles / (unsigned)a.c.kv_heads);
    int first, count;
    rows_of(a.starts, s, a.n_rows, &first, &count);
    const int length = sequence_length(a.c, s);
    if (count > a.max_rows) count = a.max_rows;
    if (tile * kColumns >= count * a.group) return;
    int from, to;
    seen_records(a, count, length, tile, &from, &to);
    from += split * a.split_records;
    if (split > 0 && from >= to) return;
    if (to > from + a.split_records) to = from + a.split_records;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    Queries<NB, NQ> q;
    load_queries<NB, TY>(a, h, first, count, length, tile * kColumns + n, g, q);
    f32x4 o[NB / 2][4], low = {0, 0, 0, 0};
    for (int i = 0; i < NB / 2; ++i)
        for (int p = 0; p < 4; ++p) o[i][p] = f32x4{0, 0, 0, 0};
    float top = kNegInf, total = 0.0f;

    for (int it = from + wave; it < to; it += kAttendWaves) {
        const uint8_t *rec = record_of(a.c, a.c.table, a.c.table_stride, s, h, it * kRecordSlots, NB);
        if (!rec) continue;
        float x[2][4];
        record_scores<NB, NQ>(rec, lane, q, x);
        const int slot0 = it * kRecordSlots + 8 * g;
        bool seen[8];
        float most = kNegInf;
        for (int i = 0; i < 8; ++i) {
            seen[i] = slot0 + i >= q.see_from && slot0 + i < q.see_to;
            if (seen[i]) most = fmaxf(most, x[i >> 2][i & 3]);
        }
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        const float now = fmaxf(top, most), ref = now == kNegInf ? 0.0f : now;
        const float shrink = __builtin_amdgcn_exp2f(top - ref);   // (nothing so far: 0)
        top = now;
        float p[8];
        total *= shrink;
        for (int i = 0; i < 8; ++i) {
            p[i] = seen[i] ? __builtin_amdgcn_exp2f(x[i >> 2][i & 3] - ref + 64.0f) : 0.0f;
            total += p[i];
        }
        for (int r = 0; r < 4; ++r) {
            low[r] *= shrink;
            for (int i = 0; i < NB / 2; ++i)
                for (int k = 0; k < 4; ++k) o[i][k][r] *= shrink;
        }
        // what the values' lowest numbers contribute; slots behind the last one may hold anything
        u32x4 lows = *(const u32x4 *)(rec + kValueLows * NB + (g * NB + (n < NB ? n : NB - 1)) * 16);
        for (int i = 0; i < 4; ++i) {
            if (slot0 + 2 * i >= length) lows[i] &= 0xffff0000u;
            if (slot0 + 2 * i + 1 >= length) lows[i] &= 0x0000ffffu;
        }
        bf16x8 w[NP];
        split_bf16<NP>(p, w);
        for (int k = 0; k < NP; ++k) low = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, lows), w[k], low, 0, 0, 0);
        for (int b = 0; b < NB; ++b) {
            const f16x8 step = *(const f16x8 *)(rec + kValueSteps * NB + (g * NB + b) * 16);
            float ps[8];
            for (int i = 0; i < 8; ++i) ps[i] = seen[i] ? p[i] * (float)step[i] : 0.0f;
            split_bf16<NP>(ps, w);
            const u32x4 codes = *(const u32x4 *)(rec + kValueCodes * NB + g * 128 * NB + ((b >> 1) * 16 + n) * 16);
            for (int k = 0; k < 2; ++k) {
                u32x4 c;
                for (int i = 0; i < 4; ++i) c[i] = ((b & 1) ? codes[i] >> 8 : codes[i]) & (k ? 0x00f000f0u : 0x000f000fu);
                for (int e = 0; e < NP; ++e)
                    o[b >> 1][2 * (b & 1) + k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, c), w[e], o[b >> 1][2 * (b & 1) + k], 0, 0, 0);
            }
        }
    }

    // the waves' results meet in LDS
    total += __shfl_xor(total, 16, 64);
    total += __shfl_xor(total, 32, 64);
    if (g == 0) {
        s_top[wave][n] = top;
        s_total[wave][n] = total * 0x1p-64f;
    }
    for (int i = 0; i < NB / 2; ++i) {
        for (int p = 0; p < 4; ++p) {
            const int b = 2 * i + (p >> 1);
            f32x4 v;
            float base = 0.0f;
            for (int r = 0; r < 4; ++r) {
                const float other = __shfl(low[r], n + 16 * (b >> 2), 64);
                if (r == (b & 3)) base = other * 0x1p-64f;
            }
            for (int r = 0; r < 4; ++r) v[r] = fmaf(o[i][p][r], (p & 1) ? 0x1p65f : 0x1p69f, base);
            *(f32x4 *)&s_o[wave][n][64 * i + 16 * p + 4 * g] = v;
        }
    }
    __syncthreads();
    const int column = threadIdx.x >> 4, part = threadIdx.x & 15;
    float all = kNegInf;
    for (int w = 0; w < kAttendWaves; ++w) all = fmaxf(all, s_top[w][column]);
    float sum = 0.0f, x[2 * NB];
    for (int i = 0; i < 2 * NB; ++i) x[i] = 0.0f;
    for (int w = 0; w < kAttendWaves; ++w) {
        // (a wave that saw nothing holds zeros; with a NaN among what it saw its total is one)
        const float f = all == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(s_top[w][column] - all);
        sum = fmaf(s_total[w][column], f, sum);
        for (int i = 0; i < 2 * NB; ++i) x[i] = fmaf(s_o[w][column][part * 2 * NB + i], f, x[i]);
    }
    if (a.splits > 1) {
        float *to_part = a.partial + (uint64_t)blockIdx.x * (kColumns * (D + 2));
        for (int i = 0; i < 2 * NB; ++i) to_part[column * D + part * 2 * NB + i] = x[i];
        if (part == 0) {
            to_part[kColumns * D + column] = all;
            to_part[kColumns * D + kColumns + column] = sum;
        }
    } else if (tile * kColumns + column < count * a.group) {
        write_result<NB, TY>(a, h, first, tile * kColumns + column, part, all, sum, x);
    }
}

// Joins the parts of a tile.
template <int NB, int TY>
__global__ __launch_bounds__(256) void k_cache_join(AttendArgs a)
{
    constexpr int D = 32 * NB;
    const int tile = (int)(blockIdx.x % (unsigned)a.tiles);
    const int h = (int)(blockIdx.x / (unsigned)a.tiles % (unsigned)a.c.kv_heads);
    const int s = (int)(blockIdx.x / (unsigned)a.tiles / (unsigned)a.c.kv_heads);
    int first, count;
    rows_of(a.starts, s, a.n_rows, &first, &count);
    const int length = sequence_length(a.c, s);
    if (count > a.max_rows) count = a.max_rows;
    const int column = threadIdx.x >> 4, part = threadIdx.x & 15;
    if (tile * kColumns + column >= count * a.group) return;
    int from, to;
    seen_records(a, count, length, tile, &from, &to);
    int parts = (to - from + a.split_records - 1) / a.split_records;
    if (parts < 1) parts = 1;
    if (parts > a.splits) parts = a.splits;
    const float *at = a.partial + (uint64_t)blockIdx.x * (uint64_t)a.splits * (kColumns * (D + 2));
    float all = kNegInf;
    for (int i = 0; i < parts; ++i) all = fmaxf(all, at[(uint64_t)i * (kColumns * (D + 2)) + kColumns * D + column]);
    float sum = 0.0f, x[2 * NB];
    for (int i = 0; i < 2 * NB; ++i) x[i] = 0.0f;
    for (int k = 0; k < parts; ++k) {
        const float *p = at + (uint64_t)k * (kColumns * (D + 2));
        const float f = all == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(p[kColumns * D + column] - all);
        sum = fmaf(p[kColumns * D + kColumns + column], f, sum);
        for (int i = 0; i < 2 * NB; ++i) x[i] = fmaf(p[column * D + part * 2 * NB + i], f, x[i]);
    }
    write_result<NB, TY>(a, h, first, tile * kColumns + column, part, all, sum, x);
}

// The attention each slot received: a wave takes a record and goes over all columns of its sequence and head, computing the scores
// again (a pass over the keys costs less than keeping a score for every column and slot), and adds in the columns' order.
template <int NB, int TY>
__global__ __launch_bounds__(256) void k_cache_weights(AttendArgs a, int records)
{
    constexpr int NQ = query_parts<TY>();
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const uint32_t groups = ((uint32_t)records + kAttendWaves - 1) / kAttendWaves;
    const int it = (int)(blockIdx.x % groups) * kAttendWaves + wave;
    const int h = (int)(blockIdx.x / groups % (unsigned)a.c.kv_heads);
    const int s = (int)(blockIdx.x / groups / (unsigned)a.c.kv_heads);
    int first, count;
    rows_of(a.starts, s, a.n_rows, &first, &count);
    const int length = sequence_length(a.c, s);
    if (count > a.max_rows) count = a.max_rows;
    if (it * kRecordSlots >= length) return;
    const uint8_t *rec = record_of(a.c, a.c.table, a.c.table_stride, s, h, it * kRecordSlots, NB);
    float sum[8];
    for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
    const int slot0 = it * kRecordSlots + 8 * g;
    for (int tile = 0; tile * kColumns < count * a.group; ++tile) {
        int from, to;
        seen_records(a, count, length, tile, &from, &to);
        if (!rec || it < from || it >= to) continue;
        const int column = tile * kColumns + n;
        Queries<NB, NQ> q;
        load_queries<NB, TY>(a, h, first, count, length, column, g, q);
        float lse = 0.0f;
        if (column < count * a.group) {
            const int row = column / a.group, head = column - row * a.group;
            lse = a.lse[(uint64_t)(first + row) * ((uint64_t)a.c.kv_heads * a.group) + (uint64_t)(h * a.group + head)];
        }
        float x[2][4];
        record_scores<NB, NQ>(rec, lane, q, x);
        for (int i = 0; i < 8; ++i)
            if (slot0 + i >= q.see_from && slot0 + i < q.see_to) sum[i] += __builtin_amdgcn_exp2f(fmaf(lse, -kLog2e, x[i >> 2][i & 3]));
    }
    for (int i = 0; i < 8; ++i)
        for (int d = 1; d < 16; d <<= 1) sum[i] += __shfl_xor(sum[i], d, 64);
    if (n != 0) return;
    const uint64_t at = ((uint64_t)s * a.c.kv_heads + h) * a.weight_stride + (uint64_t)slot0;
    for (int i = 0; i < 8; ++i)
        if (slot0 + i < length) a.weights[at + i] = (a.prior ? a.prior[at + i] : 0.0f) + sum[i];
}

// ---------------------------------------------------------------- eviction
// An unsigned number that orders like the weight: NaN first, both zeros the same.
__device__ __forceinline__ uint32_t weight_key(float w)
{
    uint32_t u = __builtin_bit_cast(uint32_t, w);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
    if (u == 0x80000000u) u = 0;
    return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
// Exclusive prefix of two counts per thread over the workgroup (a: low half, b: high half of one number, at most 1024 each).
__device__ __forceinline__ uint32_t block_prefix(uint32_t mine, uint32_t *sums, uint32_t *all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = mine;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = (uint32_t)__shfl((int)x, lane >= d ? lane - d : lane, 64);
        if (lane >= d) x += y;
    }
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (int w = 0; w < kSelectThreads / 64; ++w) {
        const uint32_t v = sums[w];
        if (w < wave) before += v;
        total += v;
    }
    __syncthreads();
    *all = total;
    return before + x - mine;
}

// A workgroup per sequence and head finds the key of the last weight to stay, byte by byte from the top, then lists what stays in order.
__global__ __launch_bounds__(kSelectThreads) void k_cache_select(EvictArgs a)
{
    __shared__ uint32_t s_count[256];
    __shared__ uint32_t s_sums[kSelectThreads / 64];
    __shared__ uint32_t s_found[2];
    const int h = (int)(blockIdx.x % (unsigned)a.c.kv_heads), s = (int)(blockIdx.x / (unsigned)a.c.kv_heads);
    const int length = sequence_length(a.c, s), tid = threadIdx.x;
    const uint64_t unit = (uint64_t)s * a.c.kv_heads + h;
    const float *w = a.weights + unit * a.weight_stride;
    const int count = length < a.keep ? length : a.keep;
    if (h == 0 && tid == 0) a.to_lengths[s] = count;
    const bool all = length <= a.keep;
    const int low = a.first, high = length - a.recent;           // candidates: low <= slot < high
    uint32_t need = (uint32_t)(a.keep - a.first - a.recent);     // of them to stay
    uint32_t key = 0xffffffffu;
    if (!all && need > 0) {
        uint32_t prefix = 0, mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s_count[tid] = 0;
            __syncthreads();
            for (int j = low + tid; j < high; j += kSelectThreads) {
                const uint32_t k = weight_key(w[j]);
                if ((k & mask) == prefix) atomicAdd(&s_count[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t left = need;
                int digit = 255;
                while (digit > 0 && s_count[digit] < left) left -= s_count[digit--];
                s_found[0] = (uint32_t)digit;
                s_found[1] = left;
            }
            __syncthreads();
            prefix |= s_found[0] << shift;
            mask |= 255u << shift;
            need = s_found[1];
            __syncthreads();
        }
        key = prefix;   // `need` of the weights with this key stay, those in front
    }
    uint32_t kept = 0, equal = 0;
    for (int base = 0; base < length; base += kSelectThreads) {
        const int j = base + tid;
        const bool there = j < length, fixed = there && (all || j < low || j >= high);
        const float weight = there ? w[j] : 0.0f;
        const uint32_t k = weight_key(weight);
        const bool same = there && !fixed && key != 0xffffffffu && k == key;
        uint32_t total;
        const uint32_t before = block_prefix(same ? 1u : 0u, s_sums, &total);
        const bool stays = fixed || (there && !fixed && key != 0xffffffffu && (k > key || (same && equal + before < need)));
        equal += total;
        const uint32_t at = block_prefix(stays ? 1u : 0u, s_sums, &total);
        if (stays && kept + at < (uint32_t)count) {
            a.kept[unit * a.keep + kept + at] = j;
            a.to_weights[unit * a.keep + kept + at] = weight;
        }
        kept += total;
    }
    for (int i = count + tid; i < a.keep; i += kSelectThreads) {
        a.kept[unit * a.keep + i] = -1;
        a.to_weights[unit * a.keep + i] = 0.0f;
    }
}

// A wave moves the kept rows into one record of the new pages.
template <int NB>
__global__ __launch_bounds__(256) void k_cache_move(EvictArgs a, int records)
{
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t groups = ((uint32_t)records + 3) / 4;
    const int it = (int)(blockIdx.x % groups) * 4 + wave;
    const int h = (int)(blockIdx.x / groups % (unsigned)a.c.kv_heads);
    const int s = (int)(blockIdx.x / groups / (unsigned)a.c.kv_heads);
    const int length = sequence_length(a.c, s), count = length < a.keep ? length : a.keep;
    const int left = count - it * kRecordSlots;     // rows of this record
    if (left <= 0) return;
    uint8_t *to = record_of(a.c, a.to_table, a.to_table_stride, s, h, it * kRecordSlots, NB);
    if (!to) return;
    const int32_t *kept = a.kept + ((uint64_t)s * a.c.kv_heads + h) * a.keep + it * kRecordSlots;
    // keys: 16 bytes of a row at a time
    for (int u = lane; u < 32 * NB; u += 64) {
        const int t = u / NB;
        if (t >= left) continue;
        const int slot = kept[t];
        const uint8_t *from = record_of(a.c, a.c.table, a.c.table_stride, s, h, slot, NB);
        u32x4 v = {0, 0, 0, 0};
        if (from) v = *(const u32x4 *)(from + (slot & 31) * 16 * NB + (u % NB) * 16);
        *(u32x4 *)(to + u * 16) = v;
        uint16_t lo = 0;
        if (from) lo = *(const uint16_t *)(from + kKeyLows * NB + ((slot & 31) * NB + u % NB) * 2);
        *(uint16_t *)(to + kKeyLows * NB + u * 2) = lo;
    }
    // what lies by eights of slots: values' codes (8 NB units of 16 bytes for every eight), steps and lowest numbers (NB units)
    constexpr uint32_t kParts[4] = {kValueCodes, kKeySteps, kValueSteps, kValueLows};
    for (int part = 0; part < 4; ++part) {
        const int units = part == 0 ? 8 * NB : NB;
        for (int u = lane; u < 4 * units; u += 64) {
            const int octet = u / units, unit = u % units;
            for (int e = 0; e < 8; ++e) {
                const int t = octet * 8 + e;
                if (t >= left) break;
                const int slot = kept[t];
                const uint8_t *from = record_of(a.c, a.c.table, a.c.table_stride, s, h, slot, NB);
                uint16_t v = 0;
                if (from) v = *(const uint16_t *)(from + kParts[part] * NB + ((((slot & 31) >> 3) * units) + unit) * 16 + (slot & 7) * 2);
                *(uint16_t *)(to + kParts[part] * NB + u * 16 + e * 2) = v;
            }
        }
    }
}

// ---------------------------------------------------------------- launchers
template <bool STORE, int TY>
static hipError_t rows_of_type(const CacheArgs &c, const RowsArgs &r, int nb, hipStream_t s)
{
    const uint64_t threads = (uint64_t)r.n_rows * (uint32_t)c.kv_heads * (uint32_t)nb * 4;
    const dim3 grid((uint32_t)((threads + 255) / 256)), block(256);
    if (nb == 2) hipLaunchKernelGGL((k_cache_rows<2, TY, STORE>), grid, block, 0, s, c, r);
    else if (nb == 4) hipLaunchKernelGGL((k_cache_rows<4, TY, STORE>), grid, block, 0, s, c, r);
    else hipLaunchKernelGGL((k_cache_rows<8, TY, STORE>), grid, block, 0, s, c, r);
    return hipGetLastError();
}
hipError_t launch_cache_store(const CacheArgs &c, const RowsArgs &r, int nb, int type, hipStream_t s)
{
    if (type == kBf16) return rows_of_type<true, kBf16>(c, r, nb, s);
    if (type == kF16) return rows_of_type<true, kF16>(c, r, nb, s);
    return rows_of_type<true, kF32>(c, r, nb, s);
}
hipError_t launch_cache_load(const CacheArgs &c, const RowsArgs &r, int nb, int type, hipStream_t s)
{
    if (type == kBf16) return rows_of_type<false, kBf16>(c, r, nb, s);
    if (type == kF16) return rows_of_type<false, kF16>(c, r, nb, s);
    return rows_of_type<false, kF32>(c, r, nb, s);
}

template <int NB, int TY>
static hipError_t attend_of(const AttendArgs &a, hipStream_t s)
{
    const uint32_t tiles = (uint32_t)a.c.n_seqs * (uint32_t)a.c.kv_heads * (uint32_t)a.tiles;
    hipLaunchKernelGGL((k_cache_attend<NB, TY>), dim3(tiles * (uint32_t)a.splits), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.splits > 1) {
        hipLaunchKernelGGL((k_cache_join<NB, TY>), dim3(tiles), dim3(256), 0, s, a);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.weights) {
        const uint32_t records = ((uint32_t)a.c.max_slots + kRecordSlots - 1) / kRecordSlots;
        const uint32_t groups = (records + kAttendWaves - 1) / kAttendWaves;
        hipLaunchKernelGGL((k_cache_weights<NB, TY>), dim3(groups * (uint32_t)a.c.kv_heads * (uint32_t)a.c.n_seqs), dim3(256), 0, s, a, (int)records);
        e = hipGetLastError();
    }
    return e;
}
template <int NB>
static hipError_t attend_of_blocks(const AttendArgs &a, int type, hipStream_t s)
{
    if (type == kBf16) return attend_of<NB, kBf16>(a, s);
    if (type == kF16) return attend_of<NB, kF16>(a, s);
    return attend_of<NB, kF32>(a, s);
}
hipError_t launch_cache_attend(const AttendArgs &a, int nb, int type, hipStream_t s)
{
    if (nb == 2) return attend_of_blocks<2>(a, type, s);
    if (nb == 4) return attend_of_blocks<4>(a, type, s);
    return attend_of_blocks<8>(a, type, s);
}

hipError_t launch_cache_evict(const EvictArgs &a, int nb, hipStream_t s)
{
    const uint32_t units = (uint32_t)a.c.n_seqs * (uint32_t)a.c.kv_heads;
    hipLaunchKernelGGL(k_cache_select, dim3(units), dim3(kSelectThreads), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const uint32_t records = ((uint32_t)a.keep + kRecordSlots - 1) / kRecordSlots;
    const dim3 grid((records + 3) / 4 * units), block(256);
    if (nb == 2) hipLaunchKernelGGL(k_cache_move<2>, grid, block, 0, s, a, (int)records);
    else if (nb == 4) hipLaunchKernelGGL(k_cache_move<4>, grid, block, 0, s, a, (int)records);
    else hipLaunchKernelGGL(k_cache_move<8>, grid, block, 0, s, a, (int)records);
    return hipGetLastError();
}

}  // namespace hc
