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
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

enum : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

// ---------------------------------------------------------------- numbers
__device__ __forceinline__ float bf16_to_f32(uint32_t bits) { return __builtin_bit_cast(float, bits << 16); }
__device__ __forceinline__ uint32_t f32_to_bf16(float x) { return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float f16_to_f32(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }
__device__ __forceinline__ uint32_t f32_to_f16(float x) { return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x); }

template <int TY>
__device__ __forceinline__ void store_number(void *base, uint64_t at, float x)
{
    if (TY == kBf16) ((uint16_t *)base)[at] = (uint16_t)f32_to_bf16(x);
    else if (TY == kF16) ((uint16_t *)base)[at] = (uint16_t)f32_to_f16(x);
    else ((float *)base)[at] = x;
}
// Eight adjacent numbers; `aligned`: all such addresses of the tensor are multiples of 16 bytes.  (The host says so: with a branch on each
// address every load was waited for by itself, four times the latency in front of a wave's work.)
template <int TY>
struct Eight {
    u32x4 w[TY == kF32 ? 2 : 1];
};
template <int TY>
__device__ __forceinline__ Eight<TY> load_eight(const void *base, uint64_t at, bool aligned)
{
    const uint8_t *p = (const uint8_t *)base + at * (TY == kF32 ? 4 : 2);
    Eight<TY> r;
    if (aligned) {
        r.w[0] = *(const u32x4 *)p;
        if (TY == kF32) r.w[sizeof r.w / 16 - 1] = *(const u32x4 *)(p + 16);
    } else if (TY == kF32) {
        for (int i = 0; i < 8; ++i) r.w[(i >> 2) % (sizeof r.w / 16)][i & 3] = ((const uint32_t *)p)[i];
    } else {
        for (int i = 0; i < 4; ++i) r.w[0][i] = (uint32_t)((const uint16_t *)p)[2 * i] | ((uint32_t)((const uint16_t *)p)[2 * i + 1] << 16);
    }
    return r;
}
template <int TY>
__device__ __forceinline__ void numbers_of(const Eight<TY> &r, float *x)
{
    for (int i = 0; i < 8; ++i) {
        if (TY == kF32) {
            const uint32_t bits = r.w[(i >> 2) % (sizeof r.w / 16)][i & 3];
            x[i] = __builtin_bit_cast(float, bits);
        } else {
            const uint32_t bits = (r.w[0][i >> 1] >> (16 * (i & 1))) & 0xffffu;
            x[i] = TY == kBf16 ? bf16_to_f32(bits) : f16_to_f32(bits);
        }
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

// N adjacent numbers (4, 8 or 16) in pieces of 16 bytes where the address allows them, else one by one.
template <int N, int TY>
__device__ __forceinline__ void store_run(void *base, uint64_t at, const float *x)
{
    constexpr int kSize = TY == kF32 ? 4 : 2;
    uint8_t *p = (uint8_t *)base + at * kSize;
    if (N * kSize < 16) {
        if (((uintptr_t)p & 7u) == 0) {
            u32x2 w;
            for (int i = 0; i < 2; ++i) w[i] = TY == kBf16 ? f32_to_bf16(x[2 * i]) | (f32_to_bf16(x[2 * i + 1]) << 16) : f32_to_f16(x[2 * i]) | (f32_to_f16(x[2 * i + 1]) << 16);
            *(u32x2 *)p = w;
            return;
        }
    } else if (((uintptr_t)p & 15u) == 0) {
        if (TY == kF32) {
            for (int i = 0; i < N; i += 4) *(f32x4 *)(p + 4 * i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
        } else {
            for (int i = 0; i < N; i += 8) store8<TY>(base, at + (uint64_t)i, x + i);
        }
        return;
    }
    for (int i = 0; i < N; ++i) store_number<TY>(base, at + (uint64_t)i, x[i]);
}
// N adjacent 32-bit numbers, `at` of them on, at a multiple of 16 bytes.
template <int N>
__device__ __forceinline__ void load_run(const float *base, uint64_t at, float *x)
{
    for (int i = 0; i < N; i += 4) {
        const f32x4 v = *(const f32x4 *)(base + at + (uint64_t)i);
        for (int k = 0; k < 4; ++k) x[i + k] = v[k];
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
// Page numbers of 64 records ahead, one a lane: records first, first + step, .. below `end`.  A wave reads them from its lanes; a scalar
// load for every record would have its latency in the way of every wait for LDS.
struct PagesAhead {
    uint32_t page;   // of record first + step * (64 q + lane)
    int first, step, end;
    __device__ __forceinline__ void refill(const CacheArgs &c, int s, int it, int lane)
    {
        const int own = it + step * lane;
        page = own < end ? (uint32_t)c.table[(uint64_t)s * c.table_stride + ((uint32_t)(own * kRecordSlots) >> c.page_shift)] : 0xffffffffu;
    }
    // Record `it`, null where the table names no page or it is at or beyond the end.  Calls take first, first + step, .. in turn.
    __device__ __forceinline__ const uint8_t *next(const CacheArgs &c, int s, int h, int it, int lane, int nb)
    {
        const int k = (it - first) / step & 63;
        if (k == 0) refill(c, s, it, lane);
        const uint32_t p = (uint32_t)__builtin_amdgcn_readlane((int)page, k);
        if (p >= c.n_pages || it >= end) return nullptr;
        const uint32_t in_page = ((uint32_t)it << 5) & ((1u << c.page_shift) - 1u);
        const uint64_t record = (((uint64_t)p * (uint32_t)c.kv_heads + (uint32_t)h) << (c.page_shift - 5)) + (in_page >> 5);
        return c.pages + record * record_bytes(nb);
    }
};
// Rows of a sequence: its first one and how many, inside 0 .. n_rows.
struct Rows {
    int first, count;
    int behind;    // rows from `first` to the sequence's last one, also those that are not there for us (n_rows, max_rows)
};
__device__ __forceinline__ Rows rows_of(const int32_t *starts, int s, int n_rows)
{
    int a = starts[s], b = starts[s + 1];
    a = a < 0 ? 0 : (a > n_rows ? n_rows : a);
    const int behind = b < a ? 0 : b - a;
    return Rows{a, b > n_rows ? n_rows - a : behind, behind};
}
// ---------------------------------------------------------------- the codec
struct Block8 {
    uint32_t code[8];   // of a lane's eight values
    uint32_t s, lo;     // f16 and bf16 bits, the same in the block's four lanes
};
// Four adjacent lanes hold a block; what another of them has.
template <int XOR>
__device__ __forceinline__ uint32_t of_quad(uint32_t x)
{
    static_assert(XOR == 1 || XOR == 2, "a lane of the four");
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, XOR == 1 ? 0xb1 : 0x4e, 0xf, 0xf, true);
}
template <int XOR>
__device__ __forceinline__ float of_quad(float x) { return __builtin_bit_cast(float, of_quad<XOR>(__builtin_bit_cast(uint32_t, x))); }

// What a + b, rounded to `sum`, lost: a number of its own (the two-sum of Knuth).
__device__ __forceinline__ double lost(double a, double b, double sum)
{
    const double of_b = sum - a, of_a = sum - of_b;
    return (a - of_a) + (b - of_b);
}

// Eight values a lane.  All decisions are those of exact arithmetic: the range and the borders lo + (j + 1/2) s have at most 44 significant bits (s is at
// least a fifteenth of the range, lo at most 2^8 of its own last places), so 64-bit floats hold them, unless lo and the largest value are far
// apart (1e-30 beside 15).  There a rounded sum still compares rightly with another number, but for a tie: what it lost decides.  In 32 bits
// (x - lo) / s + 1/2 is at most 15 1/2 and off by the roundings of the difference and the sum and the reciprocal's 2^-23: under
// 64 * 2^-24 = 2^-18.  Only where a value is within 2^-17 of a border are the borders looked at: in one wave of a hundred, and in
// one of five where values are bfloat16, whose differences from lo hit some borders exactly.
__device__ __forceinline__ Block8 quantise(const float *x)
{
    float mn = x[0], mx = x[0], odd = 0.0f;
    for (int i = 0; i < 8; ++i) {
        mn = fminf(mn, x[i]);
        mx = fmaxf(mx, x[i]);
        odd = fmaf(x[i], 0.0f, odd);   // a NaN, where there is one or an infinity
    }
    if (!(odd == odd)) mx = __builtin_inff();   // (the block is none then)
    mn = fminf(mn, of_quad<1>(mn));
    mx = fmaxf(mx, of_quad<1>(mx));
    mn = fminf(mn, of_quad<2>(mn));
    mx = fmaxf(mx, of_quad<2>(mx));
    Block8 r;
    // toward minus infinity: cutting the low bits moves toward zero, a negative number that loses some goes one further
    const uint32_t bits = __builtin_bit_cast(uint32_t, mn);
    r.lo = (bits >> 16) + (((bits >> 31) != 0 && (bits & 0xffffu) != 0) ? 1u : 0u);
    const float lo = bf16_to_f32(r.lo);
    const double range = (double)mx - (double)lo;
    r.s = f32_to_f16((float)range * (1.0f / 15.0f));   // (within one place of the quotient: put right below, upward and down)
    if ((r.s & 0x7fffu) < 0x7c00u && r.s > 0 && 15.0 * (double)f16_to_f32(r.s - 1) >= range) --r.s;
    if ((r.s & 0x7fffu) < 0x7c00u && 15.0 * (double)f16_to_f32(r.s) < range) ++r.s;
    const bool none = !(range <= 1.0e38) || (r.s & 0x7fffu) >= 0x7c00u;
    if (none) {
        r.s = 0x7e00u;
        r.lo = 0;
    }
    const float s = f16_to_f32(r.s), rs = s > 0.0f ? __builtin_amdgcn_rcpf(s) : 0.0f;   // (0: all codes are)
    constexpr float near = 0x1p-17f;
    float far = 0.0f;   // from the middle between two borders
    for (int i = 0; i < 8; ++i) {
        const float t = fmaxf(fmaf(x[i] - lo, rs, 0.5f), 0.5f);   // (a NaN: 1/2)
        r.code[i] = (uint32_t)t;
        far = fmaxf(far, fabsf(__builtin_amdgcn_fractf(t) - 0.5f));
    }
    if (far > 0.5f - near) {
        for (int i = 0; i < 8; ++i) {
            const uint32_t c = r.code[i];
            const double v = (double)x[i], at = (double)c;
            if (c < 15 && v >= fma(at + 0.5, (double)s, (double)lo)) r.code[i] = c + 1;
            else if (c > 0 && v < fma(at - 0.5, (double)s, (double)lo)) r.code[i] = c - 1;
        }
    }
    const float lesser = fminf(fabsf(mx), fabsf(lo));
    if (lesser < fmaxf(fabsf(mx), fabsf(lo)) * 0x1p-20f && lesser > 0.0f && !none) {
        // far apart (seldom): a step that only seemed to reach, then every code anew, from an estimate that is at most one off.  (A loop whose
        // body takes the first of the values and turns them round: in line it is much code for every block.)
        if (15.0 * (double)s == range && lost((double)mx, -(double)lo, range) > 0.0) ++r.s;
        const double step = (double)f16_to_f32(r.s);
        const float rstep = __builtin_amdgcn_rcpf((float)step);
        float y[8];
        for (int i = 0; i < 8; ++i) y[i] = x[i];
#pragma unroll 1
        for (int n = 0; n < 8; ++n) {
            uint32_t c = (uint32_t)fmaxf(fmaf(y[0] - lo, rstep, 0.5f), 0.5f);
            auto reaches = [&](double halves) __attribute__((always_inline)) {   // the border lo + halves s
                const double v = (double)y[0], border = (double)lo + halves * step;
                return v > border || (v == border && lost((double)lo, halves * step, border) <= 0.0);
            };
            if (c < 15 && reaches((double)c + 0.5)) ++c;
            else if (c > 0 && !reaches((double)c - 0.5)) --c;
            const float first = y[0];
            for (int i = 0; i < 7; ++i) {
                y[i] = y[i + 1];
                r.code[i] = r.code[i + 1];
            }
            y[7] = first;
            r.code[7] = r.s < 0x7c00u ? c : 0;
        }
        if (r.s >= 0x7c00u) {   // (the step was the largest one)
            r.s = 0x7e00u;
            r.lo = 0;
        }
    }
    return r;
}

// Offsets of the parts of a record, in units of nb bytes (keys' codes at 0).
constexpr uint32_t kValueCodes = 512, kKeySteps = 1024, kValueSteps = 1088, kKeyLows = 1152, kValueLows = 1216;

// A wave takes 16 slots of one head that lie together in a record, as far as they belong to the batch's rows.  Work items: sequence s
// begins at item starts[s] / 16 + 2 s, which leaves room for its rows however they lie to the sixteens.
constexpr int kRowsOfWave = 16;

struct RowsItem {
    int s, h;           // sequence (-1: nothing to do) and head
    int slot0;          // first slot, a multiple of 16
    int begin, end;     // slots of it that are rows: slot0 + begin .. slot0 + end - 1
    int row0;           // packed row of slot0 (may be in front of the first)
};
__device__ __forceinline__ RowsItem rows_item(const CacheArgs &c, const RowsArgs &a, uint32_t item, int lane)
{
    RowsItem r = {-1, (int)(item % (uint32_t)c.kv_heads), 0, 0, 0, 0};
    const int v = (int)(item / (uint32_t)c.kv_heads);
    // the last sequence whose first item is at or in front of v: 64 of them looked at together
    int lo = 0;
    for (int n = c.n_seqs; n > 1;) {
        const int step = (n + 63) >> 6, own = lo + lane * step;
        int at = lane * step < n ? a.starts[own] : 0;
        at = at < 0 ? 0 : (at > a.n_rows ? a.n_rows : at);
        const int m = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane * step < n && (at >> 4) + 2 * own <= v));
        const int skip = m > 0 ? (m - 1) * step : 0;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    const Rows rows = rows_of(a.starts, lo, a.n_rows);
    const int first = rows.first, count = rows.count, length = sequence_length(c, lo);
    const int from = length - rows.behind;        // slot of the first row, in front of 0 where there are more rows than slots
    const int begin = from > 0 ? from : 0;
    const int last = from + count < length ? from + count : length;
    const int group = (begin >> 4) + v - (first >> 4) - 2 * lo;
    if (group < (begin >> 4) || group * kRowsOfWave >= last) return r;
    r.s = lo;
    r.slot0 = group * kRowsOfWave;
    r.begin = begin > r.slot0 ? begin - r.slot0 : 0;
    r.end = last - r.slot0 < kRowsOfWave ? last - r.slot0 : kRowsOfWave;
    r.row0 = first + (r.slot0 - from);
    return r;
}
__device__ __forceinline__ void wave_lds_order()
{
    // a wave's LDS accesses take effect in order; this keeps the compiler from changing it
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 123 thousand slots and heads of 128 values take 30 us, 2.7 TB/s of rows and records.  Quantising, 1590 vector instructions for sixteen slots, keeps the
// vector units busy for 55 % of it; the rest is that 1942 workgroups are one and a half times what the chip holds at once, and that a
// wave loads nothing ahead.  (36 us with neighbours exchanged through LDS and borders looked at value by value; 29 before blocks whose
// numbers lie far apart were decided exactly, which costs registers.)
// Keys: four lanes to a slot, a lane's eight values of every block.  Values' codes of a slot lie two bytes at a time among those of seven others: the
// wave gathers eight slots' words in LDS and writes them whole, except where not all eight are its own.
template <int NB, int TY>
__global__ __launch_bounds__(256) void k_cache_store(CacheArgs c, RowsArgs a, uint32_t items)
{
    __shared__ __align__(16) uint16_t s_words[4][2][8 * NB][8];   // [wave][octet][unit][slot]
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const uint32_t item = blockIdx.x * 4u + (uint32_t)wave;
    if (item >= items) return;
    const RowsItem r = rows_item(c, a, item, lane);
    if (r.s < 0) return;
    uint8_t *rec = record_of(c, c.table, c.table_stride, r.s, r.h, r.slot0, NB);
    if (!rec) return;
    const int t = lane >> 2, j = lane & 3, slot = (r.slot0 & 31) + t;   // slot of the record
    const bool own = t >= r.begin && t < r.end;
    const uint64_t at = (uint64_t)(int64_t)(r.row0 + (own ? t : r.begin)) * a.row_stride + (uint64_t)r.h * a.head_stride + (uint64_t)(8 * j);
    Eight<TY> keys[NB], values[NB];
    if (a.aligned) {
        for (int b = 0; b < NB; ++b) keys[b] = load_eight<TY>(a.k, at + (uint64_t)(32 * b), true);
        for (int b = 0; b < NB; ++b) values[b] = load_eight<TY>(a.v, at + (uint64_t)(32 * b), true);
    } else {
        for (int b = 0; b < NB; ++b) keys[b] = load_eight<TY>(a.k, at + (uint64_t)(32 * b), false);
        for (int b = 0; b < NB; ++b) values[b] = load_eight<TY>(a.v, at + (uint64_t)(32 * b), false);
    }
    float x[8];
#pragma unroll
    for (int half = 0; half < (NB + 3) / 4; ++half) {
        uint32_t w[4] = {0, 0, 0, 0}, step = 0, low = 0;
#pragma unroll
        for (int n = 0; n < 4 && 4 * half + n < NB; ++n) {
            numbers_of<TY>(keys[4 * half + n], x);
            const Block8 q = quantise(x);
            for (int i = 0; i < 8; ++i) w[n] |= q.code[i] << (4 * (i >> 1) + 16 * (i & 1));
            if (j == n) step = q.s, low = q.lo;
        }
        if (own) {
            uint32_t *to = (uint32_t *)(rec + slot * 16 * NB + j * 4 * NB + 16 * half);
            for (int n = 0; n < 4 && 4 * half + n < NB; ++n) to[n] = w[n];
            const int b = 4 * half + j;   // a lane writes the scales of block j
            if (b < NB) {
                *(uint16_t *)(rec + kKeySteps * NB + ((slot >> 3) * NB + b) * 16 + (slot & 7) * 2) = (uint16_t)step;
                *(uint16_t *)(rec + kKeyLows * NB + (slot * NB + b) * 2) = (uint16_t)low;
            }
        }
    }
    uint32_t step[(NB + 3) / 4], low[(NB + 3) / 4];
#pragma unroll
    for (int i = 0; i < NB / 2; ++i) {
        uint32_t word[4] = {0, 0, 0, 0};   // of units 16 i + 8 (j & 1) + 4 (j >> 1) + n
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            numbers_of<TY>(values[2 * i + e], x);
            const Block8 q = quantise(x);
            // value m and value 16 + m of the block share a byte: lanes j and j ^ 2 exchange
            for (int n = 0; n < 4; ++n) {
                const uint32_t give = j < 2 ? q.code[4 + n] : q.code[n];
                const uint32_t got = of_quad<2>(give);
                word[n] |= (j < 2 ? q.code[n] | (got << 4) : got | (q.code[4 + n] << 4)) << (8 * e);
            }
            if (j == ((2 * i + e) & 3)) step[(2 * i + e) >> 2] = q.s, low[(2 * i + e) >> 2] = q.lo;
        }
        for (int n = 0; n < 4; ++n) s_words[wave][t >> 3][16 * i + 8 * (j & 1) + 4 * (j >> 1) + n][t & 7] = (uint16_t)word[n];
    }
    if (own) {
        for (int half = 0; half < (NB + 3) / 4; ++half) {
            const int b = 4 * half + j;
            if (b < NB) {
                *(uint16_t *)(rec + kValueSteps * NB + ((slot >> 3) * NB + b) * 16 + (slot & 7) * 2) = (uint16_t)step[half];
                *(uint16_t *)(rec + kValueLows * NB + ((slot >> 3) * NB + b) * 16 + (slot & 7) * 2) = (uint16_t)low[half];
            }
        }
    }
    wave_lds_order();
    for (int u = lane; u < 16 * NB; u += 64) {
        const int o = u / (8 * NB), unit = u % (8 * NB);
        const u32x4 words = *(const u32x4 *)s_words[wave][o][unit];
        uint8_t *to = rec + kValueCodes * NB + (((r.slot0 & 31) >> 3) + o) * 128 * NB + unit * 16;
        if (8 * o >= r.begin && 8 * o + 8 <= r.end) {
            *(u32x4 *)to = words;
        } else {
            for (int n = 0; n < 8; ++n)
                if (8 * o + n >= r.begin && 8 * o + n < r.end) ((uint16_t *)to)[n] = s_words[wave][o][unit][n];
        }
    }
}

// The mirror: keys straight to their rows, values through LDS, where rows come together.
// Rows leave through LDS, whole ones at a time and past the caches (nobody reads them again before hundreds of others): a cache of 668 thousand
// slots and heads of 128 values read as bfloat16, 448 MB in and out, takes 67 us.  It took 89 where the stores stayed in the caches, 133 where besides
// each lane stored the eight values it had, 64 bytes of a row by four lanes, and waited for a block before it loaded the next.
template <int NB, int TY>
__global__ __launch_bounds__(256) void k_cache_load(CacheArgs c, RowsArgs a, uint32_t items)
{
    constexpr int D = 32 * NB, kSize = TY == kF32 ? 4 : 2, kUnits = (16 * NB + 63) / 64;
    __shared__ __align__(16) uint8_t s_rows[4][kRowsOfWave][D * kSize + 16];   // (16: rows begin at other banks)
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const uint32_t item = blockIdx.x * 4u + (uint32_t)wave;
    if (item >= items) return;
    const RowsItem r = rows_item(c, a, item, lane);
    if (r.s < 0) return;
    const uint8_t *rec = record_of(c, c.table, c.table_stride, r.s, r.h, r.slot0, NB);
    const int t = lane >> 2, j = lane & 3, slot = (r.slot0 & 31) + t;
    // everything of the sixteen slots on its way before any of it is waited for (slots that are not rows are loaded too, from the same record)
    uint32_t codes[NB], step[NB], low[NB / 2];
    u32x4 words[kUnits], steps[kUnits][2], lows[kUnits][2];
    if (rec) {
        for (int b = 0; b < NB; ++b) codes[b] = ((const uint32_t *)(rec + slot * 16 * NB + j * 4 * NB))[b];
        for (int b = 0; b < NB; ++b) step[b] = *(const uint16_t *)(rec + kKeySteps * NB + ((slot >> 3) * NB + b) * 16 + (slot & 7) * 2);
        for (int b = 0; b < NB / 2; ++b) low[b] = ((const uint32_t *)(rec + kKeyLows * NB + slot * NB * 2))[b];
        for (int k = 0; k < kUnits; ++k) {
            const int u = 64 * k + lane, o = u / (8 * NB), unit = u % (8 * NB), octet = ((r.slot0 & 31) >> 3) + o;
            if (u >= 16 * NB) continue;
            words[k] = *(const u32x4 *)(rec + kValueCodes * NB + octet * 128 * NB + unit * 16);
            for (int e = 0; e < 2; ++e) {
                steps[k][e] = *(const u32x4 *)(rec + kValueSteps * NB + (octet * NB + 2 * (unit >> 4) + e) * 16);
                lows[k][e] = *(const u32x4 *)(rec + kValueLows * NB + (octet * NB + 2 * (unit >> 4) + e) * 16);
            }
        }
    } else {
        for (int b = 0; b < NB; ++b) codes[b] = step[b] = low[b / 2] = 0;
        for (int k = 0; k < kUnits; ++k) words[k] = steps[k][0] = steps[k][1] = lows[k][0] = lows[k][1] = u32x4{0, 0, 0, 0};
    }
    // whole rows from LDS to the array
    auto write_rows = [&](void *base) __attribute__((always_inline)) {
        constexpr int kPieces = D * kSize / 16;   // of a row
        wave_lds_order();
        for (int u = lane; u < kRowsOfWave * kPieces; u += 64) {
            const int row = u / kPieces, piece = u % kPieces;
            if (row < r.begin || row >= r.end) continue;
            const u32x4 v = *(const u32x4 *)(s_rows[wave][row] + piece * 16);
            uint8_t *to = (uint8_t *)base + ((uint64_t)(int64_t)(r.row0 + row) * a.row_stride + (uint64_t)r.h * a.head_stride) * kSize + (uint64_t)(piece * 16);
            if (a.aligned) {
                __builtin_nontemporal_store(v, (u32x4 *)to);
            } else if (TY == kF32) {
                for (int n = 0; n < 4; ++n) ((uint32_t *)to)[n] = v[n];
            } else {
                for (int n = 0; n < 8; ++n) ((uint16_t *)to)[n] = (uint16_t)(v[n >> 1] >> (16 * (n & 1)));
            }
        }
        wave_lds_order();
    };
    for (int b = 0; b < NB; ++b) {
        float x[8];
        const float s = f16_to_f32(step[b]), lo = (b & 1) ? __builtin_bit_cast(float, low[b >> 1] & 0xffff0000u) : bf16_to_f32(low[b >> 1] & 0xffffu);
        for (int i = 0; i < 8; ++i) x[i] = fmaf(s, (float)((codes[b] >> (4 * (i >> 1) + 16 * (i & 1))) & 15u), lo);
        store8<TY>(s_rows[wave][t], (uint64_t)(32 * b + 8 * j), x);
    }
    write_rows(a.k);
    for (int k = 0; k < kUnits; ++k) {
        const int u = 64 * k + lane, o = u / (8 * NB), unit = u % (8 * NB), i = unit >> 4, m = unit & 15;
        if (u >= 16 * NB) continue;
        for (int n = 0; n < 8; ++n) {
            const uint32_t word = words[k][n >> 1] >> (16 * (n & 1));
            for (int p = 0; p < 4; ++p) {
                const uint32_t own = steps[k][p >> 1][n >> 1], lowest = lows[k][p >> 1][n >> 1];
                const float s = f16_to_f32((own >> (16 * (n & 1))) & 0xffffu);
                const float lo = (n & 1) ? __builtin_bit_cast(float, lowest & 0xffff0000u) : bf16_to_f32(lowest & 0xffffu);
                store_number<TY>(s_rows[wave][8 * o + n], (uint64_t)(64 * i + 16 * p + m), fmaf(s, (float)((word >> (4 * p)) & 15u), lo));
            }
        }
    }
    write_rows(a.v);
}

// ---------------------------------------------------------------- attention
//
// One workgroup takes 16 columns -- (row, head of the group) pairs of one sequence and key/value head -- over a part of the
// sequence's records; one wave takes one record (32 slots) at a time.
//
// Codes enter the matrix instructions as they are stored.  A nibble in the low bits of a 16-bit lane is a float16 or bfloat16 below
// the normal range: the float16 of bits c is c 2^-24 and that of 16 c is c 2^-20, the bfloat16 are c 2^-133 and c 2^-129, exactly, and the
// matrix unit takes them at their value.  So an AND and at most one shift is all a pair of codes costs.
//   scores   S[slot, column] = sum_b s_b[slot] (sum_{j in b} c_j q_j) + sum_b lo_b[slot] (sum_{j in b} q_j)
//            one 16x16x32 product per block of 32 values with slots as rows; its result is scaled in 32 bits.  q is float16, scaled by a power
//            of two of its own row so that its largest value is near 2^14 (nothing that counts falls below float16's range), in three
//            parts where q is 32 bits wide.  The lo part is one more product over (block, part of the sums of q).
//   values   O[value, column] = sum_slots c[slot, value] (p s_b)[slot, column] + (sum_slots lo_b p)
//            p s_b is rounded to bfloat16 (two or three parts for outputs of 16 and 32 bits' precision); p carries 2^64 so that
//            products with codes of 2^-133 stay normal numbers (see there for lo of 2^40 and more).  For 16-bit outputs a record whose
//            values all fit float16 is multiplied as float16 numbers lo + s c instead: a third of the vector instructions.
// A wave's two products of 16 slots each take the slots so that what lane group g gets as scores (rows 4 g + r of both) is
// exactly what it owes the values' product as operand (slots 8 g .. 8 g + 7): nothing is exchanged between lanes.
//
// What bounds it is reading the records.  64 sequences of up to 8192 slots, 8 heads of 128 values, four columns each: 327 MB in 85 us, 3.8 TB/s, vector
// instructions busy for 42 % of it (355 for a record); joining the parts adds 6 us.  One sequence of 131072
// slots: 168 MB in 35 us, 4.8 TB/s, nearly what a copy of the same bytes reaches.  Values as codes: 106 and 47 us.  Records through LDS
// one ahead, from where operands are taken: without it (operands loaded from memory in their order) 236 us for the batch.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -INFINITY;

template <int TY>
constexpr int query_parts() { return TY == kF32 ? 3 : 1; }

template <int NB, int NQ>
struct Queries {
    f16x8 q[NB][NQ];    // values 32 b + 8 g .. + 7 of the column's row, scaled; with codes at bits 4 .. 7 (sixteen times as high) by 1/16 more
    bf16x8 sums;        // g-th part (of three) of the sums over each block, times what the codes are
    float factor;       // what turns a score into the exponent of a power of two, short of
    int shift;          // 2^shift: 0 but for queries and scales near the end of 32 bits (the same in all lanes)
    int see_from, see_to;   // slots see_from <= j < see_to are seen
};

template <int NB, int NQ>
__device__ __forceinline__ bool sees(const Queries<NB, NQ> &q, int slot) { return slot >= q.see_from && slot < q.see_to; }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b}); }

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
// How codes enter the products of the scores.  kFine: see code_pairs; kWhole: keys as numbers, lo + s c.
enum : int { kFine = 0, kWhole = 1 };
template <int NB, int TY, int FORM>
__device__ __forceinline__ void load_queries(const AttendArgs &a, int h, int first, int count, int slot0, int length, int column, int g,
                                             Queries<NB, query_parts<TY>()> &r)
{
    constexpr int NQ = query_parts<TY>();
    const bool there = column < count * a.group;
    const int row = there ? column / a.group : 0, head = there ? column - row * a.group : 0;
    // (a column that is not there reads row 0 of the sequence, which is, and counts as zeros)
    const uint64_t at = (uint64_t)(first + row) * a.q_row_stride + (uint64_t)(h * a.group + head) * a.q_head_stride + (uint64_t)(8 * g);
    Eight<TY> raw[NB];
    if (a.q_aligned) {
        for (int b = 0; b < NB; ++b) raw[b] = load_eight<TY>(a.q, at + (uint64_t)(32 * b), true);
    } else {
        for (int b = 0; b < NB; ++b) raw[b] = load_eight<TY>(a.q, at + (uint64_t)(32 * b), false);
    }
    float x[NB][8];
    float top = 0.0f;
    for (int b = 0; b < NB; ++b) {
        numbers_of<TY>(raw[b], x[b]);
        for (int i = 0; i < 8; ++i) {
            x[b][i] = there ? x[b][i] : 0.0f;
            top = fmaxf(top, fabsf(x[b][i]));
        }
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
        sums[b] = FORM == kWhole ? total : total * 0x1p-24f;
        float rest[8];
        for (int i = 0; i < 8; ++i) rest[i] = x[b][i] * up;
        for (int p = 0; p < NQ; ++p) {
            for (int i = 0; i < 8; ++i) {
                const _Float16 part = (_Float16)rest[i];
                rest[i] -= (float)part;
                r.q[b][p][i] = FORM == kFine ? (_Float16)((float)part * 0.0625f) : part;
            }
        }
    }
    bf16x8 parts[3];
    split_bf16<3>(sums, parts);
    const bf16x8 none = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
    r.sums = g == 0 ? parts[0] : (g == 1 ? parts[1] : (g == 2 ? parts[2] : none));
    int above = a.scale_exponent + (FORM == kWhole ? -14 : 10) + e - 126;
    r.shift = 0;
    if (__builtin_amdgcn_ballot_w64(above > 0) != 0) {
        int most = above;
        for (int lane = 1; lane < 16; lane *= 2) {
            const int other = __shfl_xor(most, lane, 64);
            most = other > most ? other : most;
        }
        r.shift = __builtin_amdgcn_readfirstlane(most);
    }
    r.factor = ldexpf(a.scale, above + 126 - r.shift);
    const int own = slot0 + row;
    r.see_to = !there ? 0 : (a.causal ? (own + 1 < length ? own + 1 : length) : length);
    r.see_from = a.window > 0 && own + 1 > a.window ? own + 1 - a.window : 0;
}

// What a lane holds of a record: rows of the products' operands, and the scales of what it gets back.
template <int NB>
struct KeyPart {
    uint32_t codes[2][NB];      // slots 8 (m / 4) + 4 T + m % 4, m = lane % 16: values 32 b + 8 g .. + 7
    uint32_t lows[2][NB / 2];   // the same slots' lowest numbers
    f16x8 steps[NB];            // of slots 8 g .. + 7
};
template <int NB>
struct ValuePart {
    u32x4 codes[NB / 2];        // slots 8 g .. + 7: values 64 i + 16 p + m
    f16x8 steps[NB];
    u32x4 lows;                 // of block m % NB
    u32x4 own_steps;            // likewise, bits of float16
};
// A record on its way: 16-byte pieces lane, lane + 64, .. of it, loaded ahead, then laid into the wave's own part of LDS, from
// where lanes take what they need (a scale goes to sixteen lanes; LDS hands it to all of them at once).  Keys' codes are laid so that
// the lanes of a read lie side by side: [half of a row's share][T][g][m] instead of [slot][g][half].
template <int NB>
struct RawRecord {
    static constexpr int kPieces = (80 * NB + 63) / 64;
    u32x4 piece[kPieces];
};
template <int NB>
__device__ __forceinline__ void load_record(const uint8_t *rec, int lane, RawRecord<NB> &raw)
{
    for (int i = 0; i < RawRecord<NB>::kPieces; ++i)
        if (64 * i + 64 <= 80 * NB || 64 * i + lane < 80 * NB) raw.piece[i] = *(const u32x4 *)(rec + (64 * i + lane) * 16);
}
template <int NB>
__device__ __forceinline__ int key_place(int piece)   // where piece `piece` of the keys' codes is laid
{
    if (NB == 2) return piece;
    constexpr int kHalves = NB / 4;
    const int half = piece % kHalves, g = piece / kHalves % 4, key = piece / (4 * kHalves);
    const int T = (key >> 2) & 1, m = 4 * (key >> 3) + (key & 3);
    return ((half * 2 + T) * 4 + g) * 16 + m;
}
template <int NB>
__device__ __forceinline__ void lay_record(uint8_t *at, int lane, const RawRecord<NB> &raw)
{
    for (int i = 0; i < RawRecord<NB>::kPieces; ++i) {
        const int piece = 64 * i + lane;
        if (64 * i + 64 <= 80 * NB || piece < 80 * NB) *(u32x4 *)(at + (64 * i < 32 * NB ? key_place<NB>(piece) : piece) * 16) = raw.piece[i];
    }
    // a wave's LDS accesses take effect in order; this keeps the compiler from changing it
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// STEPS, LOWS: where the keys' steps and lowest numbers lie, in units of NB bytes.
template <int NB, uint32_t STEPS = kKeySteps, uint32_t LOWS = kKeyLows>
__device__ __forceinline__ void take_keys(const uint8_t *at, int lane, KeyPart<NB> &k)
{
    const int m = lane & 15, g = lane >> 4;
    for (int T = 0; T < 2; ++T) {
        const int key = 8 * (m >> 2) + 4 * T + (m & 3);
        if (NB == 2) {
            const u32x2 w = *(const u32x2 *)(at + key * 32 + g * 8);
            k.codes[T][0] = w[0];
            k.codes[T][1] = w[1];
        } else {
            for (int half = 0; half < NB / 4; ++half) {
                const u32x4 w = *(const u32x4 *)(at + (((half * 2 + T) * 4 + g) * 16 + m) * 16);
                for (int i = 0; i < 4; ++i) k.codes[T][4 * half + i] = w[i];
            }
        }
        const uint32_t *lows = (const uint32_t *)(at + LOWS * NB + key * 2 * NB);
        for (int i = 0; i < NB / 2; ++i) k.lows[T][i] = lows[i];
    }
    for (int b = 0; b < NB; ++b) k.steps[b] = *(const f16x8 *)(at + STEPS * NB + (g * NB + b) * 16);
}
template <int NB>
__device__ __forceinline__ void take_values(const uint8_t *at, int lane, ValuePart<NB> &v)
{
    const int m = lane & 15, g = lane >> 4, own = m & (NB - 1);
    for (int i = 0; i < NB / 2; ++i) v.codes[i] = *(const u32x4 *)(at + kValueCodes * NB + g * 128 * NB + (i * 16 + m) * 16);
    for (int b = 0; b < NB; ++b) v.steps[b] = *(const f16x8 *)(at + kValueSteps * NB + (g * NB + b) * 16);
    v.lows = *(const u32x4 *)(at + kValueLows * NB + (g * NB + own) * 16);
    v.own_steps = *(const u32x4 *)(at + kValueSteps * NB + (g * NB + own) * 16);
}

// The four pairs of codes of a word, as numbers of 16 bits below or at the foot of the normal range.  FINE: all at bits 4 .. 7, for two
// more shifts: the matrix unit aligns products by their exponents, a number below the normal range counts as if it
// had the smallest one, and what a product has in front of its first bit it lacks behind the last (measured for a score of a few
// units: 4e-6 off with codes at bits 0 .. 3, 3e-7 at bits 4 .. 7).  So scores, which lse and the weights are made of, take that form, whatever the type
// of the results: 0.5 us of 91 for a batch of 64 sequences.  Values for 16-bit results take the other.
template <bool FINE>
__device__ __forceinline__ u32x4 code_pairs(uint32_t w)
{
    if (FINE) return u32x4{(w << 4) & 0x00f000f0u, w & 0x00f000f0u, (w >> 4) & 0x00f000f0u, (w >> 8) & 0x00f000f0u};
    const uint32_t high = w >> 8;
    return u32x4{w & 0x000f000fu, w & 0x00f000f0u, high & 0x000f000fu, high & 0x00f000f0u};
}

// x[T][r]: the score, short of `factor`, of slot 8 g + 4 T + r of the record for the lane's column.
template <int NB, int NQ>
__device__ __forceinline__ void record_scores(const KeyPart<NB> &k, const Queries<NB, NQ> &q, const f32x4 &zero, f32x4 (&x)[2])
{
    f32x4 part[2][NB];
    for (int T = 0; T < 2; ++T) {
        u32x4 lo = {0, 0, 0, 0};
        for (int i = 0; i < NB / 2; ++i) lo[i] = k.lows[T][i];
        x[T] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, lo), q.sums, zero, 0, 0, 0);
        for (int b = 0; b < NB; ++b) {
            const f16x8 c = __builtin_bit_cast(f16x8, code_pairs<true>(k.codes[T][b]));
            for (int p = 0; p < NQ; ++p) part[T][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c, q.q[b][p], p ? part[T][b] : zero, 0, 0, 0);
        }
    }
    for (int T = 0; T < 2; ++T)
        for (int b = 0; b < NB; ++b)
            for (int r = 0; r < 4; ++r) x[T][r] = fmaf((float)k.steps[b][4 * T + r], part[T][b][r], x[T][r]);
}

// Records that a tile's columns can see at all: [*from, *to).
__device__ __forceinline__ void seen_records(const AttendArgs &a, int count, int slot0, int length, int tile, int *from, int *to, int columns = kColumns)
{
    const int first_row = tile * columns / a.group;
    int last_row = (tile * columns + columns - 1) / a.group;
    if (last_row >= count) last_row = count - 1;
    int end = length, begin = 0;
    if (a.causal && slot0 + last_row + 1 < end) end = slot0 + last_row + 1;
    if (a.window > 0 && slot0 + first_row + 1 > a.window) begin = slot0 + first_row + 1 - a.window;
    if (end < 0) end = 0;
    *from = begin >> 5;
    *to = begin < end ? (end + 31) >> 5 : begin >> 5;
}
// The record a tile's parts are counted from: the first that it can see, or that the wide tile can which it belongs to (whose parts they
// are then).
__device__ __forceinline__ int parts_origin(const AttendArgs &a, int count, int slot0, int length, int tile)
{
    int from, to;
    if (a.wide_tiles) seen_records(a, count, slot0, length, tile / a.tiles_in_wide, &from, &to, kColumns * a.tiles_in_wide);
    else seen_records(a, count, slot0, length, tile, &from, &to);
    return from;
}
// Records of a part counted from `origin`.  The host plans parts for window + max_rows slots, which is all that causal rows under a window see.
// Others see up to the sequence's last slot, and rows that are left out (max_rows, n_rows) stand between: parts are longer then.
__device__ __forceinline__ int records_of_part(const AttendArgs &a, int length, int origin)
{
    if (a.causal || a.window == 0) return a.split_records;
    const int each = (((length + 31) >> 5) - origin + a.splits - 1) / a.splits;
    return each <= a.split_records ? a.split_records : (each + kAttendWaves - 1) / kAttendWaves * kAttendWaves;
}
// Slots that every one of a tile's columns sees: [*from, *to).
template <int COLUMNS = kColumns>
__device__ __forceinline__ void seen_by_all(const AttendArgs &a, int count, int slot0, int length, int tile, int *from, int *to)
{
    const int first_row = tile * COLUMNS / a.group;
    int last_row = (tile * COLUMNS + COLUMNS - 1) / a.group;
    if (last_row >= count) last_row = count - 1;
    *to = a.causal && slot0 + first_row + 1 < length ? slot0 + first_row + 1 : length;
    *from = a.window > 0 && slot0 + last_row + 1 > a.window ? slot0 + last_row + 1 - a.window : 0;
}

// One column's share of a workgroup's result: out rows of 16 columns, 16 threads each.  o: the mean of the values; total: the sum of the weights,
// relative to 2^top.
template <int NB, int TY>
__device__ __forceinline__ void write_result(const AttendArgs &a, int h, int first, int column, int part, float top, float total, const float *o)
{
    const int row = column / a.group, head = column - row * a.group;
    constexpr int N = 2 * NB;   // values of this thread: part * N ..
    const uint64_t at = (uint64_t)(first + row) * a.out_row_stride + (uint64_t)(h * a.group + head) * a.out_head_stride + (uint64_t)(part * N);
    store_run<N, TY>(a.out, at, o);
    if (a.lse && part == 0)
        a.lse[(uint64_t)(first + row) * ((uint64_t)a.c.kv_heads * a.group) + (uint64_t)(h * a.group + head)] =
            total == 0.0f ? kNegInf : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

// Values the compiler is not to look through: a register of zeros for products to start from (it would clear one for each), a number that
// comparisons under a rare branch depend on (it would make them in front of the branch).
__device__ __forceinline__ f32x4 kept_zero()
{
    f32x4 zero = {0, 0, 0, 0};
    asm volatile("" : "+v"(zero));
    return zero;
}
__device__ __forceinline__ int kept_here(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}

// Two codes as float16 numbers: at bits 0 .. 3 under 1024, at bits 4 .. 7 under 64, both exact.
// (The numbers they stand under are held in registers: one instruction then joins and masks.)
struct Under {
    uint32_t of_0, of_4;
    float minus;   // -1, which the compiler would make a conversion and a difference of
};
__device__ __forceinline__ Under under_codes() { return {(uint32_t)kept_here(0x64006400), (uint32_t)kept_here(0x54005400), __builtin_bit_cast(float, kept_here((int)0xbf800000))}; }
__device__ __forceinline__ f16x2 codes_at_0(uint32_t w, const Under &u) { return __builtin_bit_cast(f16x2, (w & 0x000f000fu) | u.of_0) - (_Float16)1024.0f; }
__device__ __forceinline__ f16x2 codes_at_4(uint32_t w, const Under &u) { return __builtin_bit_cast(f16x2, (w & 0x00f000f0u) | u.of_4) - (_Float16)64.0f; }
__device__ __forceinline__ f16x2 fma_pair(f16x2 a, f16x2 b, f16x2 c) { return __builtin_elementwise_fma(a, b, c); }

// Whether a block is for float16: s from 2^-13 to 2^11 and lo up to 2^15 in size; where s is 0, lo 0 or from 2^-13.
__device__ __forceinline__ bool for_float16(uint32_t s, uint32_t lo)
{
    lo &= 0x7fffu;
    return s <= 0x6800u && lo <= 0x4700u && (s >= 0x0800u || (s == 0 && (lo == 0 || lo >= 0x3900u)));
}
// What a wave has gathered for its columns.
template <int NB>
struct Gathered {
    f32x4 o[NB / 2][4];   // sum of value * p, values 64 i + 16 p + 4 g + r, times 2^7
    float top;            // exponent p is relative to; at most 8 below the largest so far
    float total;          // sum of the lane's p, times 2^7
    uint32_t far;         // 1: a value of 2^40 or more was among them, o is times 2^-48 more (the same in all lanes)
};

// The values' product in exact codes, for any values: p s_b in NP parts of bfloat16 against the codes.
// Codes count from the middle, c - 8 in even slots and c - 7 in odd ones (numbers of the codes' own form; on the average the
// middle itself), the rest is lo + 8 s or lo + 7 s: with codes from 0 the two sums would grow with the number of slots and nearly
// cancel where a block's values lie around zero, each with roundings of its own.
// A block's lowest number can be as large as a bfloat16.  From 2^40 on p goes to its product small instead of large, and all that is gathered
// is held 2^-48 times: room for 2^31 slots of the largest number, and what is far below that is off by less than 2^-100.
// seen, held: a bit for each of the lane's slots, for the column and for the sequence; looked at where masked.
template <int NB, int NP>
__device__ __forceinline__ void values_by_codes(const uint8_t *at, int lane, bool masked, uint32_t seen, uint32_t held, float (&p)[8], Gathered<NB> &s)
{
    constexpr bool kFineValues = NP == 3;
    const f32x4 zero = kept_zero();
    const int n16 = lane & 15;
    ValuePart<NB> v;
    take_values<NB>(at, lane, v);
    bf16x8 w[NP], middle[NP];
    bool large = false;
    {
        float mid[8];
        for (int i = 0; i < 8; ++i) {
            const float step = (float)__builtin_bit_cast(f16x8, v.own_steps)[i];
            mid[i] = fmaf(step, (i & 1) ? 7.0f : 8.0f, (i & 1) ? __builtin_bit_cast(float, v.lows[i >> 1] & 0xffff0000u) : bf16_to_f32(v.lows[i >> 1]));
        }
        // slots that only some columns see, or none: a NaN there reaches those that see it by p s_b
        if (masked)
            for (int i = 0; i < 8; ++i)
                if (!(held >> i & 1) || !(mid[i] == mid[i])) mid[i] = 0.0f;
        for (int i = 0; i < 8; ++i) large = large || fabsf(mid[i]) >= 0x1p40f;
        split_bf16<NP>(mid, middle);
    }
    const bool small = __builtin_amdgcn_ballot_w64(large) != 0;   // (p is to be)
    if (small && !s.far) {
        s.far = 1;
        for (int i = 0; i < NB / 2; ++i)
            for (int n = 0; n < 4; ++n)
                for (int r = 0; r < 4; ++r) s.o[i][n][r] *= 0x1p-48f;
    }
    const float down = s.far ? 0x1p-48f : 1.0f, lift = small ? 0x1p-48f : 0x1p57f, back = small ? 1.0f : 0x1p-57f * down;
    {
        float lifted[8];
        for (int i = 0; i < 8; ++i) lifted[i] = p[i] * lift;
        split_bf16<NP>(lifted, w);
    }
    f32x4 low = zero;   // what block 4 g + r adds to all its values, times `lift` and the 2^7 of p
    for (int n = 0; n < NP; ++n)
        for (int e = 0; n + e < NP; ++e) low = __builtin_amdgcn_mfma_f32_16x16x32_bf16(middle[n], w[e], low, 0, 0, 0);
    for (int i = 0; i < 8; ++i) p[i] *= 0x1p57f;   // 2^64 with the 2^7 they have: products with codes of 2^-133 stay normal numbers
    for (int b = 0; b < NB; ++b) {
        float ps[8];
        for (int i = 0; i < 8; ++i) ps[i] = fmaf((float)v.steps[b][i], p[i], 0.0f);
        if (masked) {
            const uint32_t those = (uint32_t)kept_here((int)seen);
            for (int i = 0; i < 8; ++i) ps[i] = (those >> i & 1) ? ps[i] : 0.0f;
        }
        split_bf16<NP>(ps, w);
        const u32x4 codes = v.codes[b >> 1];
        const float base = __shfl(low[b & 3], n16 + 16 * (b >> 2), 64) * back;
        for (int n = 0; n < 2; ++n) {
            u32x4 c;
            for (int i = 0; i < 4; ++i) c[i] = code_pairs<kFineValues>(codes[i])[2 * (b & 1) + n];
            const uint32_t back = kFineValues || n ? 0x80708080u : 0x80078008u;
            f32x4 o = zero;   // times 2^-69, 2^-65 where codes stand higher
            for (int e = 0; e < NP; ++e) {
                o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, c), w[e], o, 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u32x4{back, back, back, back}), w[e], o, 0, 0, 0);
            }
            for (int r = 0; r < 4; ++r) s.o[b >> 1][2 * (b & 1) + n][r] += fmaf(o[r], (kFineValues || n ? 0x1p72f : 0x1p76f) * down, base);
        }
    }
}

// The same as a call of its own, for the records of 16-bit caches that need it: in line it would cost the usual record's registers.
template <int NB>
struct Apart {
    float p[8];
    Gathered<NB> sums;
};
template <int NB>
__device__ __attribute__((noinline)) void values_apart(const uint8_t *at, int lane, bool masked, uint32_t seen, uint32_t held, Apart<NB> *x)
{
    values_by_codes<NB, 2>(at, lane, masked, seen, held, x->p, x->sums);
}

// Values as float16 numbers, where all of a record's blocks are for float16 (for 16-bit results): p in one part, two for float16 results.
// A third of the vector instructions of the product in codes, and no more off than the results' own rounding.
template <int NB, int NP>
__device__ __forceinline__ void values_by_numbers(const uint8_t *at, const uint8_t *lows, const Under &under, int lane, const float (&p)[8], Gathered<NB> &s)
{
    const int m = lane & 15, g = lane >> 4;
    f16x8 w[NP];
    for (int i = 0; i < 8; ++i) {
        w[0][i] = (_Float16)p[i];
        if (NP == 2) w[NP - 1][i] = (_Float16)(p[i] - (float)w[0][i]);
    }
    for (int b = 0; b < NB; ++b) {
        const u32x4 codes = *(const u32x4 *)(at + kValueCodes * NB + g * 128 * NB + ((b >> 1) * 16 + m) * 16);
        const u32x4 step = *(const u32x4 *)(at + kValueSteps * NB + (g * NB + b) * 16), low = *(const u32x4 *)(lows + (g * NB + b) * 16);
        for (int n = 0; n < 2; ++n) {
            u32x4 v;
            for (int i = 0; i < 4; ++i) {
                // (copies: a cast of an element in place takes the vector's first one)
                const uint32_t word = (b & 1) ? codes[i] >> 8 : codes[i], sw = step[i], lw = low[i];
                const f16x2 c = n ? codes_at_4(word, under) : codes_at_0(word, under);
                v[i] = __builtin_bit_cast(uint32_t, fma_pair(c, __builtin_bit_cast(f16x2, sw), __builtin_bit_cast(f16x2, lw)));
            }
            f32x4 &o = s.o[b >> 1][2 * (b & 1) + n];
            for (int e = 0; e < NP; ++e) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, v), w[e], o, 0, 0, 0);
        }
    }
}

// One record.  A new reference exponent costs a multiplication of everything gathered, so it is taken only where a weight
// would exceed 2^8 (32-bit sums have room for that); a lane looks at its own eight slots alone, and lanes exchange only then.
template <int NB, int TY>
__device__ __forceinline__ void attend_record(uint8_t *at, const Queries<NB, query_parts<TY>()> &q, int lane, int slot0, int length, bool masked,
                                              const f32x4 &zero, const Under &under, Gathered<NB> &s)
{
    constexpr int NQ = query_parts<TY>();
    f32x4 x[2];
    {
        KeyPart<NB> k;
        take_keys<NB>(at, lane, k);
        record_scores<NB, NQ>(k, q, zero, x);
    }
    // Values for float16?  The lanes look at the blocks together, and leave the lowest numbers as float16 behind the record.
    bool numbers = false;
    if (TY != kF32) {
        bool fine = true;
        for (int i = 0; i < (NB + 3) / 4; ++i) {
            const int pair = 64 * i + lane;
            if (pair < 16 * NB) {
                const uint32_t step = *(const uint32_t *)(at + kValueSteps * NB + pair * 4), low = *(const uint32_t *)(at + kValueLows * NB + pair * 4);
                fine = fine && for_float16(step & 0xffffu, low & 0xffffu) && for_float16(step >> 16, low >> 16);
                const f16x2 l = {(_Float16)bf16_to_f32(low & 0xffffu), (_Float16)__builtin_bit_cast(float, low & 0xffff0000u)};
                *(uint32_t *)(at + record_bytes(NB) + pair * 4) = __builtin_bit_cast(uint32_t, l);
            }
        }
        numbers = __builtin_amdgcn_ballot_w64(!fine) == 0 && !s.far;
        wave_lds_order();
    }
    float p[8], most = kNegInf;
    const float bias = 7.0f - s.top;      // (nothing seen yet: +infinity, which asks for a reference)
    for (int i = 0; i < 8; ++i) p[i] = fmaf(x[i >> 2][i & 3], q.factor, bias);
    uint32_t seen = 0xff, held = 0xff;
    if (masked) {
        const int from = kept_here(slot0);
        seen = held = 0;
        for (int i = 0; i < 8; ++i) {
            const bool sees_it = sees(q, from + i);
            p[i] = sees_it ? p[i] : kNegInf;
            seen |= sees_it ? 1u << i : 0u;
            held |= from + i < length ? 1u << i : 0u;
        }
    }
    for (int i = 0; i < 8; ++i) most = fmaxf(most, p[i]);
    if (__builtin_amdgcn_ballot_w64(most > 15.0f || !(fabsf(bias) < 0x1p16f)) != 0 || q.shift != 0) {
        float e[8];   // (rounded before the reference is taken off: with exponents above 2^16 the product's rounding would count)
        most = kNegInf;
        for (int i = 0; i < 8; ++i) {
            e[i] = x[i >> 2][i & 3] * q.factor;
            if (q.shift != 0) e[i] = ldexpf(e[i], q.shift);
            if (seen >> i & 1) most = fmaxf(most, e[i]);
        }
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        const float now = fmaxf(s.top, most);
        const float shrink = now == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(s.top - now);   // (nothing so far: 0)
        s.top = now;
        s.total *= shrink;
        for (int r = 0; r < 4; ++r)
            for (int i = 0; i < NB / 2; ++i)
                for (int n = 0; n < 4; ++n) s.o[i][n][r] *= shrink;
        for (int i = 0; i < 8; ++i) p[i] = (seen >> i & 1) ? e[i] - now + 7.0f : kNegInf;
    }
    for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(p[i]);
        s.total += p[i];
    }
    if constexpr (TY == kF32) {
        values_by_codes<NB, 3>(at, lane, masked, seen, held, p, s);
    } else if (numbers) {
        values_by_numbers<NB, TY == kF16 ? 2 : 1>(at, at + record_bytes(NB), under, lane, p, s);
    } else {
        Apart<NB> x;
        for (int i = 0; i < 8; ++i) x.p[i] = p[i];
        x.sums = s;
        values_apart<NB>(at, lane, masked, seen, held, &x);
        s = x.sums;
        s.far = (uint32_t)__builtin_amdgcn_readfirstlane((int)s.far);
    }
}

template <int NB, int TY>
__global__ __launch_bounds__(256, NB == 8 || (NB == 4 && TY == kF32) ? 1 : 2) void k_cache_attend(AttendArgs a)
{
    constexpr int NQ = query_parts<TY>(), D = 32 * NB;
    // the waves' records on their way, and afterwards their results
    constexpr int kStage = (int)record_bytes(NB) + 64 * NB, kMem = kAttendWaves * (kColumns * (D + 4) * 4 > kStage ? kColumns * (D + 4) * 4 : kStage);
    __shared__ __align__(16) uint8_t s_mem[kMem];
    float (*s_o)[kColumns][D + 4] = (float (*)[kColumns][D + 4])s_mem;
    __shared__ float s_top[kAttendWaves][kColumns], s_total[kAttendWaves][kColumns];
    // parts outermost: workgroups go to the eight dies in turn, and later parts are the ones that shorter sequences lack (parts
    // innermost: half of the compute units idle on a batch of lengths from a tenth to all of 8192, 144 us when this order took 109)
    const uint32_t units = gridDim.x / (unsigned)a.splits;
    const int split = (int)(blockIdx.x / units);
    const uint32_t unit = blockIdx.x % units;    // (sequence, head, tile)
    const int tile = (int)(unit % (unsigned)a.tiles);
    const int h = (int)(unit / (unsigned)a.tiles % (unsigned)a.c.kv_heads);
    const int s = (int)(unit / (unsigned)a.tiles / (unsigned)a.c.kv_heads);
    if (a.left_over && a.left_over[(unit / (unsigned)a.tiles * (unsigned)a.wide_tiles + (unsigned)(tile / a.tiles_in_wide)) * (unsigned)a.splits + (unsigned)split] == 0) return;
    const Rows rows = rows_of(a.starts, s, a.n_rows);
    const int first = rows.first, count = rows.count < a.max_rows ? rows.count : a.max_rows;
    const int length = sequence_length(a.c, s), slot0 = length - rows.behind;   // slot of the first row (in front of 0: more rows than slots)
    if (tile * kColumns >= count * a.group) return;
    int from, to, all_from, all_to;
    seen_records(a, count, slot0, length, tile, &from, &to);
    seen_by_all(a, count, slot0, length, tile, &all_from, &all_to);
    const int origin = parts_origin(a, count, slot0, length, tile), part_records = records_of_part(a, length, origin);
    const int part_from = origin + split * part_records;
    if (split > 0 && part_from >= to) return;   // (one in front of what the tile sees is written all the same, with nothing in it)
    if (from < part_from) from = part_from;
    if (to > part_from + part_records) to = part_from + part_records;

    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    Queries<NB, NQ> q;
    load_queries<NB, TY, kFine>(a, h, first, count, slot0, length, tile * kColumns + n, g, q);
    Gathered<NB> acc;
    for (int i = 0; i < NB / 2; ++i)
        for (int p = 0; p < 4; ++p) acc.o[i][p] = f32x4{0, 0, 0, 0};
    acc.top = kNegInf;
    acc.total = 0.0f;
    acc.far = 0;
    uint8_t *stage = s_mem + wave * kStage;
    const f32x4 zero = kept_zero();
    const Under under = under_codes();
    RawRecord<NB> raw;
    int it = from + wave;
    PagesAhead pages = {0, it, kAttendWaves, to};
    const uint8_t *rec = pages.next(a.c, s, h, it, lane, NB);
    if (rec) load_record<NB>(rec, lane, raw);
    while (it < to) {
        const int next = it + kAttendWaves;
        const uint8_t *next_rec = pages.next(a.c, s, h, next, lane, NB);
        if (rec) lay_record<NB>(stage, lane, raw);
        if (next_rec) load_record<NB>(next_rec, lane, raw);
        if (rec) {
            attend_record<NB, TY>(stage, q, lane, it * kRecordSlots + 8 * g, length,
                                        it * kRecordSlots < all_from || (it + 1) * kRecordSlots > all_to, zero, under, acc);
        }
        it = next;
        rec = next_rec;
    }
    __syncthreads();
    float total = acc.total;
    const float top = acc.top;

    // the waves' results meet in LDS, as means: no sum of values is larger than they are
    total += __shfl_xor(total, 16, 64);
    total += __shfl_xor(total, 32, 64);
    const float share = total == 0.0f ? 0.0f : 1.0f / total, raise = acc.far ? 0x1p48f : 1.0f;   // (both times 2^7)
    if (g == 0) {
        s_top[wave][n] = top;
        s_total[wave][n] = total * 0x1p-7f;
    }
    for (int i = 0; i < NB / 2; ++i) {
        for (int p = 0; p < 4; ++p) {
            f32x4 v;
            for (int r = 0; r < 4; ++r) v[r] = acc.o[i][p][r] * share * raise;
            *(f32x4 *)&s_o[wave][n][64 * i + 16 * p + 4 * g] = v;
        }
    }
    __syncthreads();
    const int column = threadIdx.x >> 4, part = threadIdx.x & 15;
    float all = kNegInf;
    for (int w = 0; w < kAttendWaves; ++w) all = fmaxf(all, s_top[w][column]);
    float sum = 0.0f, of[kAttendWaves], x[2 * NB];
    for (int i = 0; i < 2 * NB; ++i) x[i] = 0.0f;
    for (int w = 0; w < kAttendWaves; ++w) {
        // (a wave that saw nothing holds zeros; with a NaN among what it saw its total is one)
        of[w] = s_total[w][column] * (all == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(s_top[w][column] - all));
        sum += of[w];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    for (int w = 0; w < kAttendWaves; ++w)
        for (int i = 0; i < 2 * NB; ++i) x[i] = fmaf(s_o[w][column][part * 2 * NB + i], of[w] * inv, x[i]);
    if (tile * kColumns + column >= count * a.group) return;
    if (a.splits > 1) {
        const uint64_t at = ((uint64_t)unit * kColumns + (uint32_t)column) * (uint32_t)a.splits + (uint32_t)split;
        store_run<2 * NB, kF32>(a.partial, at * D + (uint32_t)(part * 2 * NB), x);
        if (part == 0) {
            a.partial_sums[2 * at] = all;
            a.partial_sums[2 * at + 1] = sum;
        }
    } else {
        write_result<NB, TY>(a, h, first, tile * kColumns + column, part, all, sum, x);
    }
}

// ---------------------------------------------------------------- attention of many rows
//
// With more columns than one tile the records are unpacked once for all of them.  A workgroup of W waves takes 16 CT W columns; all threads
// together unpack records into LDS, ahead of the products, as float16 numbers: values in one part, keys in two (22 bits: scores are exponents,
// and lse is a 32-bit result; where a second part is below the normal range it still holds the places of s, which are 2^-23 and more).  That
// rounding, and the one of p to float16 (in two parts for float16 results), need numbers within float16's range.  A record with a NaN, or with
// blocks too large or too small for it, is not for this kernel: the workgroup notes so, and k_cache_attend does its columns afterwards.
//
// Vector and matrix instructions about balance: for a record and 16 columns 8 multiply-adds, 8 exponentials (four times the cost
// of others) and 25 more against 24 products of 16 cycles; a wave's share of the unpacking, which all 32 workgroups of a sequence and head do
// again, of finding records and keeping step is about 150 for its two tiles.  (With whole codes as keys, their scores scaled in 32 bits as
// above, it was 64 more vector instructions for 8 products less, and 1410 us when this took 1190.)
//
// 2 x 2048 rows of 32 heads over 10007 slots, 8 heads of 128 values, bfloat16: 1050 us, 574 TFLOP/s of the two products (603 GFLOP), in a row of
// calls; the first ones after other work, at a lower clock, take 1190.  The matrix unit is busy 34 % of it (a third of that with the keys'
// second parts), vector instructions 48 %, LDS 24 %; two waves for each SIMD, which a barrier for every two records keeps in step, do not
// put them beside each other fully.  Keys in one part: a fifth less, but lse off by 1e-4.
template <int NB>
struct WideRecord {
    static constexpr uint32_t kRest = 2048u * NB, kValues = 4096u * NB, kBytes = 6144u * NB;   // keys from 0, their second parts
    // steps and lowest numbers, as a record has them from kKeySteps on
    static constexpr uint32_t kSides = 256u * NB, kVSteps = 64u * NB, kKLows = 128u * NB, kVLows = 192u * NB;
    static constexpr int kPerStep = NB == 8 ? 1 : 2;   // records of a step: two steps fit into LDS
};

// A unit of unpacking work, a wave's: keys of blocks 2 half, 2 half + 1 of sixteen slots (unit = T * NB / 2 + half), or values 64 i + 32 half .. + 31
// (unit = NB + 2 i + half).
template <int NB>
__device__ __forceinline__ u32x4 load_unit(const uint8_t *rec, int unit, int lane)
{
    const int m = lane & 15, g = lane >> 4;
    u32x4 codes = {0, 0, 0, 0};
    if (unit < NB) {
        const int T = unit / (NB / 2), half = unit % (NB / 2), key = 8 * (m >> 2) + 4 * T + (m & 3);
        const u32x2 w = *(const u32x2 *)(rec + key * 16 * NB + g * 4 * NB + half * 8);
        codes[0] = w[0];
        codes[1] = w[1];
    } else {
        codes = *(const u32x4 *)(rec + kValueCodes * NB + g * 128 * NB + (((unit - NB) >> 1) * 16 + m) * 16);
    }
    return codes;
}
// Halves of a word that belong to slots in front of `left`: slots 8 g + 2 n and 8 g + 2 n + 1.
__device__ __forceinline__ uint32_t held_halves(int g, int n, int left)
{
    return (8 * g + 2 * n < left ? 0x0000ffffu : 0u) | (8 * g + 2 * n + 1 < left ? 0xffff0000u : 0u);
}
// Lays a unit into `at`; sides: the record's; left: slots of the record that the sequence holds (what lies behind counts for nothing).
// False where a key's block is not for float16.
template <int NB>
__device__ __forceinline__ bool lay_unit(uint8_t *at, const uint8_t *sides, const Under &under, int unit, int lane, const u32x4 &codes, int left)
{
    const int m = lane & 15, g = lane >> 4;
    if (unit < NB) {
        const int T = unit / (NB / 2), half = unit % (NB / 2), key = 8 * (m >> 2) + 4 * T + (m & 3);
        const uint32_t lows = *(const uint32_t *)(sides + WideRecord<NB>::kKLows + (key * NB + 2 * half) * 2);
        bool fine = true;
        for (int n = 0; n < 2; ++n) {
            const uint32_t step = *(const uint16_t *)(sides + ((key >> 3) * NB + 2 * half + n) * 16 + (key & 7) * 2);
            const uint32_t w = codes[n], high = w >> 8;
            const float s = f16_to_f32(step), lo = n ? __builtin_bit_cast(float, lows & 0xffff0000u) : bf16_to_f32(lows & 0xffffu);
            fine = fine && for_float16(step, (lows >> (16 * n)) & 0xffffu);
            const f16x2 c[4] = {codes_at_0(w, under), codes_at_4(w, under), codes_at_0(high, under), codes_at_4(high, under)};
            u32x4 first, rest;
            for (int i = 0; i < 4; ++i) {
                const float x = fmaf((float)c[i][0], s, lo), y = fmaf((float)c[i][1], s, lo);
                const f16x2 k = {(_Float16)x, (_Float16)y};
                const f16x2 r = {(_Float16)fmaf((float)k[0], under.minus, x), (_Float16)fmaf((float)k[1], under.minus, y)};   // (exact, one instruction each)
                first[i] = __builtin_bit_cast(uint32_t, k);
                rest[i] = __builtin_bit_cast(uint32_t, r);
            }
            const int place = ((T * NB + 2 * half + n) * 64 + lane) * 16;
            *(u32x4 *)(at + place) = first;
            *(u32x4 *)(at + WideRecord<NB>::kRest + place) = rest;
        }
        return fine || key >= left;
    }
    const int i = (unit - NB) >> 1, half = (unit - NB) & 1;
    u32x4 steps = *(const u32x4 *)(sides + WideRecord<NB>::kVSteps + (g * NB + unit - NB) * 16);
    u32x4 lows = *(const u32x4 *)(sides + WideRecord<NB>::kVLows + (g * NB + unit - NB) * 16);
    if (left < kRecordSlots) {
        for (int n = 0; n < 4; ++n) {
            steps[n] &= held_halves(g, n, left);
            lows[n] &= held_halves(g, n, left);
        }
    }
    u32x4 out[2];
    for (int n = 0; n < 4; ++n) {
        const uint32_t pair = steps[n];   // (a cast of the element in place takes the vector's first one)
        const f16x2 s = __builtin_bit_cast(f16x2, pair);
        const f16x2 lo = {(_Float16)bf16_to_f32(lows[n] & 0xffffu), (_Float16)__builtin_bit_cast(float, lows[n] & 0xffff0000u)};
        const uint32_t w = half ? codes[n] >> 8 : codes[n];
        out[0][n] = __builtin_bit_cast(uint32_t, fma_pair(codes_at_0(w, under), s, lo));
        out[1][n] = __builtin_bit_cast(uint32_t, fma_pair(codes_at_4(w, under), s, lo));
    }
    for (int n = 0; n < 2; ++n) *(u32x4 *)(at + WideRecord<NB>::kValues + ((i * 4 + 2 * half + n) * 64 + lane) * 16) = out[n];
    return true;
}
template <int NB>
struct WideGathered {
    f32x4 o[NB / 2][4];   // sum of value * p, values 64 i + 16 p + 4 g + r
    float top;            // exponent p is relative to, one that 32 bits hold: about 7 below the largest so far, at most 15
    float total;          // sum of the lane's p
};

// The CT tiles of a wave together: what is read from LDS serves all of them.
template <int NB, int CT, int NP>
__device__ __forceinline__ void attend_wide(const uint8_t *at, const Queries<NB, 1> (&q)[CT], int lane, int slot0, bool masked, const f32x4 &zero, WideGathered<NB> (&s)[CT])
{
    f32x4 e[CT][2];   // exponents of slots slot0 + 4 T ..
    // Operands are read kAhead products in front of their own: left to itself the compiler reads each where it is needed, to save registers, and a
    // wave then waits for LDS in front of every pair of products (1190 us instead of 1070 then, at 2 x 2048 rows over 10007 slots).
    constexpr int kAhead = 3;
    static_assert(4 * NB % (kAhead + 1) == 0, "values follow keys in the ring");
    f16x8 ring[kAhead + 1];
    auto read_keys = [&](int n) __attribute__((always_inline)) {   // block n / 4: second parts of both T, then first ones
        return *(const f16x8 *)(at + ((n & 2) ? 0u : WideRecord<NB>::kRest) + (((n & 1) * NB + (n >> 2)) * 64 + lane) * 16);
    };
    auto read_values = [&](int n) __attribute__((always_inline)) { return *(const f16x8 *)(at + WideRecord<NB>::kValues + (n * 64 + lane) * 16); };
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ring[n] = read_keys(n);
#pragma unroll
    for (int n = 0; n < 4 * NB; ++n) {
        ring[(n + kAhead) % (kAhead + 1)] = n + kAhead < 4 * NB ? read_keys(n + kAhead) : read_values(n + kAhead - 4 * NB);
        __builtin_amdgcn_sched_barrier(0);
        for (int t = 0; t < CT; ++t)
            e[t][n & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[n % (kAhead + 1)], q[t].q[n >> 2][0], n < 2 ? zero : e[t][n & 1], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
    bool higher = false;
    for (int t = 0; t < CT; ++t) {
        for (int i = 0; i < 8; ++i) e[t][i >> 2][i & 3] *= q[t].factor;
        if (masked) {
            const int from = kept_here(slot0);
            for (int i = 0; i < 8; ++i) e[t][i >> 2][i & 3] = sees(q[t], from + i) ? e[t][i >> 2][i & 3] : kNegInf;
        }
        float most = kNegInf;
        for (int i = 0; i < 8; ++i) most = fmaxf(most, e[t][i >> 2][i & 3]);
        // (p up to 2^15: float16 has room for that.  The difference, not a sum with top: numbers of 2^25 and more are whole fours and further apart)
        higher = higher || most - s[t].top > 15.0f;
    }
    if (__builtin_amdgcn_ballot_w64(higher) != 0) {
        for (int t = 0; t < CT; ++t) {
            float most = kNegInf;
            for (int i = 0; i < 8; ++i) most = fmaxf(most, e[t][i >> 2][i & 3]);
            most = fmaxf(most, __shfl_xor(most, 16, 64));
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            const float now = fmaxf(s[t].top, most - 7.0f);
            const float shrink = now == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(s[t].top - now);
            s[t].top = now;
            s[t].total *= shrink;
            for (int i = 0; i < NB / 2; ++i)
                for (int n = 0; n < 4; ++n)
                    for (int r = 0; r < 4; ++r) s[t].o[i][n][r] *= shrink;
        }
    }
    f16x8 w[CT][NP];
    for (int t = 0; t < CT; ++t) {
        const float top = s[t].top == kNegInf ? 0.0f : s[t].top;
        for (int i = 0; i < 8; ++i) {
            const float p = __builtin_amdgcn_exp2f(e[t][i >> 2][i & 3] - top);
            s[t].total += p;
            w[t][0][i] = (_Float16)p;
            if (NP == 2) w[t][NP - 1][i] = (_Float16)(p - (float)w[t][0][i]);
        }
    }
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n) {
        if (n + kAhead < 2 * NB) ring[(n + kAhead) % (kAhead + 1)] = read_values(n + kAhead);
        __builtin_amdgcn_sched_barrier(0);
        for (int t = 0; t < CT; ++t)
            for (int k = 0; k < NP; ++k)
                s[t].o[n >> 2][n & 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[n % (kAhead + 1)], w[t][k], s[t].o[n >> 2][n & 3], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <int NB, int TY, int W, int CT>
__global__ __launch_bounds__(64 * W, W / 4) void k_cache_attend_rows(AttendArgs a)
{
    constexpr int NP = TY == kF16 ? 2 : 1, D = 32 * NB, kWide = kColumns * CT * W;
    constexpr int kPer = WideRecord<NB>::kPerStep, kUnits = (2 * kPer * NB + W - 1) / W;   // records of a step, units of a wave
    __shared__ __align__(16) uint8_t s_mem[2][kPer][WideRecord<NB>::kBytes];
    __shared__ __align__(16) uint8_t s_sides[2][kPer][WideRecord<NB>::kSides];
    __shared__ uint32_t s_bad;
    const uint32_t units = gridDim.x / (unsigned)a.splits;
    const int split = (int)(blockIdx.x / units);
    const uint32_t unit = blockIdx.x % units;    // (sequence, head, wide tile)
    const int wide = (int)(unit % (unsigned)a.wide_tiles);
    const int h = (int)(unit / (unsigned)a.wide_tiles % (unsigned)a.c.kv_heads);
    const int s = (int)(unit / (unsigned)a.wide_tiles / (unsigned)a.c.kv_heads);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    if (threadIdx.x == 0) s_bad = 0;
    const Rows rows = rows_of(a.starts, s, a.n_rows);
    const int first = rows.first, count = rows.count < a.max_rows ? rows.count : a.max_rows;
    const int length = sequence_length(a.c, s), slot0 = length - rows.behind;   // slot of the first row (in front of 0: more rows than slots)
    if (wide * kWide >= count * a.group) return;
    int from, to;
    seen_records(a, count, slot0, length, wide, &from, &to, kWide);
    const int part_records = records_of_part(a, length, from);
    from += split * part_records;
    if (to > from + part_records) to = from + part_records;

    Queries<NB, 1> q[CT];
    WideGathered<NB> acc[CT];
    const int wave_tile = wide * W + wave;   // of 16 CT columns
    int own_from = 0, own_to = 0, all_from = 0, all_to = 0;   // (nothing, where the wave's columns are not there)
    if (wave_tile * kColumns * CT < count * a.group) {
        seen_records(a, count, slot0, length, wave_tile, &own_from, &own_to, kColumns * CT);
        seen_by_all<kColumns * CT>(a, count, slot0, length, wave_tile, &all_from, &all_to);
    }
    for (int t = 0; t < CT; ++t) {
        load_queries<NB, TY, kWhole>(a, h, first, count, slot0, length, (wave_tile * CT + t) * kColumns + n, g, q[t]);
        acc[t].top = kNegInf;
        acc[t].total = 0.0f;
        for (int i = 0; i < NB / 2; ++i)
            for (int p = 0; p < 4; ++p) acc[t].o[i][p] = f32x4{0, 0, 0, 0};
    }

    // Codes are unpacked a step ahead of the products, and loaded a step ahead of that, the sides another.  Of a step's two records, keys
    // of the one and values of the other fall to the same wave.
    const int steps = (to - from + kPer - 1) / kPer;
    struct Pair {
        const uint8_t *first, *second;
        __device__ __forceinline__ const uint8_t *operator[](int r) const { return r ? second : first; }   // (an array would go to memory)
    };
    PagesAhead pages = {0, from, 1, to};
    auto find = [&](int j) __attribute__((always_inline)) {   // (of j = 0, 1, .. in turn)
        const int it = from + kPer * j;
        const uint8_t *first = pages.next(a.c, s, h, it, lane, NB);
        return Pair{first, kPer > 1 ? pages.next(a.c, s, h, it + 1, lane, NB) : nullptr};
    };
    u32x4 raw[kUnits], side = {0, 0, 0, 0};
    const int side_rec = (int)threadIdx.x / (16 * NB), side_piece = (int)threadIdx.x % (16 * NB);
    static_assert(64 * W >= 16 * kPer * NB, "a piece of the records' sides for every thread");
    auto load_sides = [&](const Pair &p) __attribute__((always_inline)) {
        const uint8_t *rec = p[side_rec];
        if (side_rec < kPer && rec) side = *(const u32x4 *)(rec + kKeySteps * NB + side_piece * 16);
    };
    auto lay_sides = [&](int j) __attribute__((always_inline)) {
        if (side_rec < kPer) *(u32x4 *)&s_sides[j & 1][side_rec][side_piece * 16] = side;
    };
    auto load_codes = [&](const Pair &p) __attribute__((always_inline)) {
        for (int k = 0; k < kUnits; ++k) {
            const int u = wave + k * W, r = u / (2 * NB);
            const uint8_t *rec = p[r];
            if (u < 2 * kPer * NB && rec) raw[k] = load_unit<NB>(rec, (u + r * NB) % (2 * NB), lane);
        }
    };
    bool fine = true;   // (queries that need a shift are left to the other kernel too)
    for (int t = 0; t < CT; ++t) fine = fine && q[t].shift == 0;
    const Under under = under_codes();
    auto lay_codes = [&](int j, const Pair &p) __attribute__((always_inline)) {
        for (int k = 0; k < kUnits; ++k) {
            const int u = wave + k * W, r = u / (2 * NB);
            if (u < 2 * kPer * NB && p[r])
                fine = lay_unit<NB>(s_mem[j & 1][r], s_sides[j & 1][r], under, (u + r * NB) % (2 * NB), lane, raw[k], length - (from + kPer * j + r) * kRecordSlots) && fine;
        }
        // the values' blocks, one a thread
        for (int k = 0; k < (32 * kPer * NB + 64 * W - 1) / (64 * W); ++k) {
            const int n = (int)threadIdx.x + 64 * W * k, r = n / (32 * NB), block = n % (32 * NB), slot = block / (8 * NB) * 8 + block % 8;
            if (r < kPer && p[r] && slot < length - (from + kPer * j + r) * kRecordSlots)
                fine = fine && for_float16(*(const uint16_t *)&s_sides[j & 1][r][WideRecord<NB>::kVSteps + block * 2],
                                           *(const uint16_t *)&s_sides[j & 1][r][WideRecord<NB>::kVLows + block * 2]);
        }
    };
    const f32x4 zero = kept_zero();
    Pair now = find(0), next = find(1), later = find(2);
    load_sides(now);
    load_codes(now);
    lay_sides(0);
    load_sides(next);
    __syncthreads();
    lay_codes(0, now);
    lay_sides(1);
    load_codes(next);
    load_sides(later);
    for (int j = 0; j < steps; ++j) {
        __syncthreads();
        lay_codes(j + 1, next);
        lay_sides(j);   // (of step j + 2: those of step j are done with)
        const Pair last = find(j + 3);
        load_codes(later);
        load_sides(last);
#pragma unroll 1
        for (int r = 0; r < kPer; ++r) {
            const int at = from + kPer * j + r;
            if (now[r] && at >= own_from && at < own_to)
                attend_wide<NB, CT, NP>(s_mem[j & 1][r], q, lane, at * kRecordSlots + 8 * g, at * kRecordSlots < all_from || (at + 1) * kRecordSlots > all_to, zero, acc);
        }
        now = next;
        next = later;
        later = last;
    }
    if (!fine) s_bad = 1;
    __syncthreads();
    // (the kernel's first store: behind one, the table would no longer be read by scalar loads)
    const bool left_over = s_bad != 0;
    if (threadIdx.x == 0) a.left_over[unit * (unsigned)a.splits + (unsigned)split] = left_over ? 1 : 0;
    if (left_over) return;
    for (int t = 0; t < CT; ++t) {
        const int tile = wave_tile * CT + t, column = tile * kColumns + n;
        float total = acc[t].total;
        total += __shfl_xor(total, 16, 64);
        total += __shfl_xor(total, 32, 64);
        if (column >= count * a.group) continue;
        const int row = column / a.group, head = column - row * a.group;
        const uint64_t line = (uint64_t)(first + row) * a.out_row_stride + (uint64_t)(h * a.group + head) * a.out_head_stride;
        const uint64_t place = (((uint64_t)(unit / (unsigned)a.wide_tiles) * (unsigned)a.tiles + (unsigned)tile) * kColumns + (unsigned)n) * (unsigned)a.splits + (unsigned)split;
        const float scale = total == 0.0f ? 0.0f : 1.0f / total;
        for (int i = 0; i < NB / 2; ++i) {
            for (int p = 0; p < 4; ++p) {
                float v[4];
                for (int r = 0; r < 4; ++r) v[r] = acc[t].o[i][p][r] * scale;
                const uint64_t at = (uint64_t)(64 * i + 16 * p + 4 * g);
                if (a.splits > 1) store_run<4, kF32>(a.partial, place * D + at, v);
                else store_run<4, TY>(a.out, line + at, v);
            }
        }
        if (g == 0 && a.splits > 1) {
            a.partial_sums[2 * place] = acc[t].top;
            a.partial_sums[2 * place + 1] = total;
        } else if (g == 0 && a.lse) {
            a.lse[(uint64_t)(first + row) * ((uint64_t)a.c.kv_heads * a.group) + (uint64_t)(h * a.group + head)] =
                total == 0.0f ? kNegInf : (acc[t].top + __builtin_amdgcn_logf(total)) * kLn2;
        }
    }
}

// Joins the parts of a column, means and sums of weights: a workgroup each, its waves taking parts in turn, 2 NB of the column's values a lane (the
// waves' other lanes further parts).
template <int NB, int TY>
__global__ __launch_bounds__(256) void k_cache_join(AttendArgs a)
{
    constexpr int D = 32 * NB, kStrands = 16;   // 16 lanes hold a column
    __shared__ float s_sum[kStrands][D + 4];
    __shared__ float s_total[kStrands], s_top[kStrands];
    const int column = (int)(blockIdx.x % (unsigned)a.columns);
    const uint32_t unit = blockIdx.x / (unsigned)a.columns;
    const int tile = (int)(unit % (unsigned)a.tiles);
    const int h = (int)(unit / (unsigned)a.tiles % (unsigned)a.c.kv_heads);
    const int s = (int)(unit / (unsigned)a.tiles / (unsigned)a.c.kv_heads);
    const Rows rows = rows_of(a.starts, s, a.n_rows);
    const int first = rows.first, count = rows.count < a.max_rows ? rows.count : a.max_rows;
    const int length = sequence_length(a.c, s), slot0 = length - rows.behind;   // slot of the first row (in front of 0: more rows than slots)
    if (tile * kColumns + column >= count * a.group) return;
    int from, to;
    seen_records(a, count, slot0, length, tile, &from, &to);
    const int origin = parts_origin(a, count, slot0, length, tile), part_records = records_of_part(a, length, origin);
    int parts = (to - origin + part_records - 1) / part_records;
    if (parts < 1) parts = 1;
    if (parts > a.splits) parts = a.splits;
    const uint64_t at = ((uint64_t)unit * kColumns + (uint32_t)column) * (uint32_t)a.splits;
    const int strand = threadIdx.x >> 4, place = threadIdx.x & 15;
    float x[2 * NB], total = 0.0f, top = kNegInf;
    for (int i = 0; i < 2 * NB; ++i) x[i] = 0.0f;
    for (int k = strand; k < parts; k += kStrands) top = fmaxf(top, a.partial_sums[2 * (at + (uint32_t)k)]);
    if (place == 0) s_top[strand] = top;
    __syncthreads();
    for (int k = 0; k < kStrands; ++k) top = fmaxf(top, s_top[k]);
    auto weight = [&](int k) __attribute__((always_inline)) {
        const uint64_t p = at + (uint32_t)k;
        return a.partial_sums[2 * p + 1] * (top == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(a.partial_sums[2 * p] - top));
    };
    float own = 0.0f;
    for (int k = strand; k < parts; k += kStrands) own += weight(k);
    if (place == 0) s_total[strand] = own;
    __syncthreads();
    for (int k = 0; k < kStrands; ++k) total += s_total[k];
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    for (int k = strand; k < parts; k += kStrands) {
        float y[2 * NB];
        load_run<2 * NB>(a.partial, (at + (uint32_t)k) * D + (uint32_t)(place * 2 * NB), y);
        const float f = weight(k) * inv;
        for (int i = 0; i < 2 * NB; ++i) x[i] = fmaf(y[i], f, x[i]);
    }
    for (int i = 0; i < 2 * NB; ++i) s_sum[strand][place * 2 * NB + i] = x[i];
    __syncthreads();
    if (strand != 0) return;
    const int strands = parts < kStrands ? parts : kStrands;
    for (int k = 1; k < strands; ++k)
        for (int i = 0; i < 2 * NB; ++i) x[i] += s_sum[k][place * 2 * NB + i];
    write_result<NB, TY>(a, h, first, tile * kColumns + column, place, top, total, x);
}

// The attention each slot received.  A wave holds two records' keys in LDS (the next two on their way) and goes over all columns of their
// sequence and head, computing the scores again, and adds in the columns' order.  (Keeping the scores of the attention kernel instead
// would write and read 4 bytes for every column and slot: with four columns 32 bytes a slot, with eight 64, against the 80 of the keys of
// 128 values.)  Between reading a cache's keys and computing: 25000 records and four columns take 30 us, six more where a workgroup ends after
// eight records (its start - positions, page, queries - costs as much as four).  For many rows it is far from its products' time: 2 x 2048 rows of
// 32 heads on 10007 slots take 2.0 ms, as codes are unpacked, and scores scaled block by block, again for every 16 columns.
// Four or eight records held: the same for few columns, 8 and 20 % slower for many (fewer waves fit).
constexpr int kHeldRecords = 2, kWeightsPerUnit = 2;   // workgroups for a compute unit, where there are batches for more

// The keys of a record: codes, steps, lowest numbers, in 16-byte pieces lane, lane + 64, ..
template <int NB>
struct RawKeys {
    static constexpr int kPieces = (40 * NB + 63) / 64;
    u32x4 piece[kPieces];
};
template <int NB>
__device__ __forceinline__ void load_raw_keys(const uint8_t *rec, int lane, RawKeys<NB> &raw)
{
    for (int i = 0; i < RawKeys<NB>::kPieces; ++i) {
        const int u = 64 * i + lane;
        if (u < 40 * NB) raw.piece[i] = *(const u32x4 *)(rec + (u < 32 * NB ? u : (u < 36 * NB ? u + 32 * NB : u + 36 * NB)) * 16);
    }
}
template <int NB>
__device__ __forceinline__ void lay_keys(uint8_t *at, int lane, const RawKeys<NB> &raw)
{
    for (int i = 0; i < RawKeys<NB>::kPieces; ++i) {
        const int u = 64 * i + lane;
        if (u < 40 * NB) *(u32x4 *)(at + (u < 32 * NB ? key_place<NB>(u) : u) * 16) = raw.piece[i];
    }
}

// v[i] summed over the sixteen lanes of a row: lane n gets that of i = 4 (n & 1) + (n & 2) + (n >> 2 & 1).
__device__ __forceinline__ float sum_over_row(const float *v, int n)
{
    float a[4], b[2];
    for (int i = 0; i < 4; ++i) {
        const float give = (n & 1) ? v[i] : v[4 + i], keep = (n & 1) ? v[4 + i] : v[i];
        a[i] = keep + __shfl_xor(give, 1, 64);
    }
    for (int i = 0; i < 2; ++i) {
        const float give = (n & 2) ? a[i] : a[2 + i], keep = (n & 2) ? a[2 + i] : a[i];
        b[i] = keep + __shfl_xor(give, 2, 64);
    }
    const float give = (n & 4) ? b[0] : b[1], keep = (n & 4) ? b[1] : b[0];
    const float c = keep + __shfl_xor(give, 4, 64);
    return c + __shfl_xor(c, 8, 64);
}

template <int NB, int TY>
__global__ __launch_bounds__(256, NB == 8 || TY == kF32 ? 1 : 3) void k_cache_weights(AttendArgs a, int records, int batches)
{
    constexpr int NQ = query_parts<TY>(), kBytes = 640 * NB, kBatch = kAttendWaves * kHeldRecords;
    __shared__ __align__(16) uint8_t s_mem[kAttendWaves][kHeldRecords][kBytes];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const uint32_t groups = ((uint32_t)records + (uint32_t)(kBatch * batches) - 1) / (uint32_t)(kBatch * batches);
    const int unit = (int)(blockIdx.x / groups), h = unit % a.c.kv_heads, s = unit / a.c.kv_heads;
    const int begin = (int)(blockIdx.x % groups) * kBatch * batches + wave * kHeldRecords;
    const Rows rows = rows_of(a.starts, s, a.n_rows);
    const int first = rows.first, count = rows.count < a.max_rows ? rows.count : a.max_rows;
    const int length = sequence_length(a.c, s), slot0 = length - rows.behind;   // slot of the first row (in front of 0: more rows than slots)
    const uint32_t own = (uint32_t)(8 * g + 4 * (n & 1) + (n & 2) + ((n >> 2) & 1));   // the lane's slot of a record's weights
    // (records are counted, not slots: the last batch may reach past the last slot, and with it past 2^31)
    const int held = (int)(((uint32_t)length + 31) >> 5);
    const uint64_t line = ((uint64_t)s * a.c.kv_heads + h) * a.weight_stride;
    RawKeys<NB> raw[kHeldRecords];
    float before[kHeldRecords];
    uint32_t coming = 0;   // a bit for each record that is there
    auto load_batch = [&](int it0) __attribute__((always_inline)) {
        coming = 0;
        for (int k = 0; k < kHeldRecords; ++k) {
            const uint8_t *rec = it0 + k < held ? record_of(a.c, a.c.table, a.c.table_stride, s, h, (it0 + k) * kRecordSlots, NB) : nullptr;
            if (!rec) continue;
            coming |= 1u << k;
            load_raw_keys<NB>(rec, lane, raw[k]);
        }
        for (int k = 0; k < kHeldRecords; ++k) {
            const uint32_t slot = (uint32_t)(it0 + k) * kRecordSlots + own;
            before[k] = a.prior && n < 8 && slot < (uint32_t)length ? a.prior[line + (uint64_t)slot] : 0.0f;
        }
    };
    load_batch(begin);
    int tile = -1;
    Queries<NB, NQ> q;
    // the column's lse as an exponent, negative, short of up = 2^shift; one: a NaN where lse is one
    float less = 0.0f, up = 1.0f, one = 1.0f;
    for (int it0 = begin; it0 < begin + kBatch * batches && it0 < held; it0 += kBatch) {
        // the columns of the next tile that sees any of the records (a single tile stays)
        int next = -1;
        auto next_tile = [&]() __attribute__((always_inline)) {
            int from = 0, to = 0;
            do {
                if (++next * kColumns >= count * a.group) return false;
                seen_records(a, count, slot0, length, next, &from, &to);
            } while (it0 + kHeldRecords <= from || it0 >= to);
            if (next == tile) return true;
            tile = next;
            const int column = tile * kColumns + n;
            load_queries<NB, TY, kFine>(a, h, first, count, slot0, length, column, g, q);
            less = 0.0f;
            if (column < count * a.group) {
                const int row = column / a.group, head = column - row * a.group;
                less = a.lse[(uint64_t)(first + row) * ((uint64_t)a.c.kv_heads * a.group) + (uint64_t)(h * a.group + head)] * -kLog2e;
            }
            less = ldexpf(less, -q.shift);
            up = ldexpf(1.0f, q.shift);
            one = fmaf(less, 0.0f, 1.0f);
            return true;
        };
        bool more = next_tile();
        const uint32_t there = coming;
        float sum[kHeldRecords][8], prior[kHeldRecords];
        for (int k = 0; k < kHeldRecords; ++k) {
            if (there >> k & 1) lay_keys<NB>(s_mem[wave][k], lane, raw[k]);
            prior[k] = before[k];
            for (int i = 0; i < 8; ++i) sum[k][i] = 0.0f;
        }
        wave_lds_order();
        if (it0 + kBatch < begin + kBatch * batches) load_batch(it0 + kBatch);
        for (; more; more = next_tile()) {
            for (int k = 0; k < kHeldRecords; ++k) {
                if (!(there >> k & 1)) continue;
                KeyPart<NB> keys;
                take_keys<NB, 512, 576>(s_mem[wave][k], lane, keys);
                f32x4 x[2];
                record_scores<NB, NQ>(keys, q, f32x4{0, 0, 0, 0}, x);
                const int from_slot = (it0 + k) * kRecordSlots + 8 * g;
                for (int i = 0; i < 8; ++i) {
                    // (between 0 and 1: an output modifier of the power's instruction, which makes a NaN a 0)
                    const float w = fminf(fmaxf(__builtin_amdgcn_exp2f(fmaf(x[i >> 2][i & 3], q.factor, less) * up), 0.0f), 1.0f);
                    if (sees(q, from_slot + i)) sum[k][i] = fmaf(w, one, sum[k][i]);
                }
            }
        }
        for (int k = 0; k < kHeldRecords; ++k) {
            const float all = sum_over_row(sum[k], n);
            const uint32_t slot = (uint32_t)(it0 + k) * kRecordSlots + own;
            if (n < 8 && slot < (uint32_t)length) a.weights[line + (uint64_t)slot] = prior[k] + all;
        }
        wave_lds_order();
    }
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

typedef float f32x4_of_4 __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kSelectThreads = 1024, kSelectEach = 16, kSelectTile = kSelectThreads * kSelectEach, kSelectBins = 2048;
// Exclusive prefix of a count per thread over the workgroup.
__device__ __forceinline__ uint32_t block_prefix(uint32_t mine, uint32_t *sums, uint32_t *all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = mine;
    // inside rows of sixteen lanes, then the rows' last lanes on into the rows behind
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
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

// A workgroup per sequence and head.  A thread holds sixteen neighbouring weights, so that ranks need one prefix sum over the threads; sequences
// of up to 16384 slots are read once, longer ones once for each of the passes.  The key of the last weight to stay is found 11,
// 11 and 10 bits at a time from the top: counts in LDS, then a prefix sum from the largest bin down.
// Bound by the passes' barriers and instructions, not by memory: 128 heads of up to 16384 slots take 16 us, 8 of 1100 slots 10; ten of 31995,
// whose weights are read once a pass, 40.
__global__ __launch_bounds__(kSelectThreads) void k_cache_select(EvictArgs a)
{
    __shared__ uint32_t s_bins[kSelectBins];
    __shared__ uint32_t s_sums[kSelectThreads / 64];
    __shared__ uint32_t s_found[2];
    const int h = (int)(blockIdx.x % (unsigned)a.c.kv_heads), s = (int)(blockIdx.x / (unsigned)a.c.kv_heads);
    // (slots without a sign: tiles reach past the last slot, and with it past 2^31)
    const uint32_t length = (uint32_t)sequence_length(a.c, s), tid = threadIdx.x, keep = (uint32_t)a.keep;
    const uint64_t unit = (uint64_t)s * a.c.kv_heads + h;
    const float *w = a.weights + unit * a.weight_stride;
    const uint32_t count = length < keep ? length : keep;
    const bool all = length <= keep;
    uint32_t need = (uint32_t)(a.keep - a.first - a.recent);     // of the candidates, low <= slot < high, to stay
    const bool some = !all && need > 0, once = length <= kSelectTile;
    const uint32_t low = all ? length : (uint32_t)a.first, high = all ? length : length - (uint32_t)a.recent;
    // a key that is above all weights' for slots that stay anyway, and (not looked at) behind the last
    constexpr uint32_t kStays = 0xffffffffu;
    float own[kSelectEach];
    uint32_t key[kSelectEach];
    auto load = [&](uint32_t base) __attribute__((always_inline)) {
        const uint32_t j = base + tid * kSelectEach;
        if (j + kSelectEach <= length) {   // (rows of weights lie at multiples of four bytes alone, which is enough for sixteen at once)
            for (int i = 0; i < kSelectEach / 4; ++i) {
                const f32x4_of_4 v = *(const f32x4_of_4 *)(w + j + 4 * i);
                for (int n = 0; n < 4; ++n) own[4 * i + n] = v[n];
            }
        } else {
            for (int i = 0; i < kSelectEach; ++i) own[i] = j + i < length ? w[j + i] : 0.0f;
        }
        for (int i = 0; i < kSelectEach; ++i) key[i] = j + i >= low && j + i < high ? weight_key(own[i]) : kStays;
    };
    // (waves that hold nothing go from barrier to barrier)
    const uint32_t wave_first = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid & ~63u)) * kSelectEach;
    load(0);
    uint32_t prefix = some ? 0 : kStays - 1, mask = 0;
    if (some) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
            const uint32_t digits = pass == 2 ? 1023u : 2047u;
            s_bins[tid] = 0;
            s_bins[tid + kSelectThreads] = 0;
            __syncthreads();
            for (uint32_t base = 0; base < length; base += kSelectTile) {
                if (!once) load(base);
                if (base + wave_first >= length) continue;
                for (int i = 0; i < kSelectEach; ++i)
                    if (key[i] != kStays && (key[i] & mask) == prefix) atomicAdd(&s_bins[(key[i] >> shift) & digits], 1u);
            }
            __syncthreads();
            const uint32_t bin = kSelectBins - 1 - 2 * tid, c0 = s_bins[bin], c1 = s_bins[bin - 1];
            uint32_t total;
            const uint32_t before = block_prefix(c0 + c1, s_sums, &total);
            if (before < need && need <= before + c0 + c1) {
                const bool second = need > before + c0;
                s_found[0] = second ? bin - 1 : bin;
                s_found[1] = need - before - (second ? c0 : 0u);
            }
            __syncthreads();
            prefix |= s_found[0] << shift;
            mask |= digits << shift;
            need = s_found[1];
        }
    }
    // all with a larger key than `prefix` stay, and `need` of those with that key, the ones in front
    uint32_t greater = 0, equal = 0;   // in front of a tile
    for (uint32_t base = 0; base < length; base += kSelectTile) {
        if (!once) load(base);
        const uint32_t j0 = base + tid * kSelectEach;
        const int held = (int)(length - j0);   // (of this thread, none where it is not above 0)
        uint32_t more = 0, same = 0, total;
        for (int i = 0; i < kSelectEach; ++i) {
            more |= key[i] > prefix ? 1u << i : 0u;
            same |= key[i] == prefix ? 1u << i : 0u;
        }
        if (held < kSelectEach) more &= held > 0 ? (1u << held) - 1u : 0u;
        const uint32_t front = block_prefix(((uint32_t)__builtin_popcount(more) << 16) | (uint32_t)__builtin_popcount(same), s_sums, &total);
        uint32_t rank = equal + (front & 0xffffu), at = greater + (front >> 16) + (rank < need ? rank : need);
        greater += total >> 16;
        equal += total & 0xffffu;
        if (base + wave_first >= length) continue;
        for (int i = 0; i < kSelectEach; ++i) {
            const bool tied = (same >> i) & 1u;
            if ((((more >> i) & 1u) || (tied && rank < need)) && at < count) {
                a.kept[unit * keep + at] = (int32_t)(j0 + (uint32_t)i);
                a.to_weights[unit * keep + at] = own[i];
                ++at;
            }
            rank += tied ? 1u : 0u;
        }
    }
    for (uint32_t i = count + tid; i < keep; i += kSelectThreads) {
        a.kept[unit * keep + i] = -1;
        a.to_weights[unit * keep + i] = 0.0f;
    }
    if (h == 0 && tid == 0) a.to_lengths[s] = (int32_t)count;
}

// A wave moves the kept rows into one record of the new pages: where each comes from is found once and handed out through LDS.
// Values' codes of a slot lie two bytes at a time among those of its seven neighbours, so that nearly all lines of the old records are read:
// 4096 kept of up to 16384 slots, 16 sequences of 8 heads of 128 values, 82 MB, take 40 us.
template <int NB>
__global__ __launch_bounds__(256) void k_cache_move(EvictArgs a, int records)
{
    __shared__ uint64_t s_from[4][kRecordSlots];         // its record's place among the pages, all ones: none, which is moved as zeros
    __shared__ int s_slot[4][kRecordSlots];              // its slot of that record
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const uint32_t groups = ((uint32_t)records + 3) / 4;
    const int it = (int)(blockIdx.x % groups) * 4 + wave;
    const int h = (int)(blockIdx.x / groups % (unsigned)a.c.kv_heads);
    const int s = (int)(blockIdx.x / groups / (unsigned)a.c.kv_heads);
    const int length = sequence_length(a.c, s), count = length < a.keep ? length : a.keep;
    if (it >= (int)(((uint32_t)count + 31) >> 5)) return;   // (records: slots behind the last one may pass 2^31)
    const int left = count - it * kRecordSlots < kRecordSlots ? count - it * kRecordSlots : kRecordSlots;     // rows of this record
    uint8_t *to = record_of(a.c, a.to_table, a.to_table_stride, s, h, it * kRecordSlots, NB);
    if (!to) return;
    if (lane < left) {
        const int slot = a.kept[((uint64_t)s * a.c.kv_heads + h) * a.keep + it * kRecordSlots + lane];
        const uint8_t *from = record_of(a.c, a.c.table, a.c.table_stride, s, h, slot, NB);
        s_from[wave][lane] = from ? (uint64_t)(from - a.c.pages) : ~0ull;
        s_slot[wave][lane] = slot & 31;
    }
    wave_lds_order();
    // keys: 16 bytes of a row at a time
    for (int u = lane; u < left * NB; u += 64) {
        const int t = u / NB, slot = s_slot[wave][t];
        const uint64_t place = s_from[wave][t];
        const uint8_t *from = a.c.pages + place;
        u32x4 v = {0, 0, 0, 0};
        uint16_t lo = 0;
        if (place != ~0ull) {
            v = *(const u32x4 *)(from + slot * 16 * NB + (u % NB) * 16);
            lo = *(const uint16_t *)(from + kKeyLows * NB + (slot * NB + u % NB) * 2);
        }
        *(u32x4 *)(to + u * 16) = v;
        *(uint16_t *)(to + kKeyLows * NB + u * 2) = lo;
    }
    // what lies by eights of slots, in units of 16 bytes: values' codes (8 NB units for every eight), steps of both, values' lowest numbers (NB each)
    for (int u = lane; u < 44 * NB; u += 64) {
        const int octet = u / (11 * NB), place = u % (11 * NB);
        const int part = place < 8 * NB ? 0 : 1 + (place - 8 * NB) / NB, units = part == 0 ? 8 * NB : NB;
        const int unit = part == 0 ? place : (place - 8 * NB) % NB;
        const uint32_t offset = (part == 0 ? kValueCodes : (part == 1 ? kKeySteps : (part == 2 ? kValueSteps : kValueLows))) * NB;
        uint32_t word[8];
        for (int e = 0; e < 8; ++e) {
            const int t = octet * 8 + e, slot = t < left ? s_slot[wave][t] : 0;
            const uint64_t from = t < left ? s_from[wave][t] : ~0ull;
            word[e] = from != ~0ull ? *(const uint16_t *)(a.c.pages + from + offset + ((slot >> 3) * units + unit) * 16 + (slot & 7) * 2) : 0u;
        }
        uint8_t *at = to + offset + (octet * units + unit) * 16;
        if (octet * 8 + 8 <= left) {
            *(u32x4 *)at = u32x4{word[0] | (word[1] << 16), word[2] | (word[3] << 16), word[4] | (word[5] << 16), word[6] | (word[7] << 16)};
        } else {
            for (int e = 0; e < 8; ++e)
                if (octet * 8 + e < left) ((uint16_t *)at)[e] = (uint16_t)word[e];
        }
    }
}

// ---------------------------------------------------------------- launchers
template <bool STORE, int TY>
static hipError_t rows_of_type(const CacheArgs &c, const RowsArgs &r, int nb, hipStream_t s)
{
    const uint32_t items = ((uint32_t)r.n_rows / kRowsOfWave + 2u * (uint32_t)c.n_seqs) * (uint32_t)c.kv_heads;
    const dim3 grid((items + 3) / 4), block(256);
    if (STORE) {
        if (nb == 2) hipLaunchKernelGGL((k_cache_store<2, TY>), grid, block, 0, s, c, r, items);
        else if (nb == 4) hipLaunchKernelGGL((k_cache_store<4, TY>), grid, block, 0, s, c, r, items);
        else hipLaunchKernelGGL((k_cache_store<8, TY>), grid, block, 0, s, c, r, items);
    } else {
        if (nb == 2) hipLaunchKernelGGL((k_cache_load<2, TY>), grid, block, 0, s, c, r, items);
        else if (nb == 4) hipLaunchKernelGGL((k_cache_load<4, TY>), grid, block, 0, s, c, r, items);
        else hipLaunchKernelGGL((k_cache_load<8, TY>), grid, block, 0, s, c, r, items);
    }
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
    hipError_t e = hipSuccess;
    if (tiles) {
        const dim3 grid(tiles * (uint32_t)a.splits);
        if constexpr (TY != kF32) {
            if (a.wide_tiles) {
                const dim3 wide((uint32_t)a.c.n_seqs * (uint32_t)a.c.kv_heads * (uint32_t)a.wide_tiles * (uint32_t)a.splits);
                if (a.tiles_in_wide == 4) hipLaunchKernelGGL((k_cache_attend_rows<NB, TY, 4, 1>), wide, dim3(256), 0, s, a);
                else if (a.tiles_in_wide == 8) hipLaunchKernelGGL((k_cache_attend_rows<NB, TY, 8, 1>), wide, dim3(512), 0, s, a);
                else if constexpr (NB < 8) hipLaunchKernelGGL((k_cache_attend_rows<NB, TY, 8, 2>), wide, dim3(512), 0, s, a);
                e = hipGetLastError();
                if (e != hipSuccess) return e;
            }
        }
        hipLaunchKernelGGL((k_cache_attend<NB, TY>), grid, dim3(256), 0, s, a);
        e = hipGetLastError();
        if (e == hipSuccess && a.splits > 1) {
            hipLaunchKernelGGL((k_cache_join<NB, TY>), dim3(tiles * (uint32_t)a.columns), dim3(256), 0, s, a);
            e = hipGetLastError();
        }
    }
    if (e == hipSuccess && a.weights && a.c.max_slots > 0) {
        const uint32_t records = ((uint32_t)a.c.max_slots + kRecordSlots - 1) / kRecordSlots;
        const uint32_t all = (records + kAttendWaves * kHeldRecords - 1) / (kAttendWaves * kHeldRecords);   // batches of a sequence and head
        const uint32_t units = (uint32_t)a.c.kv_heads * (uint32_t)a.c.n_seqs;
        uint32_t batches = all * units / (256 * kWeightsPerUnit);
        if (batches < 1) batches = 1;
        hipLaunchKernelGGL((k_cache_weights<NB, TY>), dim3((all + batches - 1) / batches * units), dim3(256), 0, s, a, (int)records, (int)batches);
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
