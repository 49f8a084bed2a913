// checkers_amd/csrc/ckr_attention.hip — attention of a chunk of new tokens over
// a paged cache (ckr_kv_attention).
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>
#include <utility>

#include "ckr_internal.h"
#include "ckr_kv.h"

namespace ckr {

int kv_check_cache(const ckr_kv_cache* c);
int kv_check_batch(const ckr_kv_cache* c, const ckr_kv_batch* b);
int kv_check_rows(const void* p, uint64_t rows, int64_t row_stride, uint64_t heads, int64_t head_stride, uint64_t dim,
                  int es, bool written, const char* what);

namespace {

int err(int code, const std::string& m) { return set_error(code, "[ckr] " + m); }

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArg {
    const uint8_t* q;
    uint8_t* out;
    float* lse;
    int64_t q_tok, q_head, o_tok, o_head;
    const uint8_t* ck;
    const uint8_t* cv;
    const float* sk;
    const float* sv;
    int64_t kst[3], vst[3], skst[2], svst[2];  // of rows in bytes, of scales in elements
    uint32_t n_pages, page_shift, dim, heads, group, kv_heads;  // heads: query heads
    uint32_t window;
    float scale2;   // |scale| log2(e): the softmax runs in powers of two
    uint32_t flip;  // 0x80008000 when scale is negative: the queries' signs are flipped instead
    KvBatch b;
    uint32_t tiles, splits, split_len;  // row tiles, key ranges of a tile, their length (a multiple of 128)
    uint32_t* counters;  // few rows: parts done of the item that begins in a block and goes on in the next; 0 between calls
    uint32_t min_tiles;  // few rows: tiles of a block's stretch at least
    // with splits > 1; few rows: [block][its first item's part, its last one's][row]
    float* part_o;  // [tile][kv head][split][rows of a tile][DP]
    float* part_m;  // [tile][kv head][split][rows of a tile][2]: maximum (in powers of two), sum
};

// ---- matrix instructions.  Operands are 8 elements of 16 bits a lane.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename E> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (E::tag == CKR_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename E> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (E::tag == CKR_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Four codes of a dword as two dwords of 16-bit values (exact: e4m3 values and
// int8 fit both 16-bit types).
template <typename C, typename E> __device__ __forceinline__ u32x2 widen4(uint32_t v) {
    if constexpr (C::tag == CKR_F8 && E::tag == CKR_BF16)
        return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.f, true))};
    else if constexpr (C::tag == CKR_F8)
        return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.f, true))};
    else {
        const f32x4 f = codes4<C>(v);
        return u32x2{pack16<E>(f[0], f[1]), pack16<E>(f[2], f[3])};
    }
}
// The same times a power of two, in float16.
template <typename C> __device__ __forceinline__ u32x2 widen4_by(uint32_t v, float power) {
    if constexpr (C::tag == CKR_F8)
        return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, power, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, power, true))};
    else {
        const f32x4 f = codes4<C>(v) * power;
        return u32x2{pack16<ElemF16>(f[0], f[1]), pack16<ElemF16>(f[2], f[3])};
    }
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// Maximum over the lanes l, l ^ 32 (and l ^ 16).
__device__ __forceinline__ float max_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
    return fmaxf(as_f32(r[0]), as_f32(r[1]));
}
__device__ __forceinline__ float max_quarters(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
    return max_half(fmaxf(as_f32(r[0]), as_f32(r[1])));
}
__device__ __forceinline__ float sum_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
    return as_f32(r[0]) + as_f32(r[1]);
}
__device__ __forceinline__ float sum_quarters(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
    return sum_half(as_f32(r[0]) + as_f32(r[1]));
}

// Weights meet the values in 16 bits, the matrix instructions' operands.  Rounded
// once to the queries' type, they make the output's error 1.4 times that of its own
// rounding over an 8-bit cache (their value's scale is in them; up to 1.75 for short
// chunks) and 1.1 to 1.4 times over a 16-bit one.  So:
// - few rows: two products, of the weight rounded and of what that leaves (16 bits in
//   bfloat16, 22 in float16), which memory covers: a step of 64 sequences to 16000
//   175.5 us, 174.3 with one (157 and 152 for heads of 80).
// - many rows, bfloat16 over an 8-bit cache: float16 weights (ProbMany), 11 bits, an
//   error of 1.01: a chunk of 2048 behind 30000 1.12 ms, 1.06 with bfloat16 ones (the same
//   instructions otherwise; with two products 1.41); 128 rows a head 109 us and 105.
// - 128 rows, float16 over an 8-bit cache: two products, 132 us and 109.
// - many rows else: rounded once.  Two products are 630 us instead of 505 for prompts in
//   float16, 750 instead of 560 for a chunk over bfloat16.
// Their type is the queries' but for ProbMany: bfloat16 weights take the value's scale
// without a range of their own.  float16 weights are scaled up by 2^up so that small ones
// keep their bits (their largest is 1, or 2^kLag where a running maximum lags, or
// twice that with a value's scale, so at most 2^15); of an 8-bit value's scale they
// take the fraction (1 to 2), and the codes its power of two as they are widened,
// which leaves the values' own range (up to 65504).
template <typename X, typename C> struct Prob {
    typedef X E;
    static constexpr bool split = X::tag == CKR_F16 && C::bytes == 1, scaled = false;
    static constexpr float up = X::tag == CKR_F16 ? (C::bytes == 1 ? 6.f : 7.f) : 0.f;
};
// In the kernels of many rows bfloat16 queries have float16 weights too over an 8-bit
// cache, whose codes are float16 values as well.  There a wave keeps the power of two of
// the largest value scale so far, e, besides the maximum m of its rows: weights and sums
// are held against 2^(m + e), so that a weight with its value's whole scale is at most
// 2^15 whatever the range of the scales, and a small one is off by 2^-31 of the largest
// value at most.
template <typename X, typename C> struct ProbMany : Prob<X, C> {};
struct ProbScaled {
    typedef ElemF16 E;
    static constexpr bool split = false, scaled = true;
    static constexpr float up = 6.f;
};
template <> struct ProbMany<ElemBF16, ElemF8> : ProbScaled {};
template <> struct ProbMany<ElemBF16, ElemI8> : ProbScaled {};
// e of the largest scale (at least kLeast: sums of weights without values stay in range;
// above 100, values of 10^32, a sum keeps fewer than 32 octaves below its largest weight).
constexpr float kLeast = -80.f;
__device__ __forceinline__ float scale_power(float largest) {
    return fmaxf((float)(int)(as_u32(largest) >> 23) - 127.f, kLeast);
}
// Maximum over each 16 lanes.
__device__ __forceinline__ float max_row16(float x) {
    const auto turned = [](float y, auto n) {
        return as_f32((uint32_t)__builtin_amdgcn_mov_dpp((int)as_u32(y), 0x120 + decltype(n)::value, 0xf, 0xf, true));  // row_ror:n
    };
    x = fmaxf(x, turned(x, std::integral_constant<int, 8>{}));
    x = fmaxf(x, turned(x, std::integral_constant<int, 4>{}));
    x = fmaxf(x, turned(x, std::integral_constant<int, 2>{}));
    return fmaxf(x, turned(x, std::integral_constant<int, 1>{}));
}
// Eight weights as two 16-bit values each, the second what the first leaves.
template <typename P> struct Halves {
    u32x4 hi, lo;
    __device__ __forceinline__ void add(int i, float x, float y) {
        const uint32_t h = pack16<P>(x, y);
        hi[i] = h, lo[i] = pack16<P>(x - lo16<P>(h), y - hi16<P>(h));
    }
};
// A scale as a power of two and the rest (zero, subnormal and non-finite scales: 1
// and themselves; powers that would take the largest code past 65504: the largest
// that does not).
struct SplitScale { float power, rest; };
template <typename C> __device__ __forceinline__ SplitScale split_scale(float s) {
    const uint32_t top = C::tag == CKR_F8 ? 0x43000000u : 0x44000000u;  // 2^7 x 448, 2^9 x 127
    const uint32_t e = as_u32(s) & 0x7f800000u, p = min(e, top);
    const bool normal = e - 0x00800000u < 0x7f000000u;
    return {normal ? as_f32(p) : 1.f, normal ? as_f32(as_u32(s) - p + 0x3f800000u) : s};
}

// How far a row's running maximum may lag behind (in powers of two) before the
// accumulators are scaled: sums and outputs use the same lagging maximum.
constexpr float kLag = 8.f;

// ---- infinities and NaN in 16-bit values.  A tile of keys that not every row sees
// meets weights of zero, and zero times an infinity is NaN: there the products
// take the finite values, and who sees an infinity (or NaN: both) is found by
// products of ones.  (Where every row sees the keys, and float16 weights may be zero all
// the same, the kernels of many rows look at their sums in the end: settle.)
template <typename E> __device__ __forceinline__ bool any_wild(u32x4 w) {  // E: a 16-bit type
    constexpr uint32_t one = E::tag == CKR_BF16 ? 0x00800080u : 0x04000400u;  // carries an exponent of ones into the sign's place
    uint32_t x = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) x |= (w[i] & 0x7fff7fffu) + one;
    return x & 0x80008000u;
}
// sign 0: the finite values; 1: ones where +infinity or NaN; -1: ones where -infinity or NaN.
template <typename E> __device__ __forceinline__ u32x4 wild(u32x4 w, int sign) {
    constexpr uint32_t inf = E::tag == CKR_BF16 ? 0x7f80u : 0x7c00u, one = E::tag == CKR_BF16 ? 0x3f80u : 0x3c00u;
    u32x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t x = w[i / 2] >> (16 * (i % 2)) & 0xffffu;
        const bool bad = (x & 0x7fffu) >= inf, here = bad && x != (sign > 0 ? inf | 0x8000u : inf);
        r[i / 2] |= (sign == 0 ? (bad ? 0u : x) : here ? one : 0u) << (16 * (i % 2));
    }
    return r;
}
// What rows see of wild values, from the two products of ones.
__device__ __forceinline__ float wild_sum(float plus, float minus) {
    return (plus > 0.f ? INFINITY : 0.f) + (minus > 0.f ? -INFINITY : 0.f);
}
// Ones for the keys a row sees (bits 0 to 7).
template <typename E> __device__ __forceinline__ u32x4 ones(uint32_t seen) {
    constexpr uint32_t one = E::tag == CKR_BF16 ? 0x3f80u : 0x3c00u;
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = (seen >> (2 * i) & 1 ? one : 0u) | (seen >> (2 * i + 1) & 1 ? one << 16 : 0u);
    return r;
}

constexpr uint32_t kFewRows = 16, kManyRows = 128, kWideRows = 256;  // rows of a tile
constexpr uint32_t kFewWaves = 4;                                    // waves of a block of few rows

// f(0) .. f(N - 1) with constants.
template <typename F, int... I> __device__ __forceinline__ void unroll_list(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void unroll(F f) { unroll_list(f, std::make_integer_sequence<int, N>{}); }

// Which sequence and rows a tile of BM rows is: rows of a sequence are its
// chunk's tokens times the query heads of a key/value head, in that order.
// Every thread of the block calls it; s_tmp: a word of LDS per wave and five more,
// which tile_found reads again.
struct Tile {
    uint32_t seq, row0, rows, token0;  // rows: of the whole sequence; token0: its first packed row
    int64_t start;                     // the position of its first token
};
template <uint32_t BM, uint32_t THREADS> __device__ __forceinline__ Tile tile_found(uint32_t group, const uint32_t* s_tmp) {
    constexpr uint32_t WAVES = THREADS / 64;
    Tile t;
    t.seq = s_tmp[WAVES], t.row0 = s_tmp[WAVES + 1] * BM, t.token0 = s_tmp[WAVES + 2];
    t.rows = (s_tmp[WAVES + 3] - t.token0) * group;
    t.start = (int32_t)s_tmp[WAVES + 4];
    return t;
}
template <uint32_t BM, uint32_t THREADS = 256>
__device__ __forceinline__ bool find_tile(const KvBatch& b, uint32_t group, uint32_t tile, uint32_t* s_tmp, Tile& t) {
    constexpr uint32_t WAVES = THREADS / 64;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t done = 0;
    for (uint32_t base = 0; base < b.n_seqs; base += THREADS) {
        const uint32_t i = base + threadIdx.x;
        uint32_t n = 0;
        int32_t lo = 0, hi = 0, start = 0;
        if (i < b.n_seqs) {
            lo = b.offsets[i], hi = min(b.offsets[i + 1], (int32_t)b.n_tokens), start = b.starts[i];
            n = lo >= 0 && hi > lo ? ((uint32_t)(hi - lo) * group + BM - 1) / BM : 0;
        }
        uint32_t sum = n;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t u = (uint32_t)__shfl_up((int)sum, d);
            if (lane >= (uint32_t)d) sum += u;
        }
        if (lane == 63) s_tmp[wave] = sum;
        __syncthreads();
        uint32_t before = done, all = 0;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; w++) {
            if (w < wave) before += s_tmp[w];
            all += s_tmp[w];
        }
        if (tile < done + all) {
            const uint32_t first = before + sum - n;
            if (tile >= first && tile < first + n) {
                s_tmp[WAVES] = i, s_tmp[WAVES + 1] = tile - first;
                s_tmp[WAVES + 2] = (uint32_t)lo, s_tmp[WAVES + 3] = (uint32_t)hi, s_tmp[WAVES + 4] = (uint32_t)start;
            }
            __syncthreads();
            t = tile_found<BM, THREADS>(group, s_tmp);
            return true;
        }
        done += all;
        __syncthreads();
    }
    return false;
}

// Whether a row of the tile sees a value whose scale is not finite (64 keys a step, the
// whole wave; for tiles in which there is one).
template <uint32_t BM>
__device__ __forceinline__ bool sees_wild_scale(const AttnArg& a, const Tile& t, uint32_t kvh, uint32_t row) {
    const int64_t pos_lo = t.start + t.row0 / a.group, pos_hi = t.start + min(t.row0 + BM - 1, t.rows - 1) / a.group;
    const int64_t end = min(pos_hi + 1, (int64_t)a.b.width << a.page_shift), pos = t.start + min(row, t.rows - 1) / a.group;
    const auto below = [](int64_t n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; };
    bool hit = false;
    for (int64_t k = a.window ? max((int64_t)0, pos_lo - (int64_t)a.window + 1) : 0; k < end; k += 64) {
        const int64_t key = k + (threadIdx.x & 63);
        const int32_t page = key < end ? page_of(a.b, t.seq, key, a.page_shift, a.n_pages) : -1;
        const uint32_t slot = (uint32_t)key & ((1u << a.page_shift) - 1);
        const bool bad = page >= 0 && abs_bits(a.sv[(int64_t)page * a.svst[0] + (int64_t)kvh * a.svst[1] + slot]) >= 0x7f800000u;
        hit |= __ballot(bad) & below(pos + 1 - k) & ~(a.window ? below(pos - (int64_t)a.window + 1 - k) : 0);
    }
    return hit;
}

// The kernel's arguments once more, for code that hardly ever runs: read where they are
// used, not kept in (spilled) registers from the kernel's start on.
__device__ __forceinline__ const AttnArg& args_here() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();  // AttnArg is the kernels' first argument
    asm volatile("" : "+s"(p));
    return *(const AttnArg*)p;
}

// float16 values, a tile whose sums hold NaN: a weight below 2^-31 of the largest is 0 in
// 16 bits (bfloat16 has the range of 32), and 0 times an infinity is NaN where the
// sum is infinite.  Such sums begin again at 0, and what the row sees of infinities and
// NaN is added; others are what they were (an infinity stays one).  The whole wave
// looks through the tile's keys, 64 pieces of 8 values a load; o as in the kernels of
// 32x32 products: the lane's dimensions are 32 dt + 8 (i / 4) + 4 (lane / 32) + i % 4.
template <typename P, int DP, uint32_t BM>
__device__ __forceinline__ void settle(const Tile& t, uint32_t kvh, uint32_t row, f32x16 (&o)[DP / 32]) {
    constexpr uint32_t PIECES = DP / 8, KEYS = 64 / PIECES;
    const AttnArg& a = args_here();
    uint32_t lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // as args_here: nothing of this is computed before
    const int64_t pos_lo = t.start + t.row0 / a.group, pos_hi = t.start + min(t.row0 + BM - 1, t.rows - 1) / a.group;
    const int64_t end = min(pos_hi + 1, (int64_t)a.b.width << a.page_shift), pos = t.start + min(row, t.rows - 1) / a.group;
    const uint32_t piece = lane % PIECES, slot_mask = (1u << a.page_shift) - 1;
    const uint8_t* const v = a.cv + (int64_t)kvh * a.vst[1];
#pragma unroll
    for (int dt = 0; dt < DP / 32; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[dt][i] = o[dt][i] == o[dt][i] ? o[dt][i] : 0.f;
    for (int64_t k = a.window ? max((int64_t)0, pos_lo - (int64_t)a.window + 1) : 0; k < end; k += KEYS) {
        const int64_t mine = k + lane / PIECES;
        int32_t page = mine < end ? page_of(a.b, t.seq, mine, a.page_shift, a.n_pages) : -1;
        u32x4 w = {0, 0, 0, 0};
        if (page >= 0 && piece * 8 < a.dim)
            w = *reinterpret_cast<const u32x4*>(v + (int64_t)page * a.vst[0] + (int64_t)((uint32_t)mine & slot_mask) * a.vst[2] + piece * 16);
        if (!__any(any_wild<P>(w))) continue;
        for (int64_t key = k; key < min(k + KEYS, end); key++) {
            page = page_of(a.b, t.seq, key, a.page_shift, a.n_pages);
            if (page < 0 || key > pos || (a.window && key <= pos - (int64_t)a.window)) continue;
            const uint8_t* const at = v + (int64_t)page * a.vst[0] + (int64_t)((uint32_t)key & slot_mask) * a.vst[2];
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const uint32_t d = dt * 32 + 2 * i + 4 * (lane >> 5);
                    if (d >= a.dim) continue;
                    const u32x2 x = *reinterpret_cast<const u32x2*>(at + d * 2);
                    const float y[4] = {lo16<P>(x[0]), hi16<P>(x[0]), lo16<P>(x[1]), hi16<P>(x[1])};
#pragma unroll
                    for (int e = 0; e < 4; e++) o[dt][i + e] += abs_bits(y[e]) >= 0x7f800000u ? y[e] : 0.f;
                }
        }
    }
}
template <int N> __device__ __forceinline__ bool any_nan(const f32x16 (&o)[N]) {
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < N; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) nan |= o[dt][i] != o[dt][i];
    return __any(nan);
}

// ------------------------------------------------------------ few rows
// A tile of 16 rows against tiles of 32 keys (16x16x32 matrix products), a wave at a time:
//   S^T = K Q^T: operand A holds a key per lane and row, so a lane reads whole
//   16-byte pieces of its key's row; the order of the contraction is free, and Q
//   is laid out to match;
//   O^T = V^T P^T: the lane's 8 keys of P are the rows of S^T it already holds
//   (keys 4 g + i and 16 + 4 g + i of the tile, g the lane's quarter), so P needs no
//   exchange between lanes; V's operand holds those keys for one dimension, which
//   a lane gets by loading NV = DP / 16 dimensions of 8 keys and transposing them in
//   registers.
// So no key or value goes through LDS, and two tiles (16 KiB of an 8-bit cache of 128
// dimensions) are on their way per wave: a tile's registers are loaded again as
// soon as they have been used.
//
// The work of all items (a row tile and a key/value head) is one line of key tiles,
// of which every block takes an equal stretch, whatever the sequences' lengths; its
// four waves share each item's tiles and join their sums through LDS.  A stretch
// that covers an item writes its rows; otherwise the block leaves its part (maximum,
// sum, weighted values) in the workspace, and the last block of an item's to finish
// joins the parts, in an order that does not depend on which one that is.
//
// Bound by memory: 64 sequences of 200 to 16000 tokens in e4m3, 8 heads of 128 for 32
// query heads, 919 MB in 176 us (5.2 TB/s; a kernel that only reads reaches 6.4).  Blocks
// that each took whole items, longest first, left CUs idle at the end: 234 us.  One
// sequence of 1000 tokens, 9.5 to 10 us: the launch, then a chain of about six dependent
// reads (chunk, table, rows, counter, parts).  Over 16-bit caches, heads of 128, 15
// registers spill (1.78 GB in 342 us, 5.2 TB/s all the same).
template <typename C, int DP> struct FewRegs {
    static constexpr int KL = DP * C::bytes / 64;      // 16-byte pieces of a key's row per lane
    static constexpr int VD = DP / 16 * C::bytes / 4;  // dwords of a key's value row per lane
    u32x4 k[2][KL];
    uint32_t v[8][VD];
    f32x4 sk[2], sv[2];
};

// Parts of an item go from one CU to another, perhaps on another die: their stores
// write through and their loads read past the caches (accesses of device scope), so
// that no cache has to be written back or emptied for them.
__device__ __forceinline__ void store_far(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)as_u32(y) << 32 | as_u32(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 load_far(const float* p) {
    const uint64_t x = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return f32x2{as_f32((uint32_t)x), as_f32((uint32_t)(x >> 32))};
}

// Keys of a row tile: tiles of 32 from `first` on, up to `limit`.
struct FewSpan { int64_t pos_lo, pos_hi, first, limit; };
__device__ __forceinline__ FewSpan few_span(const AttnArg& a, int64_t start, uint32_t row0, uint32_t rows) {
    FewSpan f;
    f.pos_lo = start + row0 / a.group, f.pos_hi = start + min(row0 + kFewRows - 1, rows - 1) / a.group;
    f.limit = min(f.pos_hi + 1, (int64_t)a.b.width << a.page_shift);
    f.first = a.window ? max((int64_t)0, f.pos_lo - (int64_t)a.window + 1) & ~31ll : 0;
    return f;
}
__device__ __forceinline__ uint32_t few_tiles(const FewSpan& f) {  // one at least: a row without keys is written too
    return f.limit > f.first + 32 ? (uint32_t)((f.limit - f.first + 31) / 32) : 1u;
}
template <typename X, typename C, int DP>
__global__ void __launch_bounds__(64 * kFewWaves, (DP > 128 ? 1 : 2)) attend_few_kernel(AttnArg a) {
    typedef typename Prob<X, C>::E P;
    typedef FewRegs<C, DP> Regs;
    constexpr int KL = Regs::KL, VD = Regs::VD, NV = DP / 16, KS = DP / 32;
    constexpr uint32_t THREADS = 64 * kFewWaves, QUADS = DP / 4;  // a row's outputs by fours
    __shared__ __attribute__((aligned(16))) float s_o[kFewWaves][kFewRows][DP + 4];
    __shared__ float s_m[kFewWaves][kFewRows][2];
    __shared__ uint32_t s_sum[kFewWaves];
    __shared__ uint32_t s_at[5];  // the block's first sequence, tiles of it before the block's; its rows, token, start
    __shared__ uint32_t s_last;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;

    // ---- this block's stretch of the line of key tiles.  The launch has seen to it that
    // the line of any batch is shorter than 2^31; chunks that overlap, which are no batch,
    // may add up to more: sums stop at 2^32 - 1, and nothing is done then
    struct Seq { uint32_t tiles, rows, token0; int32_t start; };
    const auto count = [&](uint32_t seq) {
        Seq q = {0, 0, 0, 0};
        if (seq >= a.b.n_seqs) return q;
        const int32_t from = a.b.offsets[seq], to = min(a.b.offsets[seq + 1], (int32_t)a.b.n_tokens);
        q.start = a.b.starts[seq];
        q.rows = from >= 0 && to > from ? (uint32_t)(to - from) * a.group : 0;
        q.token0 = (uint32_t)from;
        for (uint32_t r = 0; r < q.rows; r += kFewRows) q.tiles += few_tiles(few_span(a, q.start, r, q.rows));
        q.tiles *= a.kv_heads;
        return q;
    };
    // inclusive sum over the block's threads, and the block's total
    const auto scan = [&](uint32_t tiles, uint32_t& all) {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t x = (uint32_t)__shfl_up((int)tiles, d);
            if (lane >= (uint32_t)d) tiles = __builtin_elementwise_add_sat(tiles, x);
        }
        __syncthreads();
        if (lane == 63) s_sum[wave] = tiles;
        __syncthreads();
        all = 0;
#pragma unroll
        for (uint32_t w = 0; w < kFewWaves; w++) {
            if (w == wave) tiles = __builtin_elementwise_add_sat(tiles, all);
            all = __builtin_elementwise_add_sat(all, s_sum[w]);
        }
        return tiles;
    };
    uint32_t total;
    const Seq q0 = count(threadIdx.x);
    const uint32_t upto0 = scan(q0.tiles, total), total0 = total;
    for (uint32_t base = THREADS; base < a.b.n_seqs; base += THREADS) {
        uint32_t more;
        scan(count(base + threadIdx.x).tiles, more);
        total = __builtin_elementwise_add_sat(total, more);
    }
    if (total >= 1u << 31) return;
    const uint32_t per = max((total + gridDim.x - 1) / gridDim.x, a.min_tiles);
    if ((uint64_t)blockIdx.x * per >= total) return;
    const uint32_t p_begin = blockIdx.x * per, p_end = min(p_begin + per, total);
    {
        const auto find = [&](uint32_t seq, const Seq& x, uint32_t upto) {
            if (p_begin >= upto - x.tiles && p_begin < upto) {
                s_at[0] = seq, s_at[1] = p_begin - (upto - x.tiles);
                s_at[2] = x.rows, s_at[3] = x.token0, s_at[4] = (uint32_t)x.start;
            }
        };
        find(threadIdx.x, q0, upto0);
        uint32_t before = total0;
        for (uint32_t base = THREADS; base < a.b.n_seqs; base += THREADS) {
            const Seq x = count(base + threadIdx.x);
            uint32_t more;
            const uint32_t upto = scan(x.tiles, more);
            find(base + threadIdx.x, x, before + upto);
            before += more;
        }
        __syncthreads();
    }
    const auto scalar = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane(x); };
    uint32_t seq = scalar(s_at[0]), in_seq = scalar(s_at[1]), rows = scalar(s_at[2]), token0 = scalar(s_at[3]), row0 = 0;
    int32_t start = (int32_t)scalar(s_at[4]);
    // the item that the stretch begins in
    FewSpan span = few_span(a, start, 0, rows);
    uint32_t nt = few_tiles(span);
    while (in_seq >= nt * a.kv_heads) {
        in_seq -= nt * a.kv_heads, row0 += kFewRows;
        span = few_span(a, start, row0, rows), nt = few_tiles(span);
    }
    uint32_t kvh = scalar(in_seq / nt), t0 = scalar(in_seq % nt);

    for (uint32_t p = p_begin; p < p_end;) {
        const uint32_t t1 = scalar(min(nt, t0 + (p_end - p)));
        // the waves share the item's tiles (or this block's part of them) evenly
        const uint32_t w0 = (uint32_t)((uint64_t)(t1 - t0) * wave / kFewWaves), w1 = (uint32_t)((uint64_t)(t1 - t0) * (wave + 1) / kFewWaves);
        const int64_t lo = span.first + 32ll * (t0 + w0);
        const int n_tiles = w1 - w0;
        // from here on keys are counted from lo, in 32 bits
        const auto rel = [&](int64_t x) { return (int)max((int64_t)-0x40000000, min(x - lo, (int64_t)0x7fffffff - 256)); };
        const uint32_t row = row0 + col;
        const int64_t my_pos = span.pos_lo - row0 / a.group + min(row, rows - 1) / a.group;
        const int pos = rel(my_pos), see = a.window ? rel(my_pos - (int64_t)a.window) : -0x40000000;
        const int end = __builtin_amdgcn_readfirstlane(rel(span.limit));
        const int full_to = __builtin_amdgcn_readfirstlane(min(rel(span.pos_lo) + 1, end));  // every row sees the keys before this
        const int full_from = __builtin_amdgcn_readfirstlane(a.window ? rel(span.pos_hi - (int64_t)a.window) + 1 : -0x40000000);  // and from this on

        // queries: the elements of each 32-wide step in the order of the keys' pieces
        u32x4 q[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const uint32_t d = C::bytes == 1 ? (ks / 2) * 64 + g * 16 + (ks % 2) * 8 : ks * 32 + g * 8;
            q[ks] = u32x4{0, 0, 0, 0};
            if (row < rows && d < a.dim)
                q[ks] = *reinterpret_cast<const u32x4*>(a.q + ((int64_t)(token0 + row / a.group) * a.q_tok +
                                                              (int64_t)(kvh * a.group + row % a.group) * a.q_head + d) * 2);
        }
        const uint8_t* const ck = a.ck + (int64_t)kvh * a.kst[1];
        const uint8_t* const cv = a.cv + (int64_t)kvh * a.vst[1];
        const float* const skp = a.sk + (int64_t)kvh * a.skst[1];
        const float* const svp = a.sv + (int64_t)kvh * a.svst[1];
        const int64_t k_off = (int64_t)col * a.kst[2] + g * 16;
        // one offset and three sums a load, for 16-bit caches have no registers for four (390 us
        // a step of 64 sequences to 16000 with them, 342 without; e4m3 177 and 176); four where
        // values are widened by their scale's power (183 us, 196 with one)
        constexpr int OFFS = Prob<X, C>::split ? 4 : 1;
        int64_t v_off[OFFS];
#pragma unroll
        for (int i = 0; i < OFFS; i++) v_off[i] = (int64_t)(4 * g + i) * a.vst[2] + col * (VD * 4);
        const auto v_row = [&](int i) { return OFFS == 4 ? v_off[i % OFFS] : i * a.vst[2] + v_off[0]; };
        const bool v_in = col * NV < a.dim;
        typedef __attribute__((address_space(1))) const int32_t* global_i32;
        const global_i32 table = (global_i32)(a.b.table + (int64_t)seq * a.b.table_stride);
        const uint32_t slot_mask = (1u << a.page_shift) - 1, in0 = (uint32_t)lo & slot_mask;
        // table columns c0 .. c0 + 63 in a register of the wave, the next 64 on their way
        uint32_t c0 = (uint32_t)(lo >> a.page_shift);
        const auto page_lane = [&](uint32_t c) {
            c += lane;
            const int32_t x = c < a.b.width ? table[c] : -1;
            return (uint32_t)x < a.n_pages ? x : -1;
        };
        int32_t window_now = page_lane(c0), window_next = page_lane(c0 + 64);
        uint32_t c_now = 0;
        const auto page_at = [&](int j) {  // of key j; called with j rising by 16
            const uint32_t c = (in0 + (uint32_t)j) >> a.page_shift;
            if (c - c_now >= 64) {
                c_now += 64;
                window_now = window_next;
                window_next = page_lane(c0 + c_now + 64);
            }
            return (int32_t)__builtin_amdgcn_readlane(window_now, (int)(c - c_now));
        };
        const auto load_k = [&](Regs& r, int base, const int32_t* pages) {
            const bool whole = pages[0] >= 0 && pages[1] >= 0 && base + 32 <= end && DP == a.dim;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t slot = (in0 + (uint32_t)base + 16 * h) & slot_mask;
                const uint8_t* at = ck + (int64_t)pages[h] * a.kst[0] + (int64_t)slot * a.kst[2] + k_off;
                if (whole) {
#pragma unroll
                    for (int j = 0; j < KL; j++) r.k[h][j] = *reinterpret_cast<const u32x4*>(at + j * 64);
                } else {
#pragma unroll
                    for (int j = 0; j < KL; j++) {
                        r.k[h][j] = u32x4{0, 0, 0, 0};
                        if (pages[h] >= 0 && base + 16 * h + (int)col < end && (j * 64 + g * 16) / C::bytes < a.dim)
                            r.k[h][j] = *reinterpret_cast<const u32x4*>(at + j * 64);
                    }
                }
                if constexpr (C::bytes == 1) r.sk[h] = *reinterpret_cast<const f32x4*>(skp + (int64_t)max(pages[h], 0) * a.skst[0] + slot + 4 * g);
            }
        };
        const auto load_v = [&](Regs& r, int base, const int32_t* pages) {
            const bool whole = pages[0] >= 0 && pages[1] >= 0 && base + 32 <= end && DP == a.dim;
            const auto get = [&](uint32_t (&v)[VD], const uint8_t* at) {
                if constexpr (VD == 1) v[0] = *reinterpret_cast<const uint32_t*>(at);
                else if constexpr (VD == 2) {
                    const u32x2 y = *reinterpret_cast<const u32x2*>(at);
                    v[0] = y[0], v[1] = y[1];
                } else {
#pragma unroll
                    for (int j = 0; j < VD; j += 4) {
                        const u32x4 y = *reinterpret_cast<const u32x4*>(at + j * 4);
#pragma unroll
                        for (int k = 0; k < 4; k++) v[j + k] = y[k];
                    }
                }
            };
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t slot = (in0 + (uint32_t)base + 16 * h) & slot_mask;
                const uint8_t* at = cv + (int64_t)pages[h] * a.vst[0] + (int64_t)slot * a.vst[2];
                if constexpr (C::bytes == 1) r.sv[h] = *reinterpret_cast<const f32x4*>(svp + (int64_t)max(pages[h], 0) * a.svst[0] + slot + 4 * g);
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 4; i++) get(r.v[4 * h + i], at + v_row(i));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
#pragma unroll
                        for (int j = 0; j < VD; j++) r.v[4 * h + i][j] = 0;
                        if (pages[h] >= 0 && base + 16 * h + 4 * (int)g + i < end && v_in) get(r.v[4 * h + i], at + v_row(i));
                    }
                }
            }
        };

        float m = -INFINITY, l = 0.f;
        f32x4 o[NV];
#pragma unroll
        for (int c = 0; c < NV; c++) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        const auto scores = [&](const Regs& r, f32x4 (&s)[2]) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KL; j++) {
                    if constexpr (C::bytes == 1) {
                        const u32x4 x = r.k[h][j];
                        const u32x2 w0 = widen4<C, X>(x[0]), w1 = widen4<C, X>(x[1]), w2 = widen4<C, X>(x[2]), w3 = widen4<C, X>(x[3]);
                        s[h] = mfma16<X>(u32x4{w0[0], w0[1], w1[0], w1[1]}, q[2 * j], s[h]);
                        s[h] = mfma16<X>(u32x4{w2[0], w2[1], w3[0], w3[1]}, q[2 * j + 1], s[h]);
                    } else {
                        s[h] = mfma16<X>(r.k[h][j], q[j], s[h]);
                    }
                }
            }
        };
        // the weights of a tile, with the values' scales; what a row does not see weighs 0
        const auto weights = [&](const Regs& r, const f32x4 (&s)[2], int base, const int32_t* pages, uint32_t& seen) {
            const bool full = pages[0] >= 0 && pages[1] >= 0 && base + 32 <= full_to && base >= full_from;
            float x[8], top = -INFINITY;
            seen = ~0u;  // every row sees every key
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = s[i / 4][i % 4] * a.scale2;
                if constexpr (C::bytes == 1) x[i] *= r.sk[i / 4][i % 4];
            }
            if (!full) {
                seen = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int j = base + 16 * (i / 4) + 4 * (int)g + i % 4;
                    if (pages[i / 4] >= 0 && j <= pos && j > see && j < end) seen |= 1u << i;
                    x[i] = seen >> i & 1 ? x[i] : -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, x[i]);
            if (__any(top > m + kLag)) {
                top = max_quarters(top);
                const float m2 = fmaxf(m, top), back = m2 == -INFINITY ? 1.f : exp2_fast(m - m2);
                m = m2;
                l *= back;
#pragma unroll
                for (int c = 0; c < NV; c++) o[c] *= back;
            }
            const float ref = m == -INFINITY ? 0.f : m - Prob<X, C>::up;
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w[i] = exp2_fast(x[i] - ref);
                l += w[i];
                if constexpr (Prob<X, C>::split) w[i] *= split_scale<C>(r.sv[i / 4][i % 4]).rest;
                else if constexpr (C::bytes == 1) w[i] *= r.sv[i / 4][i % 4];
            }
            if (C::bytes == 1 && !full) {
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = seen >> i & 1 ? w[i] : 0.f;  // a scale may be NaN there
            }
            Halves<P> p;
#pragma unroll
            for (int i = 0; i < 4; i++) p.add(i, w[2 * i], w[2 * i + 1]);
            return p;
        };
        const auto gather = [&](const Regs& r, const Halves<P>& p, uint32_t seen) {
            if constexpr (Prob<X, C>::split) {
#pragma unroll
                for (int j = 0; j < VD; j++) {  // four dimensions of eight keys, widened first: each key has its power
                    u32x2 x[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = widen4_by<C>(r.v[k][j], split_scale<C>(r.sv[k / 4][k % 4]).power);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        u32x4 w;
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] = __builtin_amdgcn_perm(x[2 * e + 1][k / 2], x[2 * e][k / 2], k % 2 ? 0x07060302u : 0x05040100u);
                        o[4 * j + k] = mfma16<P>(w, p.lo, mfma16<P>(w, p.hi, o[4 * j + k]));
                    }
                }
            } else if constexpr (C::bytes == 1) {
#pragma unroll
                for (int j = 0; j < VD; j++) {  // four dimensions of eight keys
                    uint32_t w[2][4];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t a0 = r.v[4 * h][j], a1 = r.v[4 * h + 1][j], a2 = r.v[4 * h + 2][j], a3 = r.v[4 * h + 3][j];
                        const uint32_t x0 = __builtin_amdgcn_perm(a1, a0, 0x05010400u), x1 = __builtin_amdgcn_perm(a1, a0, 0x07030602u);
                        const uint32_t y0 = __builtin_amdgcn_perm(a3, a2, 0x05010400u), y1 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
                        w[h][0] = __builtin_amdgcn_perm(y0, x0, 0x05040100u);
                        w[h][1] = __builtin_amdgcn_perm(y0, x0, 0x07060302u);
                        w[h][2] = __builtin_amdgcn_perm(y1, x1, 0x05040100u);
                        w[h][3] = __builtin_amdgcn_perm(y1, x1, 0x07060302u);
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const u32x2 w0 = widen4<C, P>(w[0][k]), w1 = widen4<C, P>(w[1][k]);
                        const u32x4 v = {w0[0], w0[1], w1[0], w1[1]};
                        o[4 * j + k] = mfma16<P>(v, p.lo, mfma16<P>(v, p.hi, o[4 * j + k]));
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < VD; j++) {  // two dimensions of eight keys
                    u32x4 w0, w1;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        w0[k] = __builtin_amdgcn_perm(r.v[2 * k + 1][j], r.v[2 * k][j], 0x05040100u);
                        w1[k] = __builtin_amdgcn_perm(r.v[2 * k + 1][j], r.v[2 * k][j], 0x07060302u);
                    }
                    // a float16 weight may have become 0 though every row sees the key (see settle; here it
                    // costs nothing to look: a step of 64 sequences to 16000, 344 us with and without)
                    if (__any((P::tag == CKR_F16 || seen != ~0u) && (any_wild<P>(w0) || any_wild<P>(w1)))) {
                        const u32x4 see = ones<P>(seen);
                        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                        const f32x4 p0 = mfma16<P>(wild<P>(w0, 1), see, zero), m0 = mfma16<P>(wild<P>(w0, -1), see, zero);
                        const f32x4 p1 = mfma16<P>(wild<P>(w1, 1), see, zero), m1 = mfma16<P>(wild<P>(w1, -1), see, zero);
#pragma unroll
                        for (int i = 0; i < 4; i++) o[2 * j][i] += wild_sum(p0[i], m0[i]), o[2 * j + 1][i] += wild_sum(p1[i], m1[i]);
                        w0 = wild<P>(w0, 0), w1 = wild<P>(w1, 0);
                    }
                    o[2 * j] = mfma16<P>(w0, p.lo, mfma16<P>(w0, p.hi, o[2 * j]));
                    o[2 * j + 1] = mfma16<P>(w1, p.lo, mfma16<P>(w1, p.hi, o[2 * j + 1]));
                }
            }
        };

        Regs r[2];
        int32_t pages[2][2], coming[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            if (u < n_tiles) {
                pages[u][0] = page_at(32 * u), pages[u][1] = page_at(32 * u + 16);
                load_k(r[u], 32 * u, pages[u]);
                load_v(r[u], 32 * u, pages[u]);
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) q[ks] ^= a.flip;
        for (int i = 0; i < n_tiles; i += 2) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if (i + u >= n_tiles) break;
                const int base = 32 * (i + u);
                const bool more = i + u + 2 < n_tiles;
                f32x4 s[2];
                scores(r[u], s);
                uint32_t seen;
                const Halves<P> p = weights(r[u], s, base, pages[u], seen);
                if (more) {  // its keys' registers again, for the tile after the next
                    coming[0] = page_at(base + 64), coming[1] = page_at(base + 80);
                    load_k(r[u], base + 64, coming);
                }
                gather(r[u], p, seen);
                if (more) {
                    pages[u][0] = coming[0], pages[u][1] = coming[1];
                    load_v(r[u], base + 64, pages[u]);
                }
            }
        }
        // ---- join: lane (col, g) holds dimensions 4 g NV .. 4 (g + 1) NV of row col
        l = sum_quarters(l);
        if (l != l && m == -INFINITY) m = 0.f;  // only NaN scores so far: not a row without keys
        __syncthreads();                        // the last item's sums have been read
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < NV; c += 4)
                *reinterpret_cast<f32x4*>(&s_o[wave][col][(4 * g + i) * NV + c]) = f32x4{o[c][i], o[c + 1][i], o[c + 2][i], o[c + 3][i]};
        if (g == 0) s_m[wave][col][0] = m, s_m[wave][col][1] = l;
        __syncthreads();
        const uint32_t n_rows = min(kFewRows, rows - row0);
        // the first n sums in LDS of a row's four outputs, joined
        const auto joined = [&](uint32_t n, uint32_t rr, uint32_t d, float& top, float& sum) {
            top = -INFINITY, sum = 0.f;
            for (uint32_t w = 0; w < n; w++) top = fmaxf(top, s_m[w][rr][0]);
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            for (uint32_t w = 0; w < n; w++) {
                const float mw = s_m[w][rr][0];
                if (mw == -INFINITY) continue;
                const float f = exp2_fast(mw - top);
                sum += s_m[w][rr][1] * f;
                v += *reinterpret_cast<const f32x4*>(&s_o[w][rr][d]) * f;
            }
            return v;
        };
        const auto write = [&](uint32_t rr, uint32_t d, f32x4 v, float top, float sum) {
            const uint32_t orow = row0 + rr, token = token0 + orow / a.group, head = kvh * a.group + orow % a.group;
            const float inv = top == -INFINITY ? 0.f : 1.f / sum;
            if (d < a.dim)
                *reinterpret_cast<u32x2*>(a.out + ((int64_t)token * a.o_tok + (int64_t)head * a.o_head + d) * 2) =
                    u32x2{pack16<X>(v[0] * inv, v[1] * inv), pack16<X>(v[2] * inv, v[3] * inv)};
            if (a.lse && d == 0) a.lse[(int64_t)token * a.heads + head] = top == -INFINITY ? -INFINITY : (top - Prob<X, C>::up + log2f(sum)) * kLn2;
        };
        const bool whole = t0 == 0 && t1 == nt;
        const uint64_t part = ((uint64_t)blockIdx.x * 2 + (t0 == 0)) * kFewRows;
        for (uint32_t e = threadIdx.x; e < n_rows * QUADS; e += THREADS) {
            const uint32_t rr = e / QUADS, d = e % QUADS * 4;
            float top, sum;
            const f32x4 v = joined(kFewWaves, rr, d, top, sum);
            if (whole) {
                write(rr, d, v, top, sum);
            } else {
                float* po = a.part_o + (part + rr) * DP + d;
                store_far(po, v[0], v[1]), store_far(po + 2, v[2], v[3]);
                if (d == 0) store_far(a.part_m + (part + rr) * 2, top, sum);
            }
        }
        if (!whole) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part has arrived
            __syncthreads();                                  // and the block's
            const uint32_t begin = p - t0, b_first = begin / per, parts = (begin + nt - 1) / per - b_first + 1;
            uint32_t* const counter = a.counters + b_first;  // one item at most begins in a block and goes on
            if (threadIdx.x == 0) {
                const uint32_t seen = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                s_last = seen + 1 == parts;
                if (seen + 1 == parts) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (s_last) {
                // the last block of the item's to finish joins its parts: groups of threads take
                // every so many of them each, four at a time (loads without branches, so that
                // they do not wait for each other), then the groups' sums are joined as the waves' were
                const uint32_t quads = n_rows * QUADS, groups = min(kFewWaves, max(THREADS / quads, 1u));
                const auto part_of = [&](uint32_t k) { return (uint64_t)(k == 0 ? b_first * 2 + 1 : (b_first + k) * 2) * kFewRows; };
                for (uint32_t e = threadIdx.x; e < groups * quads; e += THREADS) {
                    const uint32_t grp = e / quads, rr = e % quads / QUADS, d = e % QUADS * 4;
                    float top = -INFINITY, sum = 0.f;
                    f32x4 v = {0.f, 0.f, 0.f, 0.f};
                    for (uint32_t k = grp; k < parts; k += 4 * groups) {
                        f32x2 ml[4], x[4], y[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const uint64_t at = part_of(min(k + u * groups, parts - 1)) + rr;
                            ml[u] = load_far(a.part_m + at * 2);
                            x[u] = load_far(a.part_o + at * DP + d), y[u] = load_far(a.part_o + at * DP + d + 2);
                        }
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            if (k + u * groups >= parts || ml[u][0] == -INFINITY) continue;
                            const float top2 = fmaxf(top, ml[u][0]), f = exp2_fast(top - top2), f2 = exp2_fast(ml[u][0] - top2);
                            top = top2, sum = sum * f + ml[u][1] * f2;
                            v = v * f + f32x4{x[u][0], x[u][1], y[u][0], y[u][1]} * f2;
                        }
                    }
                    *reinterpret_cast<f32x4*>(&s_o[grp][rr][d]) = v;
                    if (d == 0) s_m[grp][rr][0] = top, s_m[grp][rr][1] = sum;
                }
                __syncthreads();
                for (uint32_t e = threadIdx.x; e < quads; e += THREADS) {
                    const uint32_t rr = e / QUADS, d = e % QUADS * 4;
                    float top, sum;
                    const f32x4 v = joined(groups, rr, d, top, sum);
                    write(rr, d, v, top, sum);
                }
            }
        }
        // ---- on to the next item
        p += t1 - t0;
        if (p >= p_end) break;
        t0 = 0;
        if (++kvh < a.kv_heads) continue;
        kvh = 0, row0 += kFewRows;
        while (row0 >= rows) {  // p < p_end: there is one
            const int32_t from = a.b.offsets[++seq], to = min(a.b.offsets[seq + 1], (int32_t)a.b.n_tokens);
            row0 = 0, rows = from >= 0 && to > from ? (uint32_t)(to - from) * a.group : 0;
            token0 = (uint32_t)from, start = a.b.starts[seq];
        }
        span = few_span(a, start, row0, rows), nt = few_tiles(span);
    }
}

// ------------------------------------------------------------ many rows
// A block takes BM = 128 rows, a wave 32 of them (32x32x16 matrix products), against
// tiles of TK keys staged through LDS in 16 bits, double buffered: while a tile is
// computed, the next one's bytes are on their way to registers, and the one
// after's page numbers too; 8-bit codes are widened once, when they are stored to LDS.
//   S^T = K Q^T: a lane holds one row (its column) and 16 of 32 keys, 8 (i / 4) + 4 h + i % 4
//   with h its half, so a row's maximum takes one exchange between two lanes;
//   O^T = V^T P^T: P's operand is again what the lane holds (eight keys of each 16);
//   V's is read transposed from LDS, four keys of one dimension at a time.
// Its keys are split over blocks where the tiles do not fill the card.  Bound by the
// latency of staging and, with few rows, by rows of zeros in the products: 32 tokens
// of 16 sequences over 4096 (128 rows a head, e4m3) 109 us, 0.32 PFLOP/s.  Over 16-bit
// caches, heads of 128, 5 or 6 registers spill, some of them in its loop (131 us).
template <typename C, int DP> struct ManyShape {
    static constexpr int TK = DP > 128 ? 32 : 64;
    // bytes of a row in LDS: 16-byte reads of 32 rows run at 206 bytes a cycle with
    // rows 16 bytes past a multiple of 256 (126 with 32, 16 with none), transposed
    // reads of 4 rows at 121 with rows 64 past it (114 with 32, 60 with 16)
    static constexpr int KP = DP * 2 + 16, VP = DP * 2 + 64;
    static constexpr int LPR = DP * C::bytes / 16, LOADS = TK * LPR / 256;  // lanes of a row, 16-byte loads a thread
    static constexpr int ROWS = 256 / LPR;                                  // rows a load of the block covers
};

template <typename X, typename C, int DP>
__global__ void __launch_bounds__(256, (DP > 128 ? 1 : 2)) attend_many_kernel(AttnArg a) {
    typedef typename ProbMany<X, C>::E P;
    typedef ManyShape<C, DP> Sh;
    constexpr int TK = Sh::TK, KP = Sh::KP, VP = Sh::VP, LPR = Sh::LPR, LOADS = Sh::LOADS, ROWS = Sh::ROWS;
    constexpr int KS = DP / 16, DT = DP / 32, TT = TK / 32;
    static_assert(LOADS >= 1 && TK * LPR % 256 == 0, "a tile is whole loads of the block");
    __shared__ __attribute__((aligned(16))) uint8_t s_k[2][TK * KP];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[2][TK * VP];
    __shared__ __attribute__((aligned(16))) float s_sk[2][TK];
    __shared__ __attribute__((aligned(16))) float s_sv[2][TK];
    __shared__ float s_most[2];  // the largest value scale of a tile
    __shared__ uint64_t s_valid[2];
    __shared__ uint32_t s_tmp[16], s_wild;  // s_wild: there is a value scale that is not finite
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
    const uint32_t kvh = blockIdx.x % a.kv_heads, tile = blockIdx.x / a.kv_heads, split = blockIdx.y;
    Tile t;
    if (threadIdx.x == 0) s_wild = 0;
    if (!find_tile<128>(a.b, a.group, tile, s_tmp, t)) return;
    const uint32_t row = t.row0 + wave * 32 + col;
    const int64_t pos_lo = t.start + t.row0 / a.group, pos_hi = t.start + min(t.row0 + 127, t.rows - 1) / a.group;
    const int64_t limit = min(pos_hi + 1, (int64_t)a.b.width << a.page_shift);
    const int64_t first = a.window ? max((int64_t)0, pos_lo - (int64_t)a.window + 1) & ~(int64_t)(TK - 1) : 0;
    const int64_t lo = first + (int64_t)split * a.split_len;
    const int64_t hi = split + 1 == a.splits ? limit : min(limit, lo + (int64_t)a.split_len);
    const int n_tiles = hi > lo ? (int)((hi - lo + TK - 1) / TK) : 0;
    // from here on keys are counted from lo, in 32 bits
    const auto rel = [&](int64_t p) { return (int)max((int64_t)-0x40000000, min(p - lo, (int64_t)0x7fffffff - 2 * TK)); };
    const uint32_t wave_row = __builtin_amdgcn_readfirstlane(t.row0 + wave * 32);
    const int end = rel(limit), pos = rel(t.start + min(row, t.rows - 1) / a.group);
    const int wave_lo = rel(t.start + min(wave_row, t.rows - 1) / a.group), wave_hi = rel(t.start + min(wave_row + 31, t.rows - 1) / a.group);
    // a row sees the keys above `see`; the wave's first and last row's bounds
    const int see = a.window ? rel(t.start + min(row, t.rows - 1) / a.group - (int64_t)a.window) : -0x40000000;
    const int see_lo = a.window ? rel(t.start + min(wave_row, t.rows - 1) / a.group - (int64_t)a.window) : -0x40000000;
    const int see_hi = a.window ? rel(t.start + min(wave_row + 31, t.rows - 1) / a.group - (int64_t)a.window) : -0x40000000;

    u32x4 q[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        const uint32_t d = ks * 16 + half * 8;
        q[ks] = u32x4{0, 0, 0, 0};
        if (row < t.rows && d < a.dim) {
            q[ks] = *reinterpret_cast<const u32x4*>(a.q + ((int64_t)(t.token0 + row / a.group) * a.q_tok +
                                                          (int64_t)(kvh * a.group + row % a.group) * a.q_head + d) * 2);
            q[ks] ^= a.flip;
        }
    }
    // staging: thread's rows r0 + u ROWS of a tile, 16 bytes at its place in the row
    const int32_t* table = a.b.table + (int64_t)t.seq * a.b.table_stride;
    const uint32_t r0 = threadIdx.x / LPR, piece = threadIdx.x % LPR;
    const bool d_in = piece * 16 / C::bytes < a.dim;
    const uint32_t slot_mask = (1u << a.page_shift) - 1;
    const int64_t c0 = lo >> a.page_shift;               // table column of lo, and lo's place in its page
    const uint32_t in0 = (uint32_t)lo & slot_mask;
    const auto page_id = [&](int j) {
        const int64_t c = c0 + ((in0 + (uint32_t)j) >> a.page_shift);
        const int32_t p = j < end && c < (int64_t)a.b.width ? table[c] : -1;
        return (uint32_t)p < a.n_pages ? p : -1;
    };
    int32_t pg[LOADS], pg_s = -1;  // pages of the rows of the tile that is loaded next; of key threadIdx for its scales
    const auto load_pages = [&](int base) {
#pragma unroll
        for (int u = 0; u < LOADS; u++) pg[u] = page_id(base + (int)r0 + u * ROWS);
        if (threadIdx.x < TK) pg_s = page_id(base + (int)threadIdx.x);
    };
    u32x4 kr[LOADS], vr[LOADS];
    float sk = 0.f, sv = 0.f, row_sv[LOADS];
    bool in_s = false;
    const auto load_tile = [&](int base) {
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            const int64_t slot = (in0 + (uint32_t)base + r0 + u * ROWS) & slot_mask;
            kr[u] = vr[u] = u32x4{0, 0, 0, 0};
            row_sv[u] = 0.f;
            if (pg[u] >= 0 && d_in) {
                kr[u] = *reinterpret_cast<const u32x4*>(a.ck + (int64_t)pg[u] * a.kst[0] + (int64_t)kvh * a.kst[1] + slot * a.kst[2] + piece * 16);
                vr[u] = *reinterpret_cast<const u32x4*>(a.cv + (int64_t)pg[u] * a.vst[0] + (int64_t)kvh * a.vst[1] + slot * a.vst[2] + piece * 16);
                if constexpr (ProbMany<X, C>::split) row_sv[u] = a.sv[(int64_t)pg[u] * a.svst[0] + (int64_t)kvh * a.svst[1] + slot];
            }
        }
        in_s = pg_s >= 0;
        if (C::bytes == 1 && in_s) {
            const int64_t slot = (in0 + (uint32_t)base + threadIdx.x) & slot_mask;
            sk = a.sk[(int64_t)pg_s * a.skst[0] + (int64_t)kvh * a.skst[1] + slot];
            sv = a.sv[(int64_t)pg_s * a.svst[0] + (int64_t)kvh * a.svst[1] + slot];
        }
    };
    const auto store_tile = [&](int buf) {
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            uint8_t* k = s_k[buf] + (r0 + u * ROWS) * KP;
            uint8_t* v = s_v[buf] + (r0 + u * ROWS) * VP;
            if constexpr (C::bytes == 2) {
                *reinterpret_cast<u32x4*>(k + piece * 16) = kr[u];
                *reinterpret_cast<u32x4*>(v + piece * 16) = vr[u];
            } else {
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const u32x2 x = widen4<C, X>(kr[u][2 * w]), y = widen4<C, X>(kr[u][2 * w + 1]);
                    *reinterpret_cast<u32x4*>(k + piece * 32 + w * 16) = u32x4{x[0], x[1], y[0], y[1]};
                    u32x2 z, zz;
                    if constexpr (ProbMany<X, C>::split) {
                        const float power = split_scale<C>(row_sv[u]).power;
                        z = widen4_by<C>(vr[u][2 * w], power), zz = widen4_by<C>(vr[u][2 * w + 1], power);
                    } else {
                        z = widen4<C, P>(vr[u][2 * w]), zz = widen4<C, P>(vr[u][2 * w + 1]);
                    }
                    *reinterpret_cast<u32x4*>(v + piece * 32 + w * 16) = u32x4{z[0], z[1], zz[0], zz[1]};
                }
            }
        }
        if (C::bytes == 1 && threadIdx.x < TK) {
            // a value scale that is not finite is 0 here, so that a weight of 0 (a key that
            // a row does not see) always gives 0, and the rows that see it are made NaN at the end
            const bool fine = abs_bits(sv) < 0x7f800000u;
            s_sk[buf][threadIdx.x] = in_s ? sk * a.scale2 : 0.f;
            s_sv[buf][threadIdx.x] = !in_s || !fine ? 0.f : ProbMany<X, C>::split ? split_scale<C>(sv).rest : sv;
            if (in_s && !fine) s_wild = 1;
        }
        if (threadIdx.x < 64) {
            const uint64_t ok = __ballot(in_s && lane < TK);
            if (lane == 0) s_valid[buf] = ok;
            if constexpr (ProbMany<X, C>::scaled) {
                const float most = max_quarters(max_row16(in_s && lane < TK && abs_bits(sv) < 0x7f800000u ? fabsf(sv) : 0.f));
                if (lane == 0) s_most[buf] = most;
            }
        }
    };

    float m = -INFINITY, l = 0.f, e = ProbMany<X, C>::scaled ? kLeast : 0.f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[dt][i] = 0.f;
    // where this lane reads V: 4 keys x 16 dimensions per group of 16 lanes
    const uint32_t v_lane = (4 * half + (lane & 15) / 4) * VP + (16 * ((lane >> 4) & 1) + (lane & 3) * 4) * 2;

    // full: every row of the wave sees every key of the tile
    const auto compute = [&](bool full, int buf, int base, uint64_t valid) {
        f32x16 s[TT];
#pragma unroll
        for (int tt = 0; tt < TT; tt++) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[tt][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const u32x4 k = *reinterpret_cast<const u32x4*>(s_k[buf] + (tt * 32 + col) * KP + ks * 32 + half * 16);
                s[tt] = mfma32<X>(k, q[ks], s[tt]);
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < TT; tt++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                if constexpr (C::bytes == 1) {
                    const f32x4 f = *reinterpret_cast<const f32x4*>(&s_sk[buf][tt * 32 + 2 * i + 4 * half]);
#pragma unroll
                    for (int k = 0; k < 4; k++) s[tt][i + k] *= f[k];
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) s[tt][i + k] *= a.scale2;
                }
            }
        uint32_t seen[TT];
        bool care = false;
        if (!full) {
            valid >>= 4 * half;
            const int k0 = base + 4 * half;
#pragma unroll
            for (int tt = 0; tt < TT; tt++) {
                seen[tt] = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int key = tt * 32 + 8 * (i / 4) + i % 4;
                    const bool in = (valid >> key & 1) && k0 + key <= pos && k0 + key > see;
                    if constexpr (C::bytes == 2) seen[tt] |= in ? 1u << i : 0u;
                    s[tt][i] = in ? s[tt][i] : -INFINITY;
                }
            }
            if constexpr (C::bytes == 2) {  // is there an infinity or NaN among the values
#pragma unroll
                for (int u = 0; u < TK * DP / 8 / 64; u++) {
                    const uint32_t e = u * 64 + lane;
                    care |= any_wild<P>(*reinterpret_cast<const u32x4*>(s_v[buf] + e / (DP / 8) * VP + e % (DP / 8) * 16));
                }
                care = __any(care);
            }
        }
#pragma unroll
        for (int tt = 0; tt < TT; tt++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, s[tt][i]);
        top = max_half(top);
        const float e2 = ProbMany<X, C>::scaled ? fmaxf(e, scale_power(s_most[buf])) : 0.f;
        if (__any(top > m + kLag || e2 > e)) {
            const float m2 = fmaxf(m, top), back = m2 == -INFINITY ? 1.f : exp2_fast(m - m2 + (e - e2));
            m = m2, e = e2;
            l *= back;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[dt][i] *= back;
        }
        const float ref = m == -INFINITY ? 0.f : m - ProbMany<X, C>::up + e;
#pragma unroll
        for (int tt = 0; tt < TT; tt++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                float p[8];
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        p[i + k] = exp2_fast(s[tt][8 * kb + i + k] - ref);
                        l += p[i + k];
                    }
                    if constexpr (C::bytes == 1) {
                        const f32x4 f = *reinterpret_cast<const f32x4*>(&s_sv[buf][tt * 32 + 16 * kb + 2 * i + 4 * half]);
#pragma unroll
                        for (int k = 0; k < 4; k++) p[i + k] *= f[k];
                    }
                }
                Halves<P> w;  // the second for float16 queries over 8 bits only
#pragma unroll
                for (int i = 0; i < 4; i++) w.add(i, p[2 * i], p[2 * i + 1]);
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    typedef short s16x4 __attribute__((ext_vector_type(4)));
                    typedef __attribute__((address_space(3))) s16x4* lds4;
                    const uint8_t* at = s_v[buf] + (tt * 32 + kb * 16) * VP + v_lane + dt * 64;
                    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at));
                    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * VP));
                    const u32x2 xa = __builtin_bit_cast(u32x2, x), ya = __builtin_bit_cast(u32x2, y);
                    u32x4 v = {xa[0], xa[1], ya[0], ya[1]};
                    if (C::bytes == 2 && care) {
                        const u32x4 see8 = ones<P>(seen[tt] >> (8 * kb));
                        f32x16 zero;
#pragma unroll
                        for (int i = 0; i < 16; i++) zero[i] = 0.f;
                        const f32x16 plus = mfma32<P>(wild<P>(v, 1), see8, zero), minus = mfma32<P>(wild<P>(v, -1), see8, zero);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[dt][i] += wild_sum(plus[i], minus[i]);
                        v = wild<P>(v, 0);
                    }
                    o[dt] = mfma32<P>(v, w.hi, o[dt]);
                    if constexpr (ProbMany<X, C>::split) o[dt] = mfma32<P>(v, w.lo, o[dt]);
                }
            }
    };

    if (n_tiles > 0) {
        load_pages(0);
        load_tile(0);
        load_pages(TK);
        store_tile(0);
        __syncthreads();
        for (int i = 0; i < n_tiles; i++) {
            const int base = i * TK;
            if (i + 1 < n_tiles) {
                load_tile(base + TK);
                load_pages(base + 2 * TK);
            }
            if (base <= wave_hi && base + TK - 1 > see_lo) {  // some row sees some key
                const uint64_t valid = s_valid[i & 1];
                const bool full = valid == (TK == 64 ? ~0ull : (1ull << TK % 64) - 1) && base + TK - 1 <= wave_lo && base > see_hi;
                compute(__builtin_amdgcn_readfirstlane(full), i & 1, base, valid);
            }
            if (i + 1 < n_tiles) store_tile((i + 1) & 1);
            __syncthreads();
        }
    }
    l = sum_half(l);
    m += e;  // what sums are held against, from here on
    if (l != l && m == -INFINITY) m = 0.f;  // only NaN scores so far: not a row without keys
    if constexpr (C::tag == CKR_F16)
        if (any_nan(o)) settle<P, DP, 128>(tile_found<128, 256>(a.group, s_tmp), kvh, row, o);
    if (C::bytes == 1 && s_wild && sees_wild_scale<128>(a, tile_found<128, 256>(a.group, s_tmp), kvh, row)) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[dt][i] = as_f32(0x7fc00000u);
    }
    if (row >= t.rows) return;
    if (a.splits > 1) {
        const uint64_t p = (((uint64_t)tile * a.kv_heads + kvh) * a.splits + split) * 128 + wave * 32 + col;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(a.part_o + p * DP + dt * 32 + 2 * i + 4 * half) = f32x4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
        if (half == 0) a.part_m[p * 2] = m, a.part_m[p * 2 + 1] = l;
        return;
    }
    const uint32_t token = t.token0 + row / a.group, head = kvh * a.group + row % a.group;
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    uint8_t* out = a.out + ((int64_t)token * a.o_tok + (int64_t)head * a.o_head) * 2;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const uint32_t d = dt * 32 + 2 * i + 4 * half;
            if (d < a.dim)
                *reinterpret_cast<u32x2*>(out + d * 2) = u32x2{pack16<X>(o[dt][i] * inv, o[dt][i + 1] * inv), pack16<X>(o[dt][i + 2] * inv, o[dt][i + 3] * inv)};
        }
    if (a.lse && half == 0) a.lse[(int64_t)token * a.heads + head] = m == -INFINITY ? -INFINITY : (m - ProbMany<X, C>::up + log2f(l)) * kLn2;
}

// ------------------------------------------------------------ very many rows
// A block of eight waves takes 256 rows, a wave 32 of them, two waves a SIMD.  With
// S(i) the scores of the i-th 32 keys and P(i) their weights, a wave's turn i is
//   S(i+1) = K(i+1) Q  and  O += V(i-1) P(i-1)  on the matrix cores, beside
//   P(i) = exp(S(i) - maximum so far)           on the vector units,
// three things that do not wait for each other, written as 16 steps of a matrix
// product, the reads of LDS for the products three steps on, and one score's
// weight, in that order.  What bounds it is the issue of vector instructions (four
// and a half per score and lane; and float16 products take 6 to 8 percent longer than
// bfloat16 ones in otherwise the same code), so the maximum is not looked for at each turn:
// weights are taken against the maximum so far, and only where the sum of a lane's
// comes out above 2^kLag, or a row has no maximum yet, is the turn's softmax made
// again.
// Tiles of 64 keys go through a ring of four in LDS (the turns of a tile still read
// the last half of the one before and the first half of the one after, while the
// next but one is stored): waves 0 to 3 stage the keys, 4 to 7 the values.  A wave's
// rows of a tile lie in one page (16 slots at least), so addresses are the page's,
// in scalar registers, and an offset that never changes.
// 2048 tokens behind 30000 in e4m3, 32 query heads: 1.10 to 1.13 ms from card to card,
// 0.94 PFLOP/s (a large library product reaches 1.36); six prompts of 150 to 3000 tokens
// in float16, 64 query heads: 490 to 505 us, 0.69 PFLOP/s: a block is alone on its CU
// and takes one tile of rows, so of the 50 us that one takes on average the 12 until
// its first product runs beside nothing.
template <typename C, int DP> struct WideShape {
    static constexpr int TK = 64, BM = 256, RING = 4;
    static constexpr int KP = DP * 2 + 16, VP = DP * 2 + 64;  // as ManyShape's
    static constexpr int LPR = DP * C::bytes / 16, LOADS = TK * LPR / 256;  // lanes of a row, loads of a thread
    static constexpr int RPW = 64 / LPR, ROWS = 256 / LPR;                  // rows of a wave's load, of four waves'
};

template <typename X, typename C, int DP>
__global__ void __launch_bounds__(512, 2) attend_wide_kernel(AttnArg a) {
    typedef typename ProbMany<X, C>::E P;
    typedef WideShape<C, DP> Sh;
    constexpr int TK = Sh::TK, KP = Sh::KP, VP = Sh::VP, LPR = Sh::LPR, LOADS = Sh::LOADS, RPW = Sh::RPW, ROWS = Sh::ROWS;
    constexpr int KS = DP / 16, DT = DP / 32, NM = 2 * KS;  // KS products for the scores, as many for the values
    static_assert(KS == 2 * DT && KS % 4 == 0, "pairs of products, operands in rings of four");
    constexpr bool kScaled = ProbMany<X, C>::scaled;
    constexpr float kMost = ProbMany<X, C>::up == 0.f ? 256.f : ProbMany<X, C>::up == 6.f ? 16384.f : 32768.f;  // 2^(kLag + up)
    __shared__ __attribute__((aligned(16))) uint8_t s_k[Sh::RING * TK * KP];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[Sh::RING * TK * VP];
    constexpr int SCALES = C::bytes == 1 ? TK : 1;
    __shared__ __attribute__((aligned(16))) float s_sk[Sh::RING + 1][SCALES];  // the last: ones, for scores that carry their scale
    __shared__ __attribute__((aligned(16))) float s_sv[Sh::RING][SCALES + (kScaled ? 4 : 0)];  // and the largest of each 16
    __shared__ __attribute__((aligned(16))) uint8_t s_zero[C::bytes == 2 ? 32 * VP : 16];  // values of zero
    __shared__ uint32_t s_tmp[16], s_wild;  // s_wild: as in the 128-row kernel
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const uint32_t kvh = blockIdx.x % a.kv_heads, tile = blockIdx.x / a.kv_heads, split = blockIdx.y;
    Tile t;
    if (threadIdx.x == 0) s_wild = 0;
    if (!find_tile<Sh::BM, 512>(a.b, a.group, tile, s_tmp, t)) return;
    const int64_t pos_lo = t.start + t.row0 / a.group, pos_hi = t.start + min(t.row0 + Sh::BM - 1, t.rows - 1) / a.group;
    const int64_t limit = min(pos_hi + 1, (int64_t)a.b.width << a.page_shift);
    const int64_t first = a.window ? max((int64_t)0, pos_lo - (int64_t)a.window + 1) & ~(int64_t)(TK - 1) : 0;
    const int64_t lo = first + (int64_t)split * a.split_len;
    const int64_t hi = split + 1 == a.splits ? limit : min(limit, lo + (int64_t)a.split_len);
    const int n_tiles = __builtin_amdgcn_readfirstlane(hi > lo ? (int)((hi - lo + TK - 1) / TK) : 0);
    // from here on keys are counted from lo, in 32 bits
    const auto rel = [&](int64_t p) { return (int)max((int64_t)-0x40000000, min(p - lo, (int64_t)0x7fffffff - 8 * TK)); };
    const uint32_t wave_row = t.row0 + wave * 32, row = wave_row + col;
    const int end = __builtin_amdgcn_readfirstlane(rel(limit));
    const int wave_lo = __builtin_amdgcn_readfirstlane(rel(t.start + min(wave_row, t.rows - 1) / a.group));
    const int see_hi = __builtin_amdgcn_readfirstlane(
        a.window ? rel(t.start + min(wave_row + 31, t.rows - 1) / a.group - (int64_t)a.window) : -0x40000000);
    const int64_t my_pos = t.start + min(row, t.rows - 1) / a.group;
    const int pos = rel(my_pos), see = a.window ? rel(my_pos - (int64_t)a.window) : -0x40000000;
    u32x4 q[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        const uint32_t d = ks * 16 + half * 8;
        q[ks] = u32x4{0, 0, 0, 0};
        if (row < t.rows && d < a.dim) {
            q[ks] = *reinterpret_cast<const u32x4*>(a.q + ((int64_t)(t.token0 + row / a.group) * a.q_tok +
                                                          (int64_t)(kvh * a.group + row % a.group) * a.q_head + d) * 2);
        }
    }
    // staging.  A key of no mapped page is read from page 0 and then cleared (values)
    // or masked (scores); pieces past the head's size are the last piece again: of
    // values, and of codes, which are finite and meet queries of zero.  A 16-bit key may
    // hold an infinity, so there the lanes past it store to the 16 bytes between two
    // rows of LDS, which nobody reads, and the pieces themselves stay zero
    typedef __attribute__((address_space(4))) const int32_t* const_i32;
    const const_i32 table = (const_i32)(a.b.table + (int64_t)__builtin_amdgcn_readfirstlane(t.seq) * a.b.table_stride);
    const bool stage_k = wave < 4;
    const uint32_t w4 = wave & 3, row_of = w4 * RPW + lane / LPR, place = lane % LPR;
    const uint32_t piece = min(place, a.dim * C::bytes / 16 - 1);
    const uint32_t slot_mask = (1u << a.page_shift) - 1;
    const uint32_t st0 = (uint32_t)((stage_k ? a.kst[0] : a.vst[0]) >> 4), st2 = (uint32_t)((stage_k ? a.kst[2] : a.vst[2]) >> 4);
    const uint8_t* const from = stage_k ? a.ck + (int64_t)kvh * a.kst[1] : a.cv + (int64_t)kvh * a.vst[1];
    const uint32_t from_lane = ((row_of & 15) * st2 + piece) * 16, w4_rows = w4 * RPW / 16 * 16;
    const float* const scale_k = a.sk + (int64_t)kvh * a.skst[1];
    const float* const scale_v = a.sv + (int64_t)kvh * a.svst[1];
    const uint32_t to_place = C::bytes == 2 && stage_k && place != piece ? DP * 2 : place * (C::bytes == 1 ? 32 : 16);
    uint8_t* const to = (stage_k ? s_k + row_of * KP : s_v + row_of * VP) + to_place;
    const uint32_t to_rows = ROWS * (stage_k ? KP : VP), to_slot = TK * (stage_k ? KP : VP);
    const uint32_t c0 = (uint32_t)(lo >> a.page_shift), in0 = (uint32_t)lo & slot_mask, last_col = a.b.width - 1;
    // the page of the 16 keys from j (a multiple of 16) on; -1: none
    const auto page_id = [&](int j) {
        const int32_t p = table[min(c0 + ((in0 + (uint32_t)j) >> a.page_shift), last_col)];
        return ((j < end) & ((uint32_t)p < a.n_pages)) ? p : -1;  // end lies within the table
    };
    // a tile is part of one page, or of several small ones
    const bool one_page = a.page_shift >= 6;
    int32_t pg[4] = {-1, -1, -1, -1};  // of the tile that is loaded next (of all of it in pg[0])
    uint64_t valid[4];  // keys of mapped pages: of this tile, and of the next three
    const auto load_pages = [&](int base) {
        if (one_page) {
            pg[0] = page_id(base);
            return;
        }
        // pages of 16 or 32 slots: the tile starts with one, four columns from it on hold its pages
        const uint32_t c = c0 + ((uint32_t)base >> a.page_shift);
        if (base + TK <= end && c + 3 <= last_col) {
            const int32_t p[4] = {table[c], table[c + 1], table[c + 2], table[c + 3]};
            const bool small = a.page_shift == 4;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int32_t x = small ? p[g] : p[g / 2];
                pg[g] = (uint32_t)x < a.n_pages ? x : -1;
            }
        } else {
#pragma unroll
            for (int g = 0; g < 4; g++) pg[g] = page_id(base + 16 * g);
        }
    };
    const auto valid_of = [&](int base) {
        if (base + TK <= end && (one_page ? pg[0] : pg[0] | pg[1] | pg[2] | pg[3]) >= 0) return ~0ull;
        uint64_t v = 0;
#pragma unroll
        for (int g = 0; g < 4; g++) v |= pg[one_page ? 0 : g] >= 0 ? 0xffffull << (16 * g) : 0;
        return end - base >= TK ? v : end - base <= 0 ? 0 : v & ((1ull << (end - base)) - 1);
    };
    u32x4 held[LOADS];
    float sk = 0.f, sv = 0.f, row_sv[LOADS];  // row_sv: of the rows held, where values are widened by their scale's power
    uint64_t held_valid = 0;
    const auto load_tile = [&](int base) {
        if (one_page) {
            const uint32_t p = (uint32_t)max(pg[0], 0), slot = (in0 + (uint32_t)base) & slot_mask;
            const uint8_t* at = from + ((uint64_t)p * st0 + (uint64_t)slot * st2) * 16;
#pragma unroll
            for (int u = 0; u < LOADS; u++) held[u] = *reinterpret_cast<const u32x4*>(at + (from_lane + (w4_rows + u * ROWS) * st2 * 16));
            if constexpr (ProbMany<X, C>::split) {
                const float* f = scale_v + ((int64_t)p * a.svst[0] + slot) + row_of;
#pragma unroll
                for (int u = 0; u < LOADS; u++) row_sv[u] = f[u * ROWS];
            }
        } else {
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const uint32_t g = (w4 * RPW + u * ROWS) / 16;
                const uint32_t p = (uint32_t)max(g == 0 ? pg[0] : g == 1 ? pg[1] : g == 2 ? pg[2] : pg[3], 0);
                const uint32_t slot = (in0 + (uint32_t)base + 16 * g) & slot_mask;
                held[u] = *reinterpret_cast<const u32x4*>(from + ((uint64_t)p * st0 + (uint64_t)slot * st2) * 16 + from_lane);
                if constexpr (ProbMany<X, C>::split) row_sv[u] = (scale_v + ((int64_t)p * a.svst[0] + slot))[row_of & 15];
            }
        }
        if constexpr (C::bytes == 1) {
            const int32_t p = max(one_page || w4 == 0 ? pg[0] : w4 == 1 ? pg[1] : w4 == 2 ? pg[2] : pg[3], 0);
            const uint32_t slot = (in0 + (uint32_t)base + 16 * w4) & slot_mask;
            sk = (scale_k + ((int64_t)p * a.skst[0] + slot))[lane & 15];
            sv = (scale_v + ((int64_t)p * a.svst[0] + slot))[lane & 15];
        }
        held_valid = valid_of(base);
    };
    const auto store_rows = [&](int u, int slot) {
        u32x4 x = held[u];
        if (!stage_k && held_valid != ~0ull) {
            const bool in = held_valid >> (row_of + u * ROWS) & 1;
            x = in ? x : u32x4{0, 0, 0, 0};
        }
        uint8_t* at = to + slot * to_slot + u * to_rows;
        if constexpr (C::bytes == 2) {
            *reinterpret_cast<u32x4*>(at) = x;
        } else if (stage_k || (!ProbMany<X, C>::split && !kScaled)) {
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const u32x2 y = widen4<C, X>(x[2 * w]), z = widen4<C, X>(x[2 * w + 1]);
                *reinterpret_cast<u32x4*>(at + w * 16) = u32x4{y[0], y[1], z[0], z[1]};
            }
        } else if (kScaled) {
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const u32x2 y = widen4<C, P>(x[2 * w]), z = widen4<C, P>(x[2 * w + 1]);
                *reinterpret_cast<u32x4*>(at + w * 16) = u32x4{y[0], y[1], z[0], z[1]};
            }
        } else {
            const float power = split_scale<C>(row_sv[u]).power;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const u32x2 y = widen4_by<C>(x[2 * w], power), z = widen4_by<C>(x[2 * w + 1], power);
                *reinterpret_cast<u32x4*>(at + w * 16) = u32x4{y[0], y[1], z[0], z[1]};
            }
        }
    };
    const auto store_scales = [&](int slot) {  // four lanes write the same values
        if constexpr (C::bytes == 1) {
            if (stage_k) {
                s_sk[slot][16 * w4 + (lane & 15)] = sk * a.scale2;
            } else {  // as in the 128-row kernel
                const bool fine = abs_bits(sv) < 0x7f800000u, in = held_valid >> (16 * w4 + (lane & 15)) & 1;
                const float x = in && fine ? sv : 0.f;
                s_sv[slot][16 * w4 + (lane & 15)] = ProbMany<X, C>::split && in && fine ? split_scale<C>(sv).rest : x;
                if constexpr (kScaled) s_sv[slot][TK + w4] = max_row16(fabsf(x));
                if (in && !fine) s_wild = 1;
            }
        }
    };

    float m = -INFINITY, l = 0.f, ref = 0.f, e = kScaled ? kLeast : 0.f;
    f32x16 o[DT], s;
    u32x4 pf[2][2], kf[4], vf[4];  // weights of two turns; operands, read three pairs of steps ahead
    f32x4 fk[2], fv[2];            // the keys' scales, of keys 8 j + 4 half on
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[dt][i] = 0.f;
    const uint32_t k_lane = col * KP + half * 16;
    const uint32_t v_lane = (4 * half + (lane & 15) / 4) * VP + (16 * ((lane >> 4) & 1) + (lane & 3) * 4) * 2;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* lds4;
    const auto k_at = [&](int slot, int sub) { return s_k + slot * (TK * KP) + sub * 32 * KP + k_lane; };
    const auto v_at = [&](int slot, int sub) { return s_v + slot * (TK * VP) + sub * 32 * VP + v_lane; };
    const auto read_k = [&](int e, const uint8_t* at) { kf[e % 4] = *reinterpret_cast<const u32x4*>(at + e * 32); };
    const auto read_v = [&](int e, const uint8_t* at) {
        at += e / DT * 16 * VP + e % DT * 64;
        const u32x2 u = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at)));
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * VP)));
        vf[e % 4] = u32x4{u[0], u[1], w[0], w[1]};
    };
    const auto read_scales = [&](int j, const float* at_fk, const float* at_fv) {
        if constexpr (C::bytes == 1) {
            fk[j % 2] = *reinterpret_cast<const f32x4*>(at_fk + 8 * j + 4 * half);
            fv[j % 2] = *reinterpret_cast<const f32x4*>(at_fv + 8 * j + 4 * half);
        }
    };
    const auto weight = [&](int k, f32x4 g, float f) {
        return exp2_fast(__builtin_fmaf(s[k], C::bytes == 1 ? g[k % 4] : f, -ref));
    };
    // scores that some row of the wave must not see: scaled here, -inf where hidden.
    // 16-bit values: is there an infinity or NaN among them (care), and who sees which
    // key; those keys' values are then gathered apart, and zeros by the next turn
    uint32_t seen = 0;
    bool care = false;
    const auto mask = [&](const float* at_fk, const uint8_t* at_v, int base, uint32_t valid) __attribute__((always_inline)) {
        valid >>= 4 * half;
        const int k0 = base + 4 * half;
        seen = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int key = 8 * (i / 4) + i % 4;
            const float f = C::bytes == 1 ? at_fk[key + 4 * half] : a.scale2;
            const bool in = (valid >> key & 1) && k0 + key <= pos && k0 + key > see;
            if constexpr (C::bytes == 2) seen |= in ? 1u << i : 0u;
            s[i] = in ? s[i] * f : -INFINITY;
        }
        if constexpr (C::bytes == 2) {
#pragma unroll
            for (int u = 0; u < 32 * DP / 8 / 64; u++) {
                const uint32_t e = u * 64 + lane;
                care |= any_wild<P>(*reinterpret_cast<const u32x4*>(at_v + e / (DP / 8) * VP + e % (DP / 8) * 16));
            }
            care = __any(care);
        }
    };
    const auto gather_with_care = [&](const u32x4 (&w)[2], const uint8_t* at) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < KS; e++) {
            const uint8_t* row = at + e / DT * 16 * VP + e % DT * 64;
            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(row)));
            const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(row + 8 * VP)));
            const u32x4 v = {x[0], x[1], y[0], y[1]}, see8 = ones<P>(seen >> (8 * (e / DT)));
            f32x16 zero;
#pragma unroll
            for (int i = 0; i < 16; i++) zero[i] = 0.f;
            const f32x16 plus = mfma32<P>(wild<P>(v, 1), see8, zero), minus = mfma32<P>(wild<P>(v, -1), see8, zero);
            o[e % DT] = mfma32<P>(wild<P>(v, 0), w[e / DT], o[e % DT]);
#pragma unroll
            for (int i = 0; i < 16; i++) o[e % DT][i] += wild_sum(plus[i], minus[i]);
        }
    };
    struct Where { const uint8_t *k, *v; const float *fk, *fv; };  // what a turn reads: K(i+1), V(i-1), scales(i)
    const auto turn = [&](auto sub_tag, float f, const Where& now, const Where& after, auto side) {
        constexpr int sub = decltype(sub_tag)::value;
        f32x16 z;
#pragma unroll
        for (int i = 0; i < 16; i++) z[i] = 0.f;
        float sum = 0.f, p_even = 0.f, p_last = 0.f;
        f32x2 scales = {0.f, 0.f};
        if constexpr (kScaled) scales = *reinterpret_cast<const f32x2*>(now.fv + TK - 30 * sub);  // s_sv's last four from this half's first
        const auto use = [&](auto k_tag) {
            constexpr int k = decltype(k_tag)::value;
            sum += p_last;
            if constexpr (k % 2 == 0) {
                p_even = C::bytes == 1 ? p_last * fv[k / 4 % 2][k % 4] : p_last;
            } else {
                uint32_t w = pack16<P>(p_even, C::bytes == 1 ? p_last * fv[k / 4 % 2][k % 4] : p_last);
                asm volatile("" : "+v"(w));
                pf[sub][k / 8][k % 8 / 2] = w;
            }
        };
        unroll<16>([&](auto step_tag) {
            constexpr int S = decltype(step_tag)::value;
            if constexpr (S % (16 / NM) == 0) {
                constexpr int j = S * NM / 16, e = j / 2;
                if constexpr (j % 2 == 0) {
                    o[e % DT] = mfma32<P>(vf[e % 4], pf[1 - sub][e / DT], o[e % DT]);
                    if constexpr (e + 3 < KS) read_v(e + 3, now.v);
                    else read_v(e + 3 - KS, after.v);
                } else {
                    z = mfma32<X>(kf[e % 4], q[e], z);
                    if constexpr (e + 3 < KS) read_k(e + 3, now.k);
                    else read_k(e + 3 - KS, after.k);
                }
            }
            // a weight is used a step after its exponential
            const float p = weight(S, fk[S / 4 % 2], f);
            if constexpr (S > 0) use(std::integral_constant<int, S - 1>{});
            if constexpr (S % 4 == 1) {  // the last group's scales have been used
                if constexpr (S < 12) read_scales(S / 4 + 1, now.fk, now.fv);
                else read_scales(0, after.fk, after.fv);
            }
            side(step_tag);
            p_last = p;
            __builtin_amdgcn_sched_barrier(0);
        });
        use(std::integral_constant<int, 15>{});
        asm volatile("" : "+v"(sum));
        const float e2 = kScaled ? fmaxf(e, scale_power(fmaxf(scales[0], scales[1]))) : 0.f;
        const float most_sum = kScaled ? as_f32(as_u32(kMost) - ((uint32_t)(int)e << 23)) : kMost;  // kMost 2^-e
        if (__any(sum > most_sum || m == -INFINITY || e2 > e)) {
            float most = -INFINITY;
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
                const f32x4 g = C::bytes == 1 ? *reinterpret_cast<const f32x4*>(now.fk + 2 * k + 4 * half) : f32x4{f, f, f, f};
#pragma unroll
                for (int i = 0; i < 4; i++) most = fmaxf(most, s[k + i] * g[i]);
            }
            most = max_half(most);
            const float m2 = fmaxf(m, most), back = m2 == -INFINITY ? 1.f : exp2_fast(m - m2 + (e - e2));
            m = m2, e = e2;
            ref = m2 == -INFINITY ? 0.f : m2 - ProbMany<X, C>::up + e;
            l *= back;
            sum = 0.f;
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
                f32x4 g = {f, f, f, f}, gv = {1.f, 1.f, 1.f, 1.f};
                if constexpr (C::bytes == 1) {
                    g = *reinterpret_cast<const f32x4*>(now.fk + 2 * k + 4 * half);
                    gv = *reinterpret_cast<const f32x4*>(now.fv + 2 * k + 4 * half);
                }
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p[i] = weight(k + i, g, f);
                    sum += p[i];
                }
                pf[sub][k / 8][k % 8 / 2] = pack16<P>(p[0] * gv[0], p[1] * gv[1]);
                pf[sub][k / 8][k % 8 / 2 + 1] = pack16<P>(p[2] * gv[2], p[3] * gv[3]);
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[dt][i] *= back;
        }
        l += sum;
        asm volatile("" : "+v"(l));
        s = z;
    };

    if (n_tiles > 0) {
        if (C::bytes == 1 && wave == 0) s_sk[Sh::RING][lane] = 1.f;
        if constexpr (C::bytes == 2)
            for (uint32_t e = threadIdx.x; e < 32 * VP / 16; e += 512) *reinterpret_cast<u32x4*>(s_zero + e * 16) = u32x4{0, 0, 0, 0};
        if (C::bytes == 2 && a.dim < DP)
            for (uint32_t r = threadIdx.x; r < Sh::RING * TK; r += 512)
                for (uint32_t d = a.dim; d < DP; d += 8) *reinterpret_cast<u32x4*>(s_k + r * KP + d * 2) = u32x4{0, 0, 0, 0};
        // the first three tiles: their pages, then their rows, all on their way at once
        int32_t pages[3][4];
#pragma unroll
        for (int i = 0; i < 3; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) pages[i][g] = table[min(c0 + ((in0 + (uint32_t)(i * TK + 16 * g)) >> a.page_shift), last_col)];
#pragma unroll
        for (int i = 0; i < 3; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) pages[i][g] = ((i * TK + 16 * g < end) & ((uint32_t)pages[i][g] < a.n_pages)) ? pages[i][g] : -1;
        u32x4 rows[3][LOADS];
        float scales[3][2], row_scales[3][LOADS];
#pragma unroll
        for (int i = 0; i < 3; i++) {
#pragma unroll
            for (int g = 0; g < 4; g++) pg[g] = pages[i][g];
            load_tile(i * TK);
            valid[i] = held_valid;
#pragma unroll
            for (int u = 0; u < LOADS; u++) rows[i][u] = held[u], row_scales[i][u] = row_sv[u];
            scales[i][0] = sk, scales[i][1] = sv;
        }
#pragma unroll
        for (int i = 0; i < 3; i++) {
#pragma unroll
            for (int u = 0; u < LOADS; u++) held[u] = rows[i][u], row_sv[u] = row_scales[i][u];
            sk = scales[i][0], sv = scales[i][1], held_valid = valid[i];
            if (i == 2) break;
#pragma unroll
            for (int u = 0; u < LOADS; u++) store_rows(u, i);
            store_scales(i);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) q[ks] ^= a.flip;
        load_pages(3 * TK);
        __syncthreads();
        const auto full_at = [&](uint64_t v, int base) {
            return (uint32_t)(v >> (base & 32)) == 0xffffffffu && base + 31 <= wave_lo && base > see_hi;
        };
        bool full = full_at(valid[0], 0);
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
        for (int e = 0; e < KS; e++) {
            read_k(e, k_at(0, 0));
            s = mfma32<X>(kf[e % 4], q[e], s);
        }
        // turn 0 has no values before it: what it gathers is dropped after it
        pf[1][0] = pf[1][1] = u32x4{0, 0, 0, 0};
        Where now = {k_at(0, 1), v_at(0, 0), s_sk[full ? 0 : Sh::RING], s_sv[0]};
#pragma unroll
        for (int e = 0; e < 3; e++) read_k(e, now.k), read_v(e, now.v);
        read_scales(0, now.fk, now.fv);
        for (int i = 0; i < n_tiles; i++) {
            const int cur = i & 3, next = (i + 1) & 3, third = (i + 2) & 3;
            unroll<2>([&](auto sub_tag) {
                constexpr int sub = decltype(sub_tag)::value;
                const int base = i * TK + sub * 32;
                if (C::bytes == 2 && care) {
                    gather_with_care(pf[1 - sub], now.v);
                    now.v = s_zero + v_lane;
#pragma unroll
                    for (int e = 0; e < 3; e++) vf[e] = u32x4{0, 0, 0, 0};
                    care = false;
                }
                if (!full) mask(s_sk[cur] + sub * 32, s_v + cur * (TK * VP) + sub * 32 * VP, base, (uint32_t)(valid[0] >> (32 * sub)));
                const float f = full ? a.scale2 : 1.f;
                const bool full2 = full_at(valid[sub], base + 32);
                const int slot2 = sub ? next : cur;
                const Where after = {k_at(next, sub), v_at(cur, sub), s_sk[full2 ? slot2 : Sh::RING] + (1 - sub) * 32,
                                     s_sv[slot2] + (1 - sub) * 32};
                turn(sub_tag, f, now, after, [&](auto step_tag) {
                    constexpr int S = decltype(step_tag)::value;
                    if constexpr (sub == 0) {  // the next tile but one into LDS
                        if constexpr (S % 2 == 0 && S >= 4 && S / 2 - 2 < LOADS) store_rows(S / 2 - 2, third);
                        else if constexpr (S == 15) store_scales(third);
                    } else {  // the one after it on its way, and its successor's pages
                        if constexpr (S == 0) load_tile(i * TK + 3 * TK);
                        else if constexpr (S == 4) {
                            valid[3] = held_valid;
                            load_pages(i * TK + 4 * TK);
                        }
                    }
                });
                if (sub == 0 && i == 0) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int k = 0; k < 16; k++) o[dt][k] = 0.f;
                }
                now = after;
                full = full2;
            });
            valid[0] = valid[1], valid[1] = valid[2], valid[2] = valid[3];
            __syncthreads();
        }
        // the last turn's values: its first three operands have been read
        if (C::bytes == 2 && care) gather_with_care(pf[1], now.v);
        else
#pragma unroll
        for (int e = 0; e < KS; e++) {
            if (e + 3 < KS) read_v(e + 3, now.v);
            o[e % DT] = mfma32<P>(vf[e % 4], pf[1][e / DT], o[e % DT]);
        }
    }
    l = sum_half(l);
    m += e;  // what sums are held against, from here on
    if (l != l && m == -INFINITY) m = 0.f;  // only NaN scores so far: not a row without keys
    if constexpr (C::tag == CKR_F16)
        if (any_nan(o)) settle<P, DP, Sh::BM>(tile_found<Sh::BM, 512>(a.group, s_tmp), kvh, row, o);
    if (C::bytes == 1 && s_wild && sees_wild_scale<Sh::BM>(a, tile_found<Sh::BM, 512>(a.group, s_tmp), kvh, row)) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[dt][i] = as_f32(0x7fc00000u);
    }
    if (row >= t.rows) return;
    if (a.splits > 1) {
        const uint64_t p = (((uint64_t)tile * a.kv_heads + kvh) * a.splits + split) * Sh::BM + wave * 32 + col;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(a.part_o + p * DP + dt * 32 + 2 * i + 4 * half) = f32x4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
        if (half == 0) a.part_m[p * 2] = m, a.part_m[p * 2 + 1] = l;
        return;
    }
    const uint32_t token = t.token0 + row / a.group, head = kvh * a.group + row % a.group;
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    uint8_t* out = a.out + ((int64_t)token * a.o_tok + (int64_t)head * a.o_head) * 2;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const uint32_t d = dt * 32 + 2 * i + 4 * half;
            if (d < a.dim)
                *reinterpret_cast<u32x2*>(out + d * 2) = u32x2{pack16<X>(o[dt][i] * inv, o[dt][i + 1] * inv), pack16<X>(o[dt][i + 2] * inv, o[dt][i + 3] * inv)};
        }
    if (a.lse && half == 0) a.lse[(int64_t)token * a.heads + head] = m == -INFINITY ? -INFINITY : (m - ProbMany<X, C>::up + log2f(l)) * kLn2;
}

// ------------------------------------------------------------ the splits' join
// The splits of a row, in their order: 4 dimensions a thread.  Bound by the launch and
// by reading the parts (4 bytes a dimension and split), which are at most 512 tiles of
// 128 rows or 256 of 256: 34 MB for heads of 128, still in the last cache.
template <typename X, int DP, uint32_t BM>
__global__ void __launch_bounds__(256) attend_join_kernel(AttnArg a, float up) {
    __shared__ uint32_t s_tmp[16];
    const uint32_t kvh = blockIdx.x % a.kv_heads, tile = blockIdx.x / a.kv_heads;
    Tile t;
    if (!find_tile<BM>(a.b, a.group, tile, s_tmp, t)) return;
    constexpr uint32_t PER = 256 / (DP / 4);  // rows of a block
    const uint32_t rr = blockIdx.y * PER + threadIdx.x / (DP / 4), d = threadIdx.x % (DP / 4) * 4, row = t.row0 + rr;
    if (rr >= BM || row >= t.rows) return;
    const uint64_t part = ((uint64_t)tile * a.kv_heads + kvh) * a.splits * BM + rr;
    float top = -INFINITY, sum = 0.f;
    for (uint32_t s = 0; s < a.splits; s++) top = fmaxf(top, a.part_m[(part + (uint64_t)s * BM) * 2]);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t s = 0; s < a.splits; s++) {
        const uint64_t p = part + (uint64_t)s * BM;
        const float ms = a.part_m[p * 2];
        if (ms == -INFINITY) continue;
        const float f = exp2_fast(ms - top);
        sum += a.part_m[p * 2 + 1] * f;
        v += *reinterpret_cast<const f32x4*>(a.part_o + p * DP + d) * f;
    }
    const uint32_t token = t.token0 + row / a.group, head = kvh * a.group + row % a.group;
    const float inv = top == -INFINITY ? 0.f : 1.f / sum;  // both carry 2^up
    if (d < a.dim)
        *reinterpret_cast<u32x2*>(a.out + ((int64_t)token * a.o_tok + (int64_t)head * a.o_head + d) * 2) =
            u32x2{pack16<X>(v[0] * inv, v[1] * inv), pack16<X>(v[2] * inv, v[3] * inv)};
    if (a.lse && d == 0) a.lse[(int64_t)token * a.heads + head] = top == -INFINITY ? -INFINITY : (top - up + log2f(sum)) * kLn2;
}
// ------------------------------------------------------------ the launch
// How a batch is cut: rows of a tile, tiles (an upper bound: each sequence's last
// tile may be short), key ranges of a tile.
struct Cut {
    uint32_t bm, dp, tiles, splits, split_len, blocks, min_tiles;
    uint64_t part_m_bytes, bytes;  // of the workspace: counters, the rows' maxima and sums, their outputs
};
constexpr uint64_t kSplitMin = 128;   // keys of a split at least
// Blocks of the few rows' kernel: two a CU.  (For heads of 256 its registers leave room
// for one, so there a full launch runs in two rounds.)
constexpr uint32_t kFewBlocks = 512;
// Its tiles of 32 keys a block at least: one a wave (one token over a thousand: 9.5 us;
// 11.0 with 8, 13.5 with 16).
constexpr uint32_t kFewTiles = 4;
// Rows of a chunk up to which it is taken, in tiles of 16 that each read the cache; us,
// few / many rows, e4m3, 8 heads of 128: 32 rows of 16 sequences over 4096 tokens 53 / 78, of one
// over 32768 42 / 79, of 64 over 1024 51 / 58; 64 rows of 64 over 1024 96 / 60, of 16
// over 4096 66 / 104.
constexpr uint32_t kFewMost = 32;
// Rows from which on a tile of 256 pays: 128 rows of 16 sequences over 4096 tokens 110
// (many) / 144 (very many), 256 rows 158 / 148; 256 of one over 32768 102 / 100; float16
// caches 129 / 111 and 184 / 115.
constexpr uint32_t kManyMost = 128;
// Blocks that the card holds at once: two of 128 rows a CU (of heads of 256 one), one of 256.
uint64_t blocks_wanted(uint32_t bm) { return bm == kManyRows ? 512 : 256; }
uint32_t padded_dim(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
uint64_t most_tiles(uint32_t bm, uint64_t group, uint64_t n_seqs, uint64_t n_tokens) {
    return std::min(n_tokens * group / bm + std::min(n_seqs, n_tokens), n_tokens * ((group + bm - 1) / bm));
}
// The workspace begins with the counters, whatever else a call keeps in it: they
// are 0 between calls, the rest is not.
constexpr uint64_t kCounterBytes = kFewBlocks * 4;
void set_bytes(Cut& c, uint64_t rows) {
    c.part_m_bytes = (rows * 8 + 255) / 256 * 256;
    c.bytes = kCounterBytes + c.part_m_bytes + rows * c.dp * 4;
}
uint32_t few_blocks(uint64_t items, uint64_t max_context) {
    return (uint32_t)std::min<uint64_t>(items * ((max_context + 31) / 32) / kFewTiles + 1, kFewBlocks);
}
// Rows of parts that a workspace holds (calls keep multiples of 32, which set_bytes rounds no further).
uint64_t rows_held(uint64_t bytes, uint32_t dp) { return bytes < kCounterBytes ? 0 : (bytes - kCounterBytes) / (8 + dp * 4); }
// workspace: its bytes; blocks and splits that it does not hold are left out, down to
// one block of few rows and no split.
Cut cut(uint32_t n_heads, uint32_t n_kv, uint32_t dim, uint32_t n_seqs, uint32_t n_tokens, uint32_t max_chunk,
        uint64_t max_context, uint64_t all_keys, uint32_t window, bool near_slots, uint64_t workspace) {
    Cut c{};
    const uint64_t group = n_heads / n_kv, rows = (uint64_t)max_chunk * group;
    c.dp = padded_dim(dim);
    const bool few = rows <= kFewMost && most_tiles(kFewRows, group, n_seqs, n_tokens) * n_kv * ((all_keys + 31) / 32 + 1) < (1ull << 31);
    c.bm = few ? kFewRows : rows <= kManyMost || c.dp == 256 || !near_slots ? kManyRows : kWideRows;
    c.tiles = (uint32_t)most_tiles(c.bm, group, n_seqs, n_tokens);
    c.splits = 1;
    // the keys of a tile: a window's, and as many again as the tile has tokens
    if (window) max_context = std::min<uint64_t>(max_context, (uint64_t)window + c.bm / group + 64);
    const uint64_t items = std::max<uint64_t>((uint64_t)c.tiles * n_kv, 1);
    if (c.bm == kFewRows) {
        c.min_tiles = kFewTiles;
        c.blocks = (uint32_t)std::clamp<uint64_t>(rows_held(workspace, c.dp) / (2 * kFewRows), 1, few_blocks(items, max_context));
        set_bytes(c, (uint64_t)c.blocks * 2 * kFewRows);
        return c;
    }
    const uint64_t most = std::max<uint64_t>((max_context + kSplitMin - 1) / kSplitMin, 1);
    const uint64_t splits = std::min({blocks_wanted(c.bm) / items, most, rows_held(workspace, c.dp) / (items * c.bm)});
    if (splits > 1) {
        c.split_len = (uint32_t)((max_context + splits * kSplitMin - 1) / (splits * kSplitMin) * kSplitMin);  // half of 2^32 at most
        c.splits = (uint32_t)((max_context + c.split_len - 1) / c.split_len);
        if (c.splits > 1) set_bytes(c, items * c.splits * c.bm);
    }
    return c;
}
// What cut() asks for at most, for any batch up to these sizes.
uint64_t most_bytes(uint32_t n_heads, uint32_t n_kv, uint32_t dim, uint32_t n_seqs, uint32_t n_tokens, uint64_t max_context) {
    const uint64_t group = n_heads / n_kv;
    Cut c{};
    c.dp = padded_dim(dim);
    uint64_t items = std::max<uint64_t>(most_tiles(kFewRows, group, n_seqs, n_tokens) * n_kv, 1);
    set_bytes(c, (uint64_t)few_blocks(items, max_context) * 2 * kFewRows);
    uint64_t most = c.bytes;
    for (const uint32_t bm : {kManyRows, kWideRows}) {
        items = most_tiles(bm, group, n_seqs, n_tokens) * n_kv;
        set_bytes(c, std::min(blocks_wanted(bm), items * ((max_context + kSplitMin - 1) / kSplitMin)) * bm);
        if (max_context > kSplitMin) most = std::max(most, c.bytes);
    }
    return most;
}

template <typename X, typename C, int DP>
hipError_t launch_attend(const AttnArg& a, const Cut& c, hipStream_t s) {
    const dim3 grid(a.tiles * a.kv_heads, c.splits);
    const auto join = [&](auto kernel) {
        if (c.splits <= 1) return;
        const uint32_t per = 256 / (DP / 4);
        CKR_LAUNCH("kv_attention_join", s, kernel<<<dim3(a.tiles * a.kv_heads, (c.bm + per - 1) / per), 256, 0, s>>>(a, ProbMany<X, C>::up));
    };
    if (c.bm == kFewRows) {
        CKR_LAUNCH("kv_attention_few", s, attend_few_kernel<X, C, DP><<<dim3(c.blocks), 64 * kFewWaves, 0, s>>>(a));
    } else if (c.bm == kManyRows) {
        CKR_LAUNCH("kv_attention_many", s, attend_many_kernel<X, C, DP><<<grid, 256, 0, s>>>(a));
        join(attend_join_kernel<X, DP, kManyRows>);
    } else if constexpr (DP <= 128) {
        CKR_LAUNCH("kv_attention_wide", s, attend_wide_kernel<X, C, DP><<<grid, 512, 0, s>>>(a));
        join(attend_join_kernel<X, DP, kWideRows>);
    }
    return hipGetLastError();
}
template <typename X, typename C>
hipError_t launch_attend_dim(const AttnArg& a, const Cut& c, hipStream_t s) {
    if (c.dp == 64) return launch_attend<X, C, 64>(a, c, s);
    if (c.dp == 128) return launch_attend<X, C, 128>(a, c, s);
    return launch_attend<X, C, 256>(a, c, s);
}

}  // namespace
}  // namespace ckr

using namespace ckr;

extern "C" {

uint64_t ckr_kv_attention_workspace_bytes(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t n_seqs,
                                          uint32_t n_tokens, uint32_t max_chunk, uint32_t max_context) {
    if (n_kv_heads == 0 || n_heads == 0 || n_heads % n_kv_heads || head_dim == 0 || head_dim > 256) return 0;
    return most_bytes(n_heads, n_kv_heads, head_dim, n_seqs, n_tokens, max_context);
}

int ckr_kv_attention(const ckr_kv_cache* cache, const ckr_kv_batch* batch, const void* d_q, int64_t q_token_stride,
                     int64_t q_head_stride, int dtype, uint32_t n_heads, float scale, uint32_t window, void* d_out,
                     int64_t out_token_stride, int64_t out_head_stride, float* d_lse, void* d_workspace,
                     uint64_t workspace_bytes, void* stream) {
    int rc;
    if ((rc = kv_check_cache(cache)) || (rc = kv_check_batch(cache, batch))) return rc;
    if (dtype != CKR_BF16 && dtype != CKR_F16)
        return err(CKR_E_INVALID, "queries are of bfloat16 or float16, not dtype " + std::to_string(dtype));
    if ((cache->dtype == CKR_BF16 || cache->dtype == CKR_F16) && cache->dtype != dtype)
        return err(CKR_E_INVALID, "a 16-bit cache must be of the queries' type");
    if (n_heads == 0 || n_heads > 65535 || n_heads % cache->n_heads)
        return err(CKR_E_INVALID, std::to_string(n_heads) + " query heads: a multiple of the cache's " + std::to_string(cache->n_heads));
    if (!std::isfinite(scale)) return err(CKR_E_INVALID, "scale must be finite");
    if ((uint64_t)batch->n_tokens * n_heads > (1ull << 27)) return err(CKR_E_INVALID, "at most 2^27 rows (tokens x query heads)");
    if (batch->n_tokens == 0) return CKR_OK;
    if ((rc = kv_check_rows(d_q, batch->n_tokens, q_token_stride, n_heads, q_head_stride, cache->head_dim, 2, false, "queries")) ||
        (rc = kv_check_rows(d_out, batch->n_tokens, out_token_stride, n_heads, out_head_stride, cache->head_dim, 2, true, "output")))
        return rc;
    if (d_lse) {
        if (reinterpret_cast<uintptr_t>(d_lse) % 4) return err(CKR_E_INVALID, "lse must be aligned to 4 bytes");
        if ((rc = check_range(d_lse, (uint64_t)batch->n_tokens * n_heads * 4, "lse"))) return rc;
    }
    AttnArg a{};
    a.q = static_cast<const uint8_t*>(d_q), a.out = static_cast<uint8_t*>(d_out), a.lse = d_lse;
    a.q_tok = q_token_stride, a.q_head = q_head_stride, a.o_tok = out_token_stride, a.o_head = out_head_stride;
    a.ck = static_cast<const uint8_t*>(cache->d_k), a.cv = static_cast<const uint8_t*>(cache->d_v);
    a.sk = cache->d_k_scale, a.sv = cache->d_v_scale;
    const int ces = cache->dtype == CKR_F8 || cache->dtype == CKR_I8 ? 1 : 2;
    for (int i = 0; i < 3; i++) a.kst[i] = cache->k_stride[i] * ces, a.vst[i] = cache->v_stride[i] * ces;
    std::copy(cache->k_scale_stride, cache->k_scale_stride + 2, a.skst);
    std::copy(cache->v_scale_stride, cache->v_scale_stride + 2, a.svst);
    a.n_pages = cache->n_pages, a.page_shift = (uint32_t)__builtin_ctz(cache->page_size), a.dim = cache->head_dim;
    a.heads = n_heads, a.kv_heads = cache->n_heads, a.group = n_heads / cache->n_heads, a.window = window;
    // a scale of 0 makes every weight equal, as any scale that leaves no bit of a
    // score above 1 does; 0 itself would turn masked scores (-inf) into NaN
    a.scale2 = std::max(std::fabs(scale) * kLog2e, 0x1p-120f), a.flip = scale < 0.f ? 0x80008000u : 0u;
    a.b = {batch->d_page_table, batch->d_starts, batch->d_offsets, (int64_t)batch->table_stride, batch->table_width,
           batch->n_seqs, batch->n_tokens};
    // the slots of a page within 32-bit offsets of each other, pages within 2^36 bytes
    bool near_slots = true;
    for (const int64_t* st : {a.kst, a.vst}) near_slots = near_slots && st[2] < (1ll << 26) - 16 && (cache->n_pages == 1 || st[0] < (1ll << 36));
    const Cut c = cut(n_heads, cache->n_heads, cache->head_dim, batch->n_seqs, batch->n_tokens, batch->max_chunk,
                      std::min<uint64_t>(batch->max_context, (uint64_t)batch->table_width * cache->page_size),
                      (uint64_t)batch->table_width * cache->page_size, window, near_slots, workspace_bytes);
    if ((uint64_t)c.tiles * cache->n_heads * 512 > 0xffffffffull) return err(CKR_E_INVALID, "the batch is too large for one launch");
    a.tiles = c.tiles, a.splits = c.splits, a.split_len = c.split_len, a.min_tiles = c.min_tiles;
    if (c.bytes) {
        if (workspace_bytes < c.bytes)
            return err(CKR_E_CAPACITY, "workspace of " + std::to_string(workspace_bytes) + " bytes, " + std::to_string(c.bytes) + " needed");
        if (reinterpret_cast<uintptr_t>(d_workspace) % 256) return err(CKR_E_INVALID, "workspace must be aligned to 256 bytes");
        if ((rc = check_range(d_workspace, c.bytes, "workspace"))) return rc;
        a.counters = static_cast<uint32_t*>(d_workspace);
        a.part_m = reinterpret_cast<float*>(static_cast<uint8_t*>(d_workspace) + kCounterBytes);
        a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(d_workspace) + kCounterBytes + c.part_m_bytes);
    }
    const hipStream_t s = (hipStream_t)stream;
    hipError_t e;
    if (dtype == CKR_BF16)
        e = cache->dtype == CKR_F8   ? launch_attend_dim<ElemBF16, ElemF8>(a, c, s)
            : cache->dtype == CKR_I8 ? launch_attend_dim<ElemBF16, ElemI8>(a, c, s)
                                     : launch_attend_dim<ElemBF16, ElemBF16>(a, c, s);
    else
        e = cache->dtype == CKR_F8   ? launch_attend_dim<ElemF16, ElemF8>(a, c, s)
            : cache->dtype == CKR_I8 ? launch_attend_dim<ElemF16, ElemI8>(a, c, s)
                                     : launch_attend_dim<ElemF16, ElemF16>(a, c, s);
    return e == hipSuccess ? CKR_OK : err(CKR_E_HIP, std::string("HIP error in kv_attention: ") + hipGetErrorString(e));
}

}  // extern "C"
