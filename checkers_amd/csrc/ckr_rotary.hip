// checkers_amd/csrc/ckr_rotary.hip — rotary positions: heads turned by their tokens'
// positions (ckr_rotate, forward and backward), a chunk's keys turned on their way into a
// paged cache (ckr_kv_append), and the rows of a cache of 4 bits read back.
#include <algorithm>
#include <cmath>
#include <string>

#include "ckr_internal.h"
#include "ckr_kv.h"

namespace ckr {

int kv_check_cache(const ckr_kv_cache* c);
int kv_check_batch(const ckr_kv_cache* c, const ckr_kv_batch* b);
int kv_check_rows(const void* p, uint64_t rows, int64_t row_stride, uint64_t heads, int64_t head_stride, uint64_t dim,
                  int es, bool written, const char* what);
int kv_check_rows_apart(const ckr_kv_cache* c);

namespace {

int err(int code, const std::string& m) { return set_error(code, "[ckr] " + m); }
int hip_rc(hipError_t e, const char* what) {
    return e == hipSuccess ? CKR_OK : err(CKR_E_HIP, std::string("HIP error in ") + what + ": " + hipGetErrorString(e));
}

// ---- angles.  A pair's frequency is its turns a position, a fraction of 64 bits; its
// product with the position wraps at whole turns by itself, so angles of far positions
// are as good as near ones (off by 2^-65 of a turn a position).  What is left after the
// nearest quarter is at most pi / 4, where the Taylor series to x^15 and x^16 are off
// by less than 2^-53; in 64 bits, which this card multiplies as fast as 32, and
// rounded once, so that cosine and sine are those of a table computed in 64 bits.
struct Rot {
    const uint64_t* turns;
    double magnitude;
    uint32_t pairs, half;  // half: where the second of a pair lies (0: beside the first)
};
__device__ __forceinline__ f32x2 cos_sin(uint64_t phase, double magnitude) {
    const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
    const double x = (double)(int64_t)(phase - ((uint64_t)quarter << 62)) * (6.283185307179586476925 * 0x1p-64), z = x * x;
    double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
    s = __builtin_fma(s, z, 1.0 / 6227020800.0), c = __builtin_fma(c, z, -1.0 / 87178291200.0);
    s = __builtin_fma(s, z, -1.0 / 39916800.0), c = __builtin_fma(c, z, 1.0 / 479001600.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0), c = __builtin_fma(c, z, -1.0 / 3628800.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0), c = __builtin_fma(c, z, 1.0 / 40320.0);
    s = __builtin_fma(s, z, 1.0 / 120.0), c = __builtin_fma(c, z, -1.0 / 720.0);
    s = __builtin_fma(s, z, -1.0 / 6.0), c = __builtin_fma(c, z, 1.0 / 24.0);
    c = __builtin_fma(c, z, -0.5);
    s = __builtin_fma(s * z, x, x), c = __builtin_fma(c, z, 1.0);
    const double a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;  // cos, sin up to their signs
    return f32x2{(float)((quarter == 1 || quarter == 2 ? -a : a) * magnitude), (float)((quarter >= 2 ? -b : b) * magnitude)};
}

// Pairs (x, y) turned: (x c - y s, y c + x s), each product and sum rounded by itself, as
// in 32-bit operations one by one: codes made of the result are then those of the formula.
__device__ __forceinline__ float turned_first(float x, float y, float c, float s) {
#pragma clang fp contract(off)
    return x * c - y * s;
}
__device__ __forceinline__ float turned_second(float x, float y, float c, float s) {
#pragma clang fp contract(off)
    return y * c + x * s;
}

// ---- how tokens' rows are cut into blocks.  A thread keeps its row (a head) and its place in it
// for all of its block's tokens, so that the products of strides are made once a thread or
// once a token (whose share lies in LDS), not for each row, and several tokens' rows can be
// loaded before the first is used.
constexpr uint32_t kThreads = 512;                // of a block at most
constexpr uint32_t kMostTokens = 64;              // of a block
constexpr uint32_t kMostAngles = 32768;           // bytes of LDS for them
constexpr uint64_t kMostBlocks = (1u << 23) - 1;  // a grid holds fewer than 2^32 threads
struct RowCut {
    uint32_t shift;        // log2 of the lanes of a row
    uint32_t slab, slabs;  // rows of a token that a block takes, blocks of a token
    uint32_t sub, passes;  // tokens side by side, and one after another
    uint32_t threads;
    uint64_t blocks;
};
RowCut row_cut(uint64_t tokens, uint64_t rows, uint32_t lanes, uint32_t pairs, uint32_t passes) {
    RowCut c{};
    while ((1u << c.shift) < lanes) c.shift++;
    c.slabs = (uint32_t)(((rows << c.shift) + kThreads - 1) / kThreads);
    c.slab = (uint32_t)((rows + c.slabs - 1) / c.slabs);
    const uint32_t most = std::min(kMostTokens, kMostAngles / std::max((pairs + 7) / 8 * 64, 1u));
    c.sub = std::clamp(256u / (c.slab << c.shift), 1u, most);
    c.threads = ((c.sub * c.slab << c.shift) + 63) / 64 * 64;
    // one after another where there are blocks enough all the same: they share the look-ups and angles, and
    // the lines that neighbouring tokens' scales lie in
    c.passes = (uint32_t)std::clamp<uint64_t>(tokens * c.slabs / c.sub / 2048, 1, std::min(passes, most / c.sub));
    c.blocks = (tokens + c.sub * c.passes - 1) / (c.sub * c.passes) * c.slabs;
    return c;
}
struct Mine { uint32_t sub, row, lane; bool in; };
__device__ __forceinline__ Mine my_row(const RowCut& c) {
    const uint32_t item = threadIdx.x >> c.shift, sub = item / c.slab;
    return {sub, blockIdx.x % c.slabs * c.slab + (item - sub * c.slab), threadIdx.x & ((1u << c.shift) - 1), sub < c.sub};
}
// Cosines and sines of n tokens in LDS, `padded` pairs a token (a multiple of 8); position(t): of token t.
template <typename F> __device__ __forceinline__ void make_angles(f32x2* to, const Rot& rot, uint32_t n, F position, bool inverse) {
    const uint32_t padded = (rot.pairs + 7) & ~7u;
    for (uint32_t i = threadIdx.x; i < n * padded; i += blockDim.x) {
        const uint32_t t = i / padded, pair = i - t * padded;
        f32x2 cs = {1.f, 0.f};
        if (pair < rot.pairs) cs = cos_sin((uint64_t)(int64_t)position(t) * rot.turns[pair], rot.magnitude);
        if (inverse) cs.y = -cs.y;
        to[i] = cs;
    }
}

// ------------------------------------------------------------ rotate
struct Heads {
    const uint8_t* in;
    uint8_t* out;
    int64_t in_st[3], out_st[3];  // batch, token, head
    uint32_t heads, copy;         // copy: values behind the pairs go to `out` too
};
struct RotateArg {
    Rot rot;
    const int32_t* positions;
    int64_t pos_st[2];
    Heads x[2];
    uint32_t n_tokens;  // batch x tokens
    uint32_t tokens, dim, chunks, inverse;
    RowCut cut;
};

// Eight values as they lie in memory (at any address), and unpacked: rows of several tokens are
// loaded before the first of them is used.
template <typename E> struct Raw {
    typename Vecs<false>::U4 v[E::bytes / 2];
    __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
        for (int i = 0; i < E::bytes / 2; i++) v[i] = reinterpret_cast<const typename Vecs<false>::U4*>(p)[i];
    }
    __device__ __forceinline__ void get(float* x) const { load_vec<E, 8, false>(&v, x); }
};
template <typename E> constexpr int kAhead = E::bytes == 2 ? 4 : 2;  // tokens whose rows are loaded at once

template <typename E, int N> __device__ __forceinline__ void load_some(const uint8_t* p, uint32_t n, float* x) {
    if (n >= N) {
        load_vec<E, N, false>(p, x);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = (uint32_t)i < n ? load_one<E>(p, i) : 0.f;
    }
}
template <typename E, int N> __device__ __forceinline__ void store_some(uint8_t* p, uint32_t n, const float* x) {
    if (n >= N) {
        store_vec<E, N, false>(p, x);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if ((uint32_t)i < n) store_one<E>(p, i, x[i]);
    }
}

// Bound by memory: queries and keys of 16384 tokens, 40 heads of 128 in bfloat16, 335 MB in 64 us (5.2 TB/s, a
// copy's rate; 75 with one token's rows loaded at a time); 5997 tokens of 24 heads of 80 in float32, the first 20
// turned, 92 MB in 31 us (3 TB/s: a row of 320 bytes takes six of its eight lanes).  Threads that took tokens side
// by side and heads one after another measured the same or worse for heads that lie before tokens.
template <typename E> __global__ void __launch_bounds__(kThreads) rotate_kernel(RotateArg a) {
    extern __shared__ __attribute__((aligned(16))) f32x2 s_cs[];
    __shared__ int64_t s_at[kMostTokens][4];  // a token's place in the inputs and outputs
    const RowCut& c = a.cut;
    const uint32_t per = c.sub * c.passes, token0 = blockIdx.x / c.slabs * per, n = min(per, a.n_tokens - token0);
    const uint32_t padded = (a.rot.pairs + 7) & ~7u;
    if (threadIdx.x < n) {
        const uint32_t token = token0 + threadIdx.x, b = token / a.tokens, t = token - b * a.tokens;
#pragma unroll
        for (int x = 0; x < 2; x++) {
            s_at[threadIdx.x][2 * x] = ((int64_t)b * a.x[x].in_st[0] + (int64_t)t * a.x[x].in_st[1]) * E::bytes;
            s_at[threadIdx.x][2 * x + 1] = ((int64_t)b * a.x[x].out_st[0] + (int64_t)t * a.x[x].out_st[1]) * E::bytes;
        }
    }
    make_angles(s_cs, a.rot, n, [&](uint32_t i) {
        const uint32_t token = token0 + i, b = token / a.tokens;
        return a.positions[(int64_t)b * a.pos_st[0] + (int64_t)(token - b * a.tokens) * a.pos_st[1]];
    }, a.inverse);
    __syncthreads();
    const Mine me = my_row(c);
    const uint32_t turned = (a.rot.pairs + 7) / 8, w = me.row >= a.x[0].heads, head = me.row - (w ? a.x[0].heads : 0);
    if (!me.in || me.lane >= a.chunks || me.row >= a.x[0].heads + a.x[1].heads) return;
    const bool rest = me.lane >= turned;  // values behind the pairs
    if (rest && !(w ? a.x[1].copy : a.x[0].copy)) return;
    // 8 pairs, or 16 values behind them: the last ones end with the row (some are then done twice, alike,
    // by lanes of one wave, whose loads come before their stores), `left` of them where a row has fewer
    const uint32_t half = a.rot.half, behind = a.dim - 2 * a.rot.pairs, at = (me.lane - (rest ? turned : 0)) * (rest ? 16 : 8);
    const uint32_t all = rest ? behind : a.rot.pairs, size = rest ? 16 : 8;
    const bool back = all >= size && c.shift <= 6;
    const uint32_t pair = back ? min(at, all - size) : at, left = all - pair;
    const uint32_t d = rest ? 2 * a.rot.pairs + pair : half ? pair : 2 * pair;
    const uint8_t* const in0 = (w ? a.x[1].in : a.x[0].in) + ((int64_t)head * (w ? a.x[1].in_st[2] : a.x[0].in_st[2]) + d) * E::bytes;
    uint8_t* const out0 = (w ? a.x[1].out : a.x[0].out) + ((int64_t)head * (w ? a.x[1].out_st[2] : a.x[0].out_st[2]) + d) * E::bytes;
    const auto put = [&](uint32_t t, const float* f) {
        float y[16];
        const f32x2* cs = s_cs + t * padded + pair;
        uint8_t* const out = out0 + s_at[t][2 * w + 1];
        if (half) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                y[k] = turned_first(f[k], f[8 + k], cs[k].x, cs[k].y);
                y[8 + k] = turned_second(f[k], f[8 + k], cs[k].x, cs[k].y);
            }
            store_some<E, 8>(out, left, y), store_some<E, 8>(out + half * E::bytes, left, y + 8);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                y[2 * k] = turned_first(f[2 * k], f[2 * k + 1], cs[k].x, cs[k].y);
                y[2 * k + 1] = turned_second(f[2 * k], f[2 * k + 1], cs[k].x, cs[k].y);
            }
            store_some<E, 16>(out, 2 * left, y);
        }
    };
    if (left < size) {
        for (uint32_t t = me.sub; t < n; t += c.sub) {
            const uint8_t* const in = in0 + s_at[t][2 * w];
            float f[16];
            if (rest) {
                load_some<E, 16>(in, left, f);
                store_some<E, 16>(out0 + s_at[t][2 * w + 1], left, f);
            } else {
                if (half) load_some<E, 8>(in, left, f), load_some<E, 8>(in + half * E::bytes, left, f + 8);
                else load_some<E, 16>(in, 2 * left, f);
                put(t, f);
            }
        }
        return;
    }
    const uint32_t second = (half && !rest ? half : 8) * E::bytes;
    for (uint32_t t = me.sub; t < n; t += kAhead<E> * c.sub) {
        Raw<E> x[kAhead<E>][2];
#pragma unroll
        for (int u = 0; u < kAhead<E>; u++) {  // behind the last token it once more
            const uint8_t* const in = in0 + s_at[min(t + u * c.sub, n - 1)][2 * w];
            x[u][0].load(in), x[u][1].load(in + second);
        }
#pragma unroll
        for (int u = 0; u < kAhead<E>; u++) {
            if (t + u * c.sub >= n) break;
            float f[16];
            x[u][0].get(f), x[u][1].get(f + 8);
            if (rest) store_vec<E, 16, false>(out0 + s_at[t + u * c.sub][2 * w + 1], f);
            else put(t + u * c.sub, f);
        }
    }
}

// ------------------------------------------------------------ rows of a cache
struct AppendArg {
    Rot rot;                   // pairs 0: nothing is turned
    const int32_t* positions;  // of the angles, NULL: the cache's
    uint8_t* x[3];             // queries, keys, values
    uint8_t* q_out;
    int64_t tok[3], head[3], o_tok, o_head;
    uint8_t* cache[2];
    void* scales[2];
    int64_t st[2][3], sst[2][2];  // of rows in bytes, of scales in elements
    uint32_t n_pages, page_shift, q_heads, heads, dim;
    KvBatch b;
    RowCut cut;
};

// The count of chunks that end at or before a token, by all threads at once.
__device__ __forceinline__ uint32_t seq_of(const KvBatch& b, uint32_t token) {
    uint32_t s = 0;
    for (uint32_t base = 0; base < b.n_seqs; base += blockDim.x) {
        const uint32_t i = base + threadIdx.x;
        const int n = __syncthreads_count(i < b.n_seqs && b.offsets[i + 1] <= (int32_t)token);
        s += n;
        if ((uint32_t)n < blockDim.x) break;
    }
    return s;
}
// Where a block's tokens lie in the cache.
struct Places {
    int64_t row[kMostTokens][2], scale[kMostTokens][2];  // of keys and values: bytes, elements
    int64_t pos[kMostTokens];
    int32_t state[kMostTokens];                          // 0: of no sequence, 1: of no page, 2: held
};
__device__ __forceinline__ void find_places(const AppendArg& a, uint32_t token0, uint32_t n, Places& p) {
    uint32_t seq = seq_of(a.b, token0);
    const uint32_t i = threadIdx.x, token = token0 + i;
    if (i >= n) return;
    while (seq < a.b.n_seqs && a.b.offsets[seq + 1] <= (int32_t)token) seq++;
    int64_t pos = 0;
    int32_t page = -1;
    if (seq < a.b.n_seqs) {
        pos = (int64_t)a.b.starts[seq] + (int64_t)token - a.b.offsets[seq];
        page = page_of(a.b, seq, pos, a.page_shift, a.n_pages);
    }
    const int64_t slot = (uint32_t)pos & ((1u << a.page_shift) - 1);
#pragma unroll
    for (int v = 0; v < 2; v++) {
        p.row[i][v] = (int64_t)max(page, 0) * a.st[v][0] + slot * a.st[v][2];
        p.scale[i][v] = (int64_t)max(page, 0) * a.sst[v][0] + slot;
    }
    p.pos[i] = pos, p.state[i] = seq >= a.b.n_seqs ? 0 : page < 0 ? 1 : 2;
}

// A token's rows are its query heads, its keys' and its values'.  A lane holds 8 values of a
// row and 8 that lie 8 times the row's lanes behind them, so that loads and stores are whole lines, and for
// heads of 64, 128 and 256 dimensions that are turned as a whole, halves apart, both of its pairs; else those
// of a turned row also load the values that they are paired with, which the row's other lanes bring
// in anyway.  A row's lanes are of one wave, whose loads of a row come before its stores, so that queries
// may be turned in place.
// Bound by memory and by how many loads are on their way: 22448 tokens with 32 query heads over 8 of 128, bfloat16
// to 4 bits, 484 MB in 120 us (4.0 TB/s; to e4m3 120, to bfloat16 121; 148 with one token's rows loaded at a
// time, 108 without turning).  Blocks of one token take 400 us: eight share look-ups, angles and the lines of scales.
// One token 4.6 us, a chain of dependent reads (chunk, table, rows).
template <typename X, typename C> __global__ void __launch_bounds__(kThreads) kv_append_kernel(AppendArg a) {
    extern __shared__ __attribute__((aligned(16))) f32x2 s_cs[];
    __shared__ Places s_p;
    const RowCut& c = a.cut;
    const uint32_t per = c.sub * c.passes, token0 = blockIdx.x / c.slabs * per, n = min(per, a.b.n_tokens - token0);
    const uint32_t pairs = a.rot.pairs, half = a.rot.half, padded = (pairs + 7) & ~7u, rot = 2 * pairs;
    find_places(a, token0, n, s_p);
    __syncthreads();
    if (pairs) {
        make_angles(s_cs, a.rot, n, [&](uint32_t t) { return a.positions ? a.positions[token0 + t] : s_p.pos[t]; }, false);
        __syncthreads();
    }
    const Mine me = my_row(c);
    const uint32_t lanes = 1u << c.shift, kind = me.row < a.q_heads ? 0 : me.row < a.q_heads + a.heads ? 1 : 2, v = kind == 2;
    const uint32_t h = me.row - (kind == 0 ? 0 : kind == 1 ? a.q_heads : a.q_heads + a.heads);
    if (!me.in || me.row >= a.q_heads + 2 * a.heads) return;  // whole rows of lanes
    const auto of = [&](const auto* x) { return kind == 0 ? x[0] : kind == 1 ? x[1] : x[2]; };
    const uint32_t d0 = me.lane * 8, dist = lanes * 8;
    const bool in0 = d0 < a.dim, in1 = d0 + dist < a.dim, paired = half == dist && rot == a.dim && kind < 2, apart = half && half % 8 == 0;
    const int64_t tok = of(a.tok) * X::bytes;
    const uint8_t* const row0 = of(a.x) + (int64_t)token0 * tok + (int64_t)h * of(a.head) * X::bytes;
    uint8_t* const q_out0 = a.q_out + ((int64_t)token0 * a.o_tok + (int64_t)h * a.o_head + d0) * X::bytes;
    const int64_t q_tok = a.o_tok * X::bytes;
    const uint32_t l0 = in0 ? d0 : 0, l1 = in1 ? d0 + dist : l0;
    uint8_t* const cache = (v ? a.cache[1] : a.cache[0]) + (int64_t)h * (v ? a.st[1][1] : a.st[0][1]) + bytes_of<C>(d0);
    const int64_t s_head = (int64_t)h * (v ? a.sst[1][1] : a.sst[0][1]);
    for (uint32_t tt = me.sub; tt < n; tt += kAhead<X> * c.sub) {
    Raw<X> raw[kAhead<X>][2];
#pragma unroll
    for (int u = 0; u < kAhead<X>; u++) {  // behind the last token it once more
        const uint8_t* const row = row0 + (int64_t)min(tt + u * c.sub, n - 1) * tok;
        raw[u][0].load(row + l0 * X::bytes), raw[u][1].load(row + l1 * X::bytes);
    }
#pragma unroll
    for (int ahead = 0; ahead < kAhead<X>; ahead++) {
        const uint32_t t = tt + ahead * c.sub;
        if (t >= n) break;
        const uint8_t* const row = row0 + (int64_t)t * tok;
        uint8_t* const q_out = q_out0 + (int64_t)t * q_tok;
        const int32_t state = s_p.state[t];
        float f[2][8];
        raw[ahead][0].get(f[0]), raw[ahead][1].get(f[1]);
#pragma unroll
        for (int k = 0; k < 8; k++) f[0][k] = in0 ? f[0][k] : 0.f, f[1][k] = in1 ? f[1][k] : 0.f;
        const f32x2* const cs = s_cs + t * padded;
        if (paired) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const f32x2 w = cs[d0 + k];
                const float x = f[0][k], y = f[1][k];
                f[0][k] = turned_first(x, y, w.x, w.y), f[1][k] = turned_second(x, y, w.x, w.y);
            }
        } else if (kind < 2 && state) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t d = d0 + u * dist;
                if (d >= rot) continue;
                if (!half) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if (d / 2 + k < pairs) {
                            const f32x2 w = cs[d / 2 + k];
                            const float x = f[u][2 * k], y = f[u][2 * k + 1];
                            f[u][2 * k] = turned_first(x, y, w.x, w.y), f[u][2 * k + 1] = turned_second(x, y, w.x, w.y);
                        }
                    }
                } else if (apart) {  // 8 values lie on one side of the pairs
                    const bool low = d < half;
                    float p[8];
                    load_vec<X, 8, false>(row + (low ? d + half : d - half) * X::bytes, p);
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const f32x2 w = cs[(low ? d : d - half) + k];
                        f[u][k] = low ? turned_first(f[u][k], p[k], w.x, w.y) : turned_second(p[k], f[u][k], w.x, w.y);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const uint32_t e = d + k;
                        if (e >= rot) continue;
                        const float p = load_one<X>(row, e < half ? e + half : e - half);
                        const f32x2 w = cs[e < half ? e : e - half];
                        f[u][k] = e < half ? turned_first(f[u][k], p, w.x, w.y) : turned_second(p, f[u][k], w.x, w.y);
                    }
                }
            }
        }
        // a query's row goes out as it is, others into the cache
        if (kind == 0) {
            if (state && in0) store_vec<X, 8>(q_out, f[0]);
            if (state && in1) store_vec<X, 8>(q_out + dist * X::bytes, f[1]);
            continue;
        }
        const bool held = state == 2;
        uint8_t* const to = cache + s_p.row[t][v];
        const int64_t s_at = s_head + s_p.scale[t][v];
        if constexpr (C::tag == CKR_F4) {
            uint8_t* const bytes = static_cast<uint8_t*>(v ? a.scales[1] : a.scales[0]) + s_at;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t d = d0 + u * dist, byte = group_byte_of(f[u]);
                if (held && (u ? in1 : in0)) {
                    *reinterpret_cast<uint32_t*>(to + u * dist / 2) = encode8(f[u], byte);
                    if (me.lane % 4 == 0) bytes[(int64_t)(d / kGroup) << a.page_shift] = (uint8_t)byte;
                }
            }
        } else {
            if constexpr (C::bytes == 1) {
                uint32_t top = 0;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int k = 0; k < 8; k++) top = max(top, abs_bits(f[u][k]));
                for (uint32_t e = 1; e < lanes; e *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, (int)e));
                const RowScale rs = row_scale<C>(top);
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int k = 0; k < 8; k++) f[u][k] = scaled(f[u][k], rs.inv);
                if (held && me.lane == 0) static_cast<float*>(v ? a.scales[1] : a.scales[0])[s_at] = rs.scale;
            }
            if (held && in0) store_vec<C, 8>(to, f[0]);
            if (held && in1) store_vec<C, 8>(to + dist * C::bytes, f[1]);
        }
    }
    }
}

// A cache of 4 bits read back: the same rows (no queries), the other way round.  Bound by memory: 124592 tokens of
// 8 heads of 128 to bfloat16, 646 MB in 130 us (5.0 TB/s; 190 with 16 values a lane and a token a thread).
template <typename X> __global__ void __launch_bounds__(kThreads) kv_read_four_kernel(AppendArg a) {
    __shared__ Places s_p;
    const RowCut& c = a.cut;
    const uint32_t per = c.sub * c.passes, token0 = blockIdx.x / c.slabs * per, n = min(per, a.b.n_tokens - token0);
    find_places(a, token0, n, s_p);
    __syncthreads();
    const Mine me = my_row(c);
    const uint32_t v = me.row >= a.heads, h = me.row - (v ? a.heads : 0), d0 = me.lane * 8, dist = 8u << c.shift;
    if (!me.in || me.row >= 2 * a.heads || d0 >= a.dim) return;
    const bool in1 = d0 + dist < a.dim;
    const int64_t tok = (v ? a.tok[2] : a.tok[1]) * X::bytes;
    uint8_t* const out0 = (v ? a.x[2] : a.x[1]) + (int64_t)token0 * tok + ((int64_t)h * (v ? a.head[2] : a.head[1]) + d0) * X::bytes;
    const uint8_t* const codes = (v ? a.cache[1] : a.cache[0]) + (int64_t)h * (v ? a.st[1][1] : a.st[0][1]) + d0 / 2;
    const uint8_t* const bytes = static_cast<const uint8_t*>(v ? a.scales[1] : a.scales[0]) + (int64_t)h * (v ? a.sst[1][1] : a.sst[0][1]) +
                                 ((int64_t)(d0 / kGroup) << a.page_shift);
    const uint32_t next = in1 ? dist / 2 : 0;
    const uint64_t next_b = in1 ? (uint64_t)(dist / kGroup) << a.page_shift : 0;
    constexpr int AHEAD = 4;
    for (uint32_t tt = me.sub; tt < n; tt += AHEAD * c.sub) {
        uint32_t x[AHEAD][2], b[AHEAD][2];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {  // behind the last token it once more
            const uint32_t t = min(tt + u * c.sub, n - 1);
            const uint8_t* at = codes + s_p.row[t][v];
            const uint8_t* bt = bytes + s_p.scale[t][v];
            x[u][0] = *reinterpret_cast<const uint32_t*>(at), x[u][1] = *reinterpret_cast<const uint32_t*>(at + next);
            b[u][0] = bt[0], b[u][1] = bt[next_b];
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const uint32_t t = tt + u * c.sub;
            if (t >= n) break;
            const bool held = s_p.state[t] == 2;
            uint8_t* const out = out0 + (int64_t)t * tok;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                if (w && !in1) break;
                const uint32_t code = held ? x[u][w] : 0, byte = held ? b[u][w] : 0;
                if constexpr (X::bytes == 2) {
                    *reinterpret_cast<u32x4*>(out + w * dist * X::bytes) = widen8<X>(code, power_of(byte));
                } else {
                    float f[8];
                    decode8(code, power_of(byte), f);
                    store_vec<X, 8>(out + w * dist * X::bytes, f);
                }
            }
        }
    }
}

template <typename X> hipError_t launch_append(const AppendArg& a, int cache_dtype, uint32_t lds, hipStream_t s) {
    const auto go = [&](auto kernel) {
        CKR_LAUNCH("kv_append", s, kernel<<<dim3((uint32_t)a.cut.blocks), a.cut.threads, lds, s>>>(a));
        return hipGetLastError();
    };
    switch (cache_dtype) {
        case CKR_F4: return go(kv_append_kernel<X, ElemF4>);
        case CKR_F8: return go(kv_append_kernel<X, ElemF8>);
        case CKR_I8: return go(kv_append_kernel<X, ElemI8>);
        case CKR_BF16: return go(kv_append_kernel<X, ElemBF16>);
        default: return go(kv_append_kernel<X, ElemF16>);
    }
}

// The cache's and the batch's part, and the cut (after the rows').
void set_cache(AppendArg& a, const ckr_kv_cache* cache, const ckr_kv_batch* batch, uint32_t passes) {
    a.cache[0] = static_cast<uint8_t*>(cache->d_k), a.cache[1] = static_cast<uint8_t*>(cache->d_v);
    a.scales[0] = cache->d_k_scale, a.scales[1] = cache->d_v_scale;
    const int ces = cache->dtype == CKR_BF16 || cache->dtype == CKR_F16 ? 2 : 1;  // of a stride's unit
    for (int i = 0; i < 3; i++) a.st[0][i] = cache->k_stride[i] * ces, a.st[1][i] = cache->v_stride[i] * ces;
    for (int i = 0; i < 2; i++) a.sst[0][i] = cache->k_scale_stride[i], a.sst[1][i] = cache->v_scale_stride[i];
    a.n_pages = cache->n_pages, a.page_shift = (uint32_t)__builtin_ctz(cache->page_size);
    a.heads = cache->n_heads, a.dim = cache->head_dim;
    a.b = {batch->d_page_table, batch->d_starts, batch->d_offsets, (int64_t)batch->table_stride, batch->table_width,
           batch->n_seqs, batch->n_tokens};
    a.cut = row_cut(batch->n_tokens, a.q_heads + 2ull * a.heads, std::max((a.dim / 8 + 1) / 2, 4u), a.rot.pairs, passes);
}

inline bool multiple(const void* p, uint64_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int check_rotary(const ckr_rotary* r, uint32_t dim, Rot& rot) {
    if (!r) return err(CKR_E_INVALID, "null rotary");
    if (r->n_pairs == 0 || r->n_pairs > dim / 2)
        return err(CKR_E_INVALID, std::to_string(r->n_pairs) + " pairs: 1 to half the head size " + std::to_string(dim));
    if (!std::isfinite(r->magnitude)) return err(CKR_E_INVALID, "the rotary's magnitude must be finite");
    if (!r->d_turns) return err(CKR_E_INVALID, "null turns pointer");
    if (!multiple(r->d_turns, 8)) return err(CKR_E_INVALID, "turns must be aligned to 8 bytes");
    rot = {r->d_turns, r->magnitude, r->n_pairs, r->interleaved ? 0 : r->n_pairs};
    return check_range(r->d_turns, (uint64_t)r->n_pairs * 8, "turns");
}

}  // namespace

// ckr_kv_read of a cache of 4 bits, whose arguments have been checked.
int kv_read_four(const ckr_kv_cache* c, const ckr_kv_batch* b, void* k, int64_t kt, int64_t kh, void* v, int64_t vt, int64_t vh,
                 int dtype, void* stream) {
    AppendArg a{};
    a.x[1] = static_cast<uint8_t*>(k), a.x[2] = static_cast<uint8_t*>(v);
    a.tok[1] = kt, a.tok[2] = vt, a.head[1] = kh, a.head[2] = vh;
    set_cache(a, c, b, 4);
    if (a.cut.blocks > kMostBlocks) return err(CKR_E_INVALID, "the batch is too large for one launch");
    const hipStream_t s = (hipStream_t)stream;
    const auto go = [&](auto kernel) { CKR_LAUNCH("kv_read", s, kernel<<<dim3((uint32_t)a.cut.blocks), a.cut.threads, 0, s>>>(a)); };
    if (dtype == CKR_F32) go(kv_read_four_kernel<ElemF32>);
    else if (dtype == CKR_BF16) go(kv_read_four_kernel<ElemBF16>);
    else go(kv_read_four_kernel<ElemF16>);
    return hip_rc(hipGetLastError(), "kv_read");
}

}  // namespace ckr

using namespace ckr;

extern "C" {

int ckr_rotary_turns(const double* h_frequencies, uint32_t n, uint64_t* h_turns) {
    if (n && (!h_frequencies || !h_turns)) return err(CKR_E_INVALID, "null frequencies or turns pointer");
    for (uint32_t i = 0; i < n; i++) {
        if (!std::isfinite(h_frequencies[i])) return err(CKR_E_INVALID, "frequency " + std::to_string(i) + " is not finite");
        // to 2^-64 of a turn, for which a quotient of 53 bits would not do
        long double t = (long double)h_frequencies[i] / 6.283185307179586476925286766559L;
        t -= std::floor(t);
        const long double hi = std::floor(t * 0x1p32L), lo = (t * 0x1p32L - hi) * 0x1p32L;
        h_turns[i] = ((uint64_t)hi << 32) + (uint64_t)std::nearbyint(lo);
    }
    return CKR_OK;
}

int ckr_rotate(const ckr_rotary* rotary, const int32_t* d_positions, const int64_t* position_stride,
               const ckr_rotary_heads* heads, uint32_t n, uint32_t batch, uint32_t tokens, uint32_t head_dim, int dtype,
               int inverse, void* stream) {
    if (dtype != CKR_F32 && dtype != CKR_BF16 && dtype != CKR_F16)
        return err(CKR_E_INVALID, "heads are of float32, bfloat16 or float16, not dtype " + std::to_string(dtype));
    if (head_dim < 2 || head_dim > 1024) return err(CKR_E_INVALID, "head size " + std::to_string(head_dim) + ": 2 to 1024");
    if (n < 1 || n > 2 || !heads || !position_stride) return err(CKR_E_INVALID, "one or two tensors of heads, and the positions' strides");
    RotateArg a{};
    int rc;
    if ((rc = check_rotary(rotary, head_dim, a.rot))) return rc;
    const uint64_t n_tokens = (uint64_t)batch * tokens;
    uint64_t rows = 0;
    for (uint32_t i = 0; i < n; i++) {
        if (heads[i].n_heads > 65535) return err(CKR_E_INVALID, "at most 65535 heads");
        rows += heads[i].n_heads;
    }
    if (n_tokens > 0x7fffffffull || n_tokens * rows > 0x7fffffffull) return err(CKR_E_INVALID, "at most 2^31 - 1 rows (tokens x heads)");
    if (n_tokens == 0 || rows == 0) return CKR_OK;
    if (!d_positions) return err(CKR_E_INVALID, "null positions pointer");
    if (!multiple(d_positions, 4)) return err(CKR_E_INVALID, "positions must be aligned to 4 bytes");
    const int es = ckr_element_size(dtype);
    const auto span = [](const int64_t* st, const uint64_t* size, int axes, uint64_t run, uint64_t& bytes) {
        unsigned __int128 last = run;
        for (int i = 0; i < axes; i++) {
            if (size[i] <= 1) continue;
            if (st[i] < 0 || st[i] > (1ll << 40)) return false;
            last += (unsigned __int128)(size[i] - 1) * (uint64_t)st[i];
        }
        bytes = (uint64_t)last;
        return last <= (1ull << 46);
    };
    const uint64_t pos_size[2] = {batch, tokens};
    uint64_t bytes = 0;
    if (!span(position_stride, pos_size, 2, 1, bytes)) return err(CKR_E_INVALID, "strides of the positions out of range");
    if ((rc = check_range(d_positions, bytes * 4, "positions"))) return rc;
    a.positions = d_positions;
    for (int i = 0; i < 2; i++) a.pos_st[i] = pos_size[i] > 1 ? position_stride[i] : 0;
    bool copy = false;
    for (uint32_t i = 0; i < n; i++) {
        const ckr_rotary_heads& x = heads[i];
        Heads& y = a.x[i];
        y.heads = x.n_heads;
        if (!x.n_heads) continue;
        const uint64_t size[3] = {batch, tokens, x.n_heads};
        for (int w = 0; w < 2; w++) {
            const void* p = w ? x.d_out : x.d_in;
            const int64_t* st = w ? x.out_stride : x.in_stride;
            const std::string what = std::string(w ? "output " : "heads ") + std::to_string(i);
            if (!p) return err(CKR_E_INVALID, "null " + what + " pointer");
            if (!multiple(p, es)) return err(CKR_E_INVALID, what + " must be aligned to the element size");
            if (!span(st, size, 3, head_dim, bytes)) return err(CKR_E_INVALID, "strides of " + what + " out of range");
            if ((rc = check_range(p, bytes * es, what.c_str()))) return rc;
            if (w) {  // rows of an output lie apart, from the nearest entries to the farthest
                struct { int64_t st; uint64_t n; } ax[3] = {{st[0], size[0]}, {st[1], size[1]}, {st[2], size[2]}};
                std::sort(ax, ax + 3, [](const auto& p, const auto& q) { return p.st < q.st; });
                uint64_t extent = head_dim;
                for (const auto& e : ax) {
                    if (e.n <= 1) continue;
                    if ((uint64_t)e.st < extent) return err(CKR_E_INVALID, "rows of " + what + " overlap");
                    extent += (e.n - 1) * (uint64_t)e.st;
                }
            }
            for (int k = 0; k < 3; k++) (w ? y.out_st : y.in_st)[k] = size[k] > 1 ? st[k] : 0;
        }
        for (int k = 0; k < 3; k++)
            if (x.d_in == x.d_out && y.in_st[k] != y.out_st[k]) return err(CKR_E_INVALID, "heads turned in place have the output's strides");
        y.in = static_cast<const uint8_t*>(x.d_in), y.out = static_cast<uint8_t*>(x.d_out);
        y.copy = x.d_in != x.d_out && 2 * a.rot.pairs < head_dim;
        copy = copy || y.copy;
    }
    if (n == 2 && a.x[0].heads && a.x[1].heads && (heads[0].d_out == heads[1].d_out || heads[0].d_out == heads[1].d_in || heads[1].d_out == heads[0].d_in))
        return err(CKR_E_INVALID, "one tensor's output is the other tensor, or its output");
    a.n_tokens = (uint32_t)n_tokens, a.tokens = tokens, a.dim = head_dim, a.inverse = inverse != 0;
    a.chunks = (a.rot.pairs + 7) / 8 + (copy ? (head_dim - 2 * a.rot.pairs + 15) / 16 : 0);
    a.cut = row_cut(n_tokens, rows, a.chunks, a.rot.pairs, 4);
    if (a.cut.blocks > kMostBlocks) return err(CKR_E_INVALID, "the heads are too many for one launch");
    const uint32_t lds = a.cut.sub * a.cut.passes * ((a.rot.pairs + 7) / 8 * 8) * 8;
    const hipStream_t s = (hipStream_t)stream;
    const auto go = [&](auto kernel) { CKR_LAUNCH("rotate", s, kernel<<<dim3((uint32_t)a.cut.blocks), a.cut.threads, lds, s>>>(a)); };
    if (dtype == CKR_F32) go(rotate_kernel<ElemF32>);
    else if (dtype == CKR_BF16) go(rotate_kernel<ElemBF16>);
    else go(rotate_kernel<ElemF16>);
    return hip_rc(hipGetLastError(), "rotate");
}

int ckr_kv_append(const ckr_kv_cache* cache, const ckr_kv_batch* batch, const ckr_rotary* rotary,
                  const int32_t* d_positions, const void* d_k, int64_t k_token_stride, int64_t k_head_stride,
                  const void* d_v, int64_t v_token_stride, int64_t v_head_stride, const void* d_q,
                  int64_t q_token_stride, int64_t q_head_stride, uint32_t n_heads, void* d_out,
                  int64_t out_token_stride, int64_t out_head_stride, int dtype, void* stream) {
    int rc;
    if ((rc = kv_check_cache(cache)) || (rc = kv_check_batch(cache, batch))) return rc;
    if (dtype != CKR_F32 && dtype != CKR_BF16 && dtype != CKR_F16)
        return err(CKR_E_INVALID, "queries, keys and values are of float32, bfloat16 or float16, not dtype " + std::to_string(dtype));
    if (n_heads > 65535) return err(CKR_E_INVALID, "at most 65535 query heads");
    if ((uint64_t)batch->n_tokens * n_heads > (1ull << 27)) return err(CKR_E_INVALID, "at most 2^27 rows (tokens x query heads)");
    AppendArg a{};
    if (rotary && (rc = check_rotary(rotary, cache->head_dim, a.rot))) return rc;
    const uint32_t T = batch->n_tokens, D = cache->head_dim;
    if (T == 0 || batch->n_seqs == 0) return CKR_OK;
    const int es = ckr_element_size(dtype);
    if ((rc = kv_check_rows(d_k, T, k_token_stride, cache->n_heads, k_head_stride, D, es, false, "keys")) ||
        (rc = kv_check_rows(d_v, T, v_token_stride, cache->n_heads, v_head_stride, D, es, false, "values")) ||
        (rc = kv_check_rows_apart(cache)))
        return rc;
    if (n_heads && ((rc = kv_check_rows(d_q, T, q_token_stride, n_heads, q_head_stride, D, es, false, "queries")) ||
                    (rc = kv_check_rows(d_out, T, out_token_stride, n_heads, out_head_stride, D, es, true, "output"))))
        return rc;
    if (n_heads && (d_out == d_k || d_out == d_v)) return err(CKR_E_INVALID, "the queries' output is the keys or the values");
    if (n_heads && d_q == d_out && ((T > 1 && q_token_stride != out_token_stride) || (n_heads > 1 && q_head_stride != out_head_stride)))
        return err(CKR_E_INVALID, "queries turned in place have the output's strides");
    if (d_positions) {
        if (!multiple(d_positions, 4)) return err(CKR_E_INVALID, "positions must be aligned to 4 bytes");
        if ((rc = check_range(d_positions, (uint64_t)T * 4, "positions"))) return rc;
    }
    a.positions = d_positions;
    a.x[0] = static_cast<uint8_t*>(const_cast<void*>(d_q)), a.x[1] = static_cast<uint8_t*>(const_cast<void*>(d_k)), a.x[2] = static_cast<uint8_t*>(const_cast<void*>(d_v));
    a.q_out = static_cast<uint8_t*>(d_out);
    a.tok[0] = q_token_stride, a.tok[1] = k_token_stride, a.tok[2] = v_token_stride;
    a.head[0] = q_head_stride, a.head[1] = k_head_stride, a.head[2] = v_head_stride;
    a.o_tok = out_token_stride, a.o_head = out_head_stride, a.q_heads = n_heads;
    set_cache(a, cache, batch, 8);
    if (a.cut.blocks > kMostBlocks) return err(CKR_E_INVALID, "the batch is too large for one launch");
    const uint32_t lds = a.cut.sub * a.cut.passes * ((a.rot.pairs + 7) / 8 * 8) * 8;
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = dtype == CKR_F32    ? launch_append<ElemF32>(a, cache->dtype, lds, s)
                         : dtype == CKR_BF16 ? launch_append<ElemBF16>(a, cache->dtype, lds, s)
                                             : launch_append<ElemF16>(a, cache->dtype, lds, s);
    return hip_rc(e, "kv_append");
}

}  // extern "C"
