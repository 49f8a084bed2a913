// checkers_amd/csrc/ckr_rotary.hip — rotary positions: heads turned by their tokens'
// positions (ckr_rotate, forward and backward), and a chunk's keys turned on their way
// into a paged cache (ckr_kv_append).
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

// Cosines and sines of a block's tokens in LDS, `padded` pairs a token (a multiple of 8).
constexpr uint32_t kMostTokens = 8;               // of a block
constexpr uint64_t kMostBlocks = (1u << 24) - 1;  // a grid holds fewer than 2^32 threads

// How rows are cut into blocks: `tokens` tokens a block with `slab` of their rows (one
// token where it has more rows than a block), 256 / lanes of them at a time.
struct RowCut {
    uint32_t tokens, slab, slabs;  // slabs: blocks of a token
    uint32_t shift;                // log2 of the lanes of a row
    uint32_t magic;                // ceil(2^32 / slab)
    uint64_t blocks;
};
// Blocks take one pass over their threads when there are few, up to four (a block's
// angles and, in the cache, its look-ups are then shared by more rows).
RowCut row_cut(uint64_t tokens, uint64_t rows, uint32_t lanes) {
    RowCut c{};
    while ((1u << c.shift) < lanes) c.shift++;
    const uint64_t pass = 256u >> c.shift, passes = std::clamp<uint64_t>(tokens * rows / pass / 2048, 1, 4);
    const uint64_t per = pass * passes;
    if (rows >= per) {
        c.slabs = (uint32_t)((rows + per - 1) / per);
        c.slab = (uint32_t)((rows + c.slabs - 1) / c.slabs);
        c.tokens = 1;
    } else {
        c.slabs = 1, c.slab = (uint32_t)rows;
        c.tokens = (uint32_t)std::min<uint64_t>({per / rows, kMostTokens, std::max<uint64_t>(tokens, 1)});
    }
    c.magic = c.slab == 1 ? 0xffffffffu : (uint32_t)(((1ull << 32) + c.slab - 1) / c.slab);
    c.blocks = (tokens + c.tokens - 1) / c.tokens * c.slabs;
    return c;
}
// i / slab for i < 2^16 (slab <= 2^16).
__device__ __forceinline__ uint32_t by_slab(uint32_t i, const RowCut& c) { return c.slab == 1 ? i : __umulhi(i, c.magic); }

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
    uint64_t n_tokens;  // batch x tokens
    uint32_t tokens, dim, chunks, inverse;
    RowCut cut;
};

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

template <typename E> __global__ void __launch_bounds__(256) rotate_kernel(RotateArg a) {
    extern __shared__ __attribute__((aligned(16))) f32x2 s_cs[];
    const RowCut& c = a.cut;
    const uint32_t padded = (a.rot.pairs + 7) & ~7u;
    const uint64_t token0 = (uint64_t)(blockIdx.x / c.slabs) * c.tokens;
    const uint32_t row0 = blockIdx.x % c.slabs * c.slab, n = (uint32_t)min((uint64_t)c.tokens, a.n_tokens - token0);
    for (uint32_t i = threadIdx.x; i < n * padded; i += 256) {
        const uint32_t t = i / padded, pair = i % padded;
        const uint64_t token = token0 + t, b = token / a.tokens;
        f32x2 cs = {1.f, 0.f};
        if (pair < a.rot.pairs) {
            const int64_t p = a.positions[(int64_t)b * a.pos_st[0] + (int64_t)(token - b * a.tokens) * a.pos_st[1]];
            cs = cos_sin((uint64_t)p * a.rot.turns[pair], a.rot.magnitude);
            if (a.inverse) cs.y = -cs.y;
        }
        s_cs[i] = cs;
    }
    __syncthreads();
    const uint32_t chunk = threadIdx.x & ((1u << c.shift) - 1), turned = (a.rot.pairs + 7) / 8;
    const uint32_t all = a.x[0].heads + a.x[1].heads;
    if (chunk >= a.chunks) return;
    for (uint32_t i = threadIdx.x >> c.shift; i < n * c.slab; i += 256 >> c.shift) {
        const uint32_t t = by_slab(i, c), r = row0 + (i - t * c.slab);
        if (r >= all) continue;
        const bool second = r >= a.x[0].heads;
        const Heads& x = a.x[second];
        const uint64_t token = token0 + t, b = token / a.tokens;
        const int64_t at_b = (int64_t)b, at_t = (int64_t)(token - b * a.tokens), at_h = r - (second ? a.x[0].heads : 0);
        const uint8_t* in = x.in + (at_b * x.in_st[0] + at_t * x.in_st[1] + at_h * x.in_st[2]) * E::bytes;
        uint8_t* out = x.out + (at_b * x.out_st[0] + at_t * x.out_st[1] + at_h * x.out_st[2]) * E::bytes;
        float f[16];
        if (chunk >= turned) {  // values behind the pairs
            const uint32_t d = 2 * a.rot.pairs + (chunk - turned) * 16;
            if (!x.copy) continue;
            load_some<E, 16>(in + (int64_t)d * E::bytes, a.dim - d, f);
            store_some<E, 16>(out + (int64_t)d * E::bytes, a.dim - d, f);
            continue;
        }
        const uint32_t pair = chunk * 8, left = a.rot.pairs - pair;
        float y[16];
        const f32x2* cs = s_cs + t * padded + pair;
        if (a.rot.half) {
            const int64_t d0 = (int64_t)pair * E::bytes, d1 = (int64_t)(pair + a.rot.half) * E::bytes;
            load_some<E, 8>(in + d0, left, f), load_some<E, 8>(in + d1, left, f + 8);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                y[k] = turned_first(f[k], f[8 + k], cs[k].x, cs[k].y);
                y[8 + k] = turned_second(f[k], f[8 + k], cs[k].x, cs[k].y);
            }
            store_some<E, 8>(out + d0, left, y), store_some<E, 8>(out + d1, left, y + 8);
        } else {
            load_some<E, 16>(in + (int64_t)pair * 2 * E::bytes, 2 * left, f);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                y[2 * k] = turned_first(f[2 * k], f[2 * k + 1], cs[k].x, cs[k].y);
                y[2 * k + 1] = turned_second(f[2 * k], f[2 * k + 1], cs[k].x, cs[k].y);
            }
            store_some<E, 16>(out + (int64_t)pair * 2 * E::bytes, 2 * left, y);
        }
    }
}

// ------------------------------------------------------------ append
struct AppendArg {
    Rot rot;                   // pairs 0: nothing is turned
    const int32_t* positions;  // of the angles, NULL: the cache's
    const uint8_t* in[3];      // queries, keys, values
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
    for (uint32_t base = 0; base < b.n_seqs; base += 256) {
        const uint32_t i = base + threadIdx.x;
        const int n = __syncthreads_count(i < b.n_seqs && b.offsets[i + 1] <= (int32_t)token);
        s += n;
        if (n < 256) break;
    }
    return s;
}

// A token's rows are its query heads, its keys' and its values'.  A lane holds 16 values of a
// row; those of a turned row also load the 16 that they are paired with, which the row's
// other lanes bring in anyway.
template <typename X, typename C> __global__ void __launch_bounds__(256) kv_append_kernel(AppendArg a) {
    extern __shared__ __attribute__((aligned(16))) f32x2 s_cs[];
    __shared__ int32_t s_page[kMostTokens], s_known[kMostTokens];
    __shared__ int64_t s_pos[kMostTokens];
    constexpr bool FOUR = C::tag == CKR_F4;
    const RowCut& c = a.cut;
    const uint32_t pairs = a.rot.pairs, half = a.rot.half, padded = (pairs + 7) & ~7u, rot = 2 * pairs;
    const uint32_t token0 = blockIdx.x / c.slabs * c.tokens, row0 = blockIdx.x % c.slabs * c.slab;
    const uint32_t n = min(c.tokens, a.b.n_tokens - token0);
    const uint32_t first = seq_of(a.b, token0);
    if (threadIdx.x < n) {
        const uint32_t token = token0 + threadIdx.x;
        uint32_t seq = first;
        while (seq < a.b.n_seqs && a.b.offsets[seq + 1] <= (int32_t)token) seq++;
        int64_t pos = 0;
        int32_t page = -1;
        if (seq < a.b.n_seqs) {
            pos = (int64_t)a.b.starts[seq] + (int64_t)token - a.b.offsets[seq];
            page = page_of(a.b, seq, pos, a.page_shift, a.n_pages);
        }
        s_page[threadIdx.x] = page, s_pos[threadIdx.x] = pos, s_known[threadIdx.x] = seq < a.b.n_seqs;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n * padded; i += 256) {
        const uint32_t t = i / padded, pair = i % padded;
        const int64_t p = a.positions ? a.positions[token0 + t] : s_pos[t];
        s_cs[i] = pair < pairs ? cos_sin((uint64_t)p * a.rot.turns[pair], a.rot.magnitude) : f32x2{1.f, 0.f};
    }
    __syncthreads();
    const uint32_t lanes = 1u << c.shift, lane = threadIdx.x & (lanes - 1), d = lane * 16, all = a.q_heads + 2 * a.heads;
    for (uint32_t i0 = 0; i0 < n * c.slab; i0 += 256 >> c.shift) {  // every lane, for the rows' maxima
        const uint32_t i = i0 + (threadIdx.x >> c.shift), t = by_slab(i, c), r = row0 + (i - t * c.slab);
        const bool in = i < n * c.slab && r < all && d < a.dim;
        const uint32_t kind = r < a.q_heads ? 0 : r < a.q_heads + a.heads ? 1 : 2;
        const uint32_t h = r - (kind == 0 ? 0 : kind == 1 ? a.q_heads : a.q_heads + a.heads), tt = in ? t : 0;
        const bool mine = in && s_known[tt];
        float f[16];
#pragma unroll
        for (int k = 0; k < 16; k++) f[k] = 0.f;
        if (mine) {
            const uint8_t* row = (kind == 0 ? a.in[0] : kind == 1 ? a.in[1] : a.in[2]) +
                                 ((int64_t)(token0 + t) * (kind == 0 ? a.tok[0] : kind == 1 ? a.tok[1] : a.tok[2]) +
                                  (int64_t)h * (kind == 0 ? a.head[0] : kind == 1 ? a.head[1] : a.head[2])) * X::bytes;
            load_vec<X, 16>(row + d * X::bytes, f);
            if (kind < 2 && d < rot) {
                const f32x2* cs = s_cs + t * padded;
                if (!half) {
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        if (d / 2 + k < pairs) {
                            const f32x2 w = cs[d / 2 + k];
                            const float x = f[2 * k], y = f[2 * k + 1];
                            f[2 * k] = turned_first(x, y, w.x, w.y), f[2 * k + 1] = turned_second(x, y, w.x, w.y);
                        }
                    }
                } else if (half % 8 == 0) {  // 8 values lie on one side of the pairs
#pragma unroll
                    for (int u = 0; u < 16; u += 8) {
                        const uint32_t e = d + u;
                        if (e >= rot) continue;
                        const bool low = e < half;
                        const uint32_t pair = low ? e : e - half;
                        float p[8];
                        load_vec<X, 8, false>(row + (low ? e + half : e - half) * X::bytes, p);
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const f32x2 w = cs[pair + k];
                            f[u + k] = low ? turned_first(f[u + k], p[k], w.x, w.y) : turned_second(p[k], f[u + k], w.x, w.y);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const uint32_t e = d + k;
                        if (e >= rot) continue;
                        const bool low = e < half;
                        const float p = load_one<X>(row, low ? e + half : e - half);
                        const f32x2 w = cs[low ? e : e - half];
                        f[k] = low ? turned_first(f[k], p, w.x, w.y) : turned_second(p, f[k], w.x, w.y);
                    }
                }
            }
        }
        // ---- a query's row goes out as it is, others into the cache
        const int32_t page = s_page[tt];
        const uint32_t slot = (uint32_t)s_pos[tt] & ((1u << a.page_shift) - 1), v = kind == 2;
        const bool held = mine && kind > 0 && page >= 0;
        uint8_t* to = a.cache[v] + (int64_t)page * a.st[v][0] + (int64_t)h * a.st[v][1] + (int64_t)slot * a.st[v][2] + bytes_of<C>(d);
        const int64_t s_at = (int64_t)page * a.sst[v][0] + (int64_t)h * a.sst[v][1] + slot;
        if (mine && kind == 0) store_vec<X, 16>(a.q_out + ((int64_t)(token0 + t) * a.o_tok + (int64_t)h * a.o_head + d) * X::bytes, f);
        if constexpr (FOUR) {
            const uint32_t byte = group_byte_of<16>(f);
            if (held) {
                *reinterpret_cast<u32x2*>(to) = u32x2{encode8(f, byte), encode8(f + 8, byte)};
                if (lane % 2 == 0) static_cast<uint8_t*>(a.scales[v])[s_at + ((int64_t)(d / kGroup) << a.page_shift)] = (uint8_t)byte;
            }
        } else {
            if constexpr (C::bytes == 1) {
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < 16; k++) top = max(top, abs_bits(f[k]));
                for (uint32_t e = 1; e < lanes; e *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, (int)e));
                const RowScale rs = row_scale<C>(top);
#pragma unroll
                for (int k = 0; k < 16; k++) f[k] = scaled(f[k], rs.inv);
                if (held && lane == 0) static_cast<float*>(a.scales[v])[s_at] = rs.scale;
            }
            if (held) store_vec<C, 16>(to, f);
        }
    }
}

template <typename X> hipError_t launch_append(const AppendArg& a, int cache_dtype, uint32_t lds, hipStream_t s) {
    const auto go = [&](auto kernel) {
        CKR_LAUNCH("kv_append", s, kernel<<<dim3((uint32_t)a.cut.blocks), 256, lds, s>>>(a));
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
    a.n_tokens = (uint64_t)batch * tokens;
    uint64_t rows = 0;
    for (uint32_t i = 0; i < n; i++) {
        if (heads[i].n_heads > 65535) return err(CKR_E_INVALID, "at most 65535 heads");
        rows += heads[i].n_heads;
    }
    if (a.n_tokens * rows > 0x7fffffffull) return err(CKR_E_INVALID, "at most 2^31 - 1 rows (tokens x heads)");
    if (a.n_tokens == 0 || rows == 0) return CKR_OK;
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
        y.in = static_cast<const uint8_t*>(x.d_in), y.out = static_cast<uint8_t*>(x.d_out);
        y.copy = x.d_in != x.d_out && 2 * a.rot.pairs < head_dim;
        copy = copy || y.copy;
    }
    a.tokens = tokens, a.dim = head_dim, a.inverse = inverse != 0;
    a.chunks = (a.rot.pairs + 7) / 8 + (copy ? (head_dim - 2 * a.rot.pairs + 15) / 16 : 0);
    a.cut = row_cut(a.n_tokens, rows, a.chunks);
    if (a.cut.blocks > kMostBlocks) return err(CKR_E_INVALID, "the heads are too many for one launch");
    const uint32_t lds = a.cut.tokens * ((a.rot.pairs + 7) / 8 * 8) * 8;
    const hipStream_t s = (hipStream_t)stream;
    const auto go = [&](auto kernel) { CKR_LAUNCH("rotate", s, kernel<<<dim3((uint32_t)a.cut.blocks), 256, lds, s>>>(a)); };
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
    if (n_heads && d_q == d_out && ((T > 1 && q_token_stride != out_token_stride) || (n_heads > 1 && q_head_stride != out_head_stride)))
        return err(CKR_E_INVALID, "queries turned in place have the output's strides");
    if (d_positions) {
        if (!multiple(d_positions, 4)) return err(CKR_E_INVALID, "positions must be aligned to 4 bytes");
        if ((rc = check_range(d_positions, (uint64_t)T * 4, "positions"))) return rc;
    }
    a.positions = d_positions;
    a.in[0] = static_cast<const uint8_t*>(d_q), a.in[1] = static_cast<const uint8_t*>(d_k), a.in[2] = static_cast<const uint8_t*>(d_v);
    a.q_out = static_cast<uint8_t*>(d_out);
    a.tok[0] = q_token_stride, a.tok[1] = k_token_stride, a.tok[2] = v_token_stride;
    a.head[0] = q_head_stride, a.head[1] = k_head_stride, a.head[2] = v_head_stride;
    a.o_tok = out_token_stride, a.o_head = out_head_stride;
    a.cache[0] = static_cast<uint8_t*>(cache->d_k), a.cache[1] = static_cast<uint8_t*>(cache->d_v);
    a.scales[0] = cache->d_k_scale, a.scales[1] = cache->d_v_scale;
    const int ces = cache->dtype == CKR_BF16 || cache->dtype == CKR_F16 ? 2 : 1;  // of a stride's unit
    for (int i = 0; i < 3; i++) a.st[0][i] = cache->k_stride[i] * ces, a.st[1][i] = cache->v_stride[i] * ces;
    for (int i = 0; i < 2; i++) a.sst[0][i] = cache->k_scale_stride[i], a.sst[1][i] = cache->v_scale_stride[i];
    a.n_pages = cache->n_pages, a.page_shift = (uint32_t)__builtin_ctz(cache->page_size);
    a.q_heads = n_heads, a.heads = cache->n_heads, a.dim = D;
    a.b = {batch->d_page_table, batch->d_starts, batch->d_offsets, (int64_t)batch->table_stride, batch->table_width,
           batch->n_seqs, batch->n_tokens};
    a.cut = row_cut(T, n_heads + 2ull * cache->n_heads, D / 16);
    if (a.cut.blocks > kMostBlocks) return err(CKR_E_INVALID, "the batch is too large for one launch");
    const uint32_t lds = a.cut.tokens * ((a.rot.pairs + 7) / 8 * 8) * 8;
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = dtype == CKR_F32    ? launch_append<ElemF32>(a, cache->dtype, lds, s)
                         : dtype == CKR_BF16 ? launch_append<ElemBF16>(a, cache->dtype, lds, s)
                                             : launch_append<ElemF16>(a, cache->dtype, lds, s);
    return hip_rc(e, "kv_append");
}

}  // extern "C"
