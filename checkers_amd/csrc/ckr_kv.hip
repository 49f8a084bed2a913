// checkers_amd/csrc/ckr_kv.hip — writing and reading a paged key/value cache in
// 8 or 16 bits (4 bits: ckr_rotary.hip), and the residual sum and root-mean-square norm with an output
// in 8 bits.  All three are bound by memory: one pass, rows kept in registers
// between the reduction and the store.
#include <algorithm>
#include <array>
#include <cmath>
#include <cstring>
#include <string>
#include <utility>

#include "ckr_internal.h"
#include "ckr_kv.h"

namespace ckr {

int kv_check_cache(const ckr_kv_cache* c);
int kv_check_batch(const ckr_kv_cache* c, const ckr_kv_batch* b);
int kv_check_rows(const void* p, uint64_t rows, int64_t row_stride, uint64_t heads, int64_t head_stride, uint64_t dim,
                  int es, bool written, const char* what);
int kv_read_four(const ckr_kv_cache* c, const ckr_kv_batch* b, void* k, int64_t kt, int64_t kh, void* v, int64_t vt, int64_t vh,
                 int dtype, void* stream);

namespace {

int err(int code, const std::string& m) { return set_error(code, "[ckr] " + m); }
int hip_rc(hipError_t e, const char* what) {
    return e == hipSuccess ? CKR_OK : err(CKR_E_HIP, std::string("HIP error in ") + what + ": " + hipGetErrorString(e));
}

struct Axis { int64_t stride; uint64_t entries; };
// Whether pieces of `run` elements lie apart when the axes are taken from the
// nearest entries to the farthest (of tensors whose range has been checked).
template <size_t N> bool apart(std::array<Axis, N> axes, uint64_t run) {
    for (size_t i = 1; i < N; i++)
        for (size_t j = i; j && axes[j].stride < axes[j - 1].stride; j--) std::swap(axes[j], axes[j - 1]);
    uint64_t extent = run;
    for (const Axis& x : axes) {
        if (x.entries <= 1) continue;
        if ((uint64_t)x.stride < extent) return false;
        extent += (x.entries - 1) * (uint64_t)x.stride;
    }
    return true;
}
// Entries of a row (pairs of codes for CKR_F4) and scales of a page's head that lie side by side.
uint64_t entries_of_row(const ckr_kv_cache* c) { return c->dtype == CKR_F4 ? c->head_dim / 2 : c->head_dim; }
uint64_t scales_of_head(const ckr_kv_cache* c) {
    return (uint64_t)c->page_size * (c->dtype == CKR_F4 ? c->head_dim / kGroup : 1);
}
}  // namespace
// A cache that is written: its rows, and its scales.
int kv_check_rows_apart(const ckr_kv_cache* c) {
    const uint64_t pages = c->n_pages, heads = c->n_heads, slots = c->page_size;
    for (int which = 0; which < 2; which++) {
        const int64_t* st = which ? c->v_stride : c->k_stride;
        const int64_t* ss = which ? c->v_scale_stride : c->k_scale_stride;
        if (!apart(std::array<Axis, 3>{{{st[0], pages}, {st[1], heads}, {st[2], slots}}}, entries_of_row(c)) ||
            (c->d_k_scale && !apart(std::array<Axis, 2>{{{ss[0], pages}, {ss[1], heads}}}, scales_of_head(c))))
            return err(CKR_E_INVALID, std::string("rows of the cache ") + (which ? "values" : "keys") + " overlap");
    }
    return CKR_OK;
}
namespace {

// A lane holds 16 values of a (token, head) row: a 16-byte store of codes, and
// two to four 16-byte loads.  LPR lanes (a power of two) share a row.
constexpr int kVals = 16;

struct RowsArg {
    void* k;            // the packed tensors
    void* v;
    int64_t k_tok, k_head, v_tok, v_head;
    uint8_t* ck;        // the cache
    uint8_t* cv;
    float* sk;
    float* sv;
    int64_t kst[3], vst[3], skst[2], svst[2];
    uint32_t n_pages, page_shift, heads, dim;
    KvBatch b;
};

// The sequence of the block's first token: the count of chunks that end at or
// before it, by all threads at once.
__device__ __forceinline__ uint32_t first_seq(const KvBatch& b, uint32_t token) {
    uint32_t s = 0;
    for (uint32_t base = 0; base < b.n_seqs; base += 256) {
        const uint32_t i = base + threadIdx.x;
        const int here = i < b.n_seqs && b.offsets[i + 1] <= (int32_t)token;
        const int n = __syncthreads_count(here);
        s += n;
        if (n < 256) break;
    }
    return s;
}

// One kernel for both directions: WRITE quantises packed rows (of X) into the
// cache's pages (of C), otherwise the cached rows become values of X.  Bound by
// memory, each row read and written once: bfloat16 to e4m3, 21604 tokens of 8 heads of
// 128, 134 MB written in 29.6 us with the launch (23.2 alone: 5.8 TB/s, part of it out
// of the last cache); read back, 124592 tokens in 171 us (4.5 TB/s; a copy reaches 4.7
// to 5.2).  Stores and loads that pass the caches by measured slower in both.
template <typename X, typename C, int LPR, bool WRITE>
__global__ void __launch_bounds__(256) kv_rows_kernel(RowsArg a) {
    constexpr uint32_t ROWS = 256 / LPR;
    const uint64_t row0 = (uint64_t)blockIdx.x * ROWS;
    uint32_t seq = first_seq(a.b, (uint32_t)(row0 / a.heads));
    const uint64_t row = row0 + threadIdx.x / LPR;
    const uint32_t lane = threadIdx.x % LPR;
    const uint32_t token = (uint32_t)(row / a.heads), head = (uint32_t)(row % a.heads);
    const bool mine = lane * kVals < a.dim && token < a.b.n_tokens;
    int32_t page = -1;
    int64_t pos = 0;
    if (token < a.b.n_tokens) {
        while (seq < a.b.n_seqs && a.b.offsets[seq + 1] <= (int32_t)token) seq++;
        if (seq < a.b.n_seqs) {
            pos = (int64_t)a.b.starts[seq] + (int64_t)token - a.b.offsets[seq];
            page = page_of(a.b, seq, pos, a.page_shift, a.n_pages);
        }
    }
    const uint32_t slot = (uint32_t)pos & ((1u << a.page_shift) - 1);
#pragma unroll
    for (int which = 0; which < 2; which++) {
        uint8_t* x = static_cast<uint8_t*>(which ? a.v : a.k) +
                     ((int64_t)token * (which ? a.v_tok : a.k_tok) + (int64_t)head * (which ? a.v_head : a.k_head) +
                      lane * kVals) * X::bytes;
        const int64_t* st = which ? a.vst : a.kst;
        uint8_t* c = (which ? a.cv : a.ck) +
                     ((int64_t)page * st[0] + (int64_t)head * st[1] + (int64_t)slot * st[2] + lane * kVals) * C::bytes;
        const int64_t* sst = which ? a.svst : a.skst;
        float* s = (which ? a.sv : a.sk) + ((int64_t)page * sst[0] + (int64_t)head * sst[1] + slot);
        float f[kVals];
#pragma unroll
        for (int i = 0; i < kVals; i++) f[i] = 0.f;
        if constexpr (WRITE) {
            if (mine) load_vec<X, kVals>(x, f);
            if constexpr (C::bytes == 1) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < kVals; i++) top = max(top, abs_bits(f[i]));
#pragma unroll
                for (int d = 1; d < LPR; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
                const RowScale rs = row_scale<C>(top);
#pragma unroll
                for (int i = 0; i < kVals; i++) f[i] = scaled(f[i], rs.inv);
                if (mine && page >= 0 && lane == 0) *s = rs.scale;
            }
            if (mine && page >= 0) store_vec<C, kVals>(c, f);
        } else {
            if (mine && page >= 0) {
                load_vec<C, kVals>(c, f);
                if constexpr (C::bytes == 1) {
                    const float scale = *s;
#pragma unroll
                    for (int i = 0; i < kVals; i++) f[i] *= scale;
                }
            }
            if (mine) store_vec<X, kVals>(x, f);
        }
    }
}

template <typename X, typename C, bool WRITE>
hipError_t launch_rows(const RowsArg& a, hipStream_t s) {
    const uint64_t rows = (uint64_t)a.b.n_tokens * a.heads;
    const auto go = [&](auto kernel, uint32_t lpr) {
        const uint64_t blocks = (rows + 256 / lpr - 1) / (256 / lpr);
        CKR_LAUNCH(WRITE ? "kv_write" : "kv_read", s, kernel<<<dim3((uint32_t)blocks), 256, 0, s>>>(a));
        return hipGetLastError();
    };
    if (a.dim <= 64) return go(kv_rows_kernel<X, C, 4, WRITE>, 4);
    if (a.dim <= 128) return go(kv_rows_kernel<X, C, 8, WRITE>, 8);
    return go(kv_rows_kernel<X, C, 16, WRITE>, 16);
}

template <typename X, bool WRITE>
hipError_t launch_rows_of(const RowsArg& a, int cache_dtype, hipStream_t s) {
    switch (cache_dtype) {
        case CKR_F8: return launch_rows<X, ElemF8, WRITE>(a, s);
        case CKR_I8: return launch_rows<X, ElemI8, WRITE>(a, s);
        case CKR_BF16: return launch_rows<X, ElemBF16, WRITE>(a, s);
        default: return launch_rows<X, ElemF16, WRITE>(a, s);
    }
}

template <bool WRITE>
int rows_call(const ckr_kv_cache* c, const ckr_kv_batch* b, void* k, int64_t kt, int64_t kh, void* v, int64_t vt,
              int64_t vh, int dtype, void* stream) {
    int rc;
    if ((rc = kv_check_cache(c)) || (rc = kv_check_batch(c, b))) return rc;
    if (dtype != CKR_F32 && dtype != CKR_BF16 && dtype != CKR_F16)
        return err(CKR_E_INVALID, "keys and values are of float32, bfloat16 or float16, not dtype " + std::to_string(dtype));
    if (b->n_tokens == 0 || b->n_seqs == 0) return CKR_OK;
    const int es = ckr_element_size(dtype);
    if ((rc = kv_check_rows(k, b->n_tokens, kt, c->n_heads, kh, c->head_dim, es, !WRITE, "keys")) ||
        (rc = kv_check_rows(v, b->n_tokens, vt, c->n_heads, vh, c->head_dim, es, !WRITE, "values")) ||
        (WRITE && (rc = kv_check_rows_apart(c))))
        return rc;
    if (c->dtype == CKR_F4)
        return WRITE ? ckr_kv_append(c, b, nullptr, nullptr, k, kt, kh, v, vt, vh, nullptr, 0, 0, 0, nullptr, 0, 0, dtype, stream)
                     : kv_read_four(c, b, k, kt, kh, v, vt, vh, dtype, stream);
    RowsArg a{};
    a.k = k, a.v = v, a.k_tok = kt, a.k_head = kh, a.v_tok = vt, a.v_head = vh;
    a.ck = static_cast<uint8_t*>(c->d_k), a.cv = static_cast<uint8_t*>(c->d_v), a.sk = c->d_k_scale, a.sv = c->d_v_scale;
    std::copy(c->k_stride, c->k_stride + 3, a.kst);
    std::copy(c->v_stride, c->v_stride + 3, a.vst);
    std::copy(c->k_scale_stride, c->k_scale_stride + 2, a.skst);
    std::copy(c->v_scale_stride, c->v_scale_stride + 2, a.svst);
    a.n_pages = c->n_pages, a.page_shift = (uint32_t)__builtin_ctz(c->page_size), a.heads = c->n_heads, a.dim = c->head_dim;
    a.b = {b->d_page_table, b->d_starts, b->d_offsets, (int64_t)b->table_stride, b->table_width, b->n_seqs, b->n_tokens};
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = dtype == CKR_F32    ? launch_rows_of<ElemF32, WRITE>(a, c->dtype, s)
                         : dtype == CKR_BF16 ? launch_rows_of<ElemBF16, WRITE>(a, c->dtype, s)
                                             : launch_rows_of<ElemF16, WRITE>(a, c->dtype, s);
    return hip_rc(e, WRITE ? "kv_write" : "kv_read");
}

// ---------------------------------------------------------------- the norm
struct NormArg {
    const uint8_t* x;
    const uint8_t* r;
    const uint8_t* w;
    uint8_t* out;
    float* scales;
    uint8_t* total;
    int64_t x_stride, r_stride, out_stride, total_stride;
    uint64_t row0, rows;  // of this launch
    uint32_t n, group;
    float eps;
    int w_f32;
};

// RAGGED: n is no multiple of 8, and the last piece of a row goes one element at a
// time; elsewhere vectors are loaded and stored at any address (rows of 4095 in
// bfloat16: 130 us, one element at a time 280).  A kernel without the last piece takes 91
// registers instead of 97 for rows of 8192, so five waves a SIMD instead of four: 16384
// rows in 184 us, 200 with it.
// THREADS threads a row (a block of at least 256 holds several rows of fewer).
// Thread t of a row holds the 8 values from 8 (t + v THREADS) on, for v < VPT, so a
// row is read once and stays in registers through both reductions (the sum of
// squares, then the largest magnitude).  Bound by memory: rows of 8192 in float16,
// 16384 of them with residual, total and codes by 128, 943 MB in 175 to 185 us from card
// to card (5.2 TB/s, what a copy reaches); 2048 rows of 4096 in 12.3 us; one row 3.5 us, of which the kernel
// can save nothing (a load, two reductions, a store).
template <typename E, typename O, int THREADS, int VPT, bool RAGGED>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) add_rms_norm_kernel(NormArg a) {
    constexpr uint32_t ROWS = THREADS < 256 ? 256 / THREADS : 1;
    static_assert(THREADS <= 64 || THREADS >= 256, "a row of several waves has its block to itself");
    const uint32_t tid = threadIdx.x % THREADS;
    uint64_t row = (uint64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
    if (row >= a.rows) return;
    row += a.row0;
    const uint8_t* x = a.x + (int64_t)row * a.x_stride * E::bytes;
    const uint8_t* r = a.r ? a.r + (int64_t)row * a.r_stride * E::bytes : nullptr;
    uint8_t* total = a.total ? a.total + (int64_t)row * a.total_stride * E::bytes : nullptr;
    uint8_t* out = a.out + (int64_t)row * a.out_stride * O::bytes;
    constexpr int WAVES = THREADS < 64 ? 1 : THREADS / 64;
    __shared__ float s_sum[WAVES];
    __shared__ uint32_t s_top[WAVES];
    float h[VPT][8];
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const uint32_t col = (v * THREADS + tid) * 8;
        const uint32_t left = a.n - min(col, a.n);
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[v][i] = q[i] = 0.f;
        if (left >= 8) {
            load_vec<E, 8, false>(x + (int64_t)col * E::bytes, h[v]);
            if (r) load_vec<E, 8, false>(r + (int64_t)col * E::bytes, q);
        } else if constexpr (RAGGED) {
#pragma unroll
            for (int i = 0; i < 7; i++)
                if ((uint32_t)i < left) {
                    h[v][i] = load_one<E>(x, col + i);
                    if (r) q[i] = load_one<E>(r, col + i);
                }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            h[v][i] += q[i];
            sum = __builtin_fmaf(h[v][i], h[v][i], sum);
        }
    }
#pragma unroll
    for (int d = std::min(THREADS, 64) / 2; d; d /= 2) sum += __shfl_xor(sum, d);
    if constexpr (WAVES > 1) {
        if (threadIdx.x % 64 == 0) s_sum[threadIdx.x / 64] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) sum += s_sum[w];
    }
    const float rms = 1.f / sqrtf(sum / (float)a.n + a.eps);
    uint32_t top = 0;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const uint32_t col = (v * THREADS + tid) * 8;
        const uint32_t left = a.n - min(col, a.n);
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = 0.f;
        if (left >= 8) {
            if (total) store_vec<E, 8, false>(total + (int64_t)col * E::bytes, h[v]);
            if (a.w_f32) load_vec<ElemF32, 8, false>(a.w + (int64_t)col * 4, w);
            else load_vec<E, 8, false>(a.w + (int64_t)col * E::bytes, w);
        } else if constexpr (RAGGED) {
#pragma unroll
            for (int i = 0; i < 7; i++)
                if ((uint32_t)i < left) {
                    if (total) store_one<E>(total, col + i, h[v][i]);
                    w[i] = a.w_f32 ? load_one<ElemF32>(a.w, col + i) : load_one<E>(a.w, col + i);
                }
        }
        uint32_t part = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            h[v][i] = col + i < a.n ? h[v][i] * rms * w[i] : 0.f;
            if constexpr (O::bytes == 1) part = max(part, abs_bits(h[v][i]));
        }
        if constexpr (O::bytes == 1) {
            if (a.group) {  // group / 8 adjacent lanes hold a group
                for (uint32_t d = 1; d < a.group / 8; d *= 2) part = max(part, (uint32_t)__shfl_xor((int)part, (int)d));
                const RowScale rs = row_scale<O>(part);
#pragma unroll
                for (int i = 0; i < 8; i++) h[v][i] = scaled(h[v][i], rs.inv);
                if (col < a.n && col % a.group == 0) a.scales[row * (a.n / a.group) + col / a.group] = rs.scale;
            } else {
                top = max(top, part);
            }
        }
    }
    if constexpr (O::bytes == 1) {
        if (!a.group) {
#pragma unroll
            for (int d = std::min(THREADS, 64) / 2; d; d /= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
            if constexpr (WAVES > 1) {
                if (threadIdx.x % 64 == 0) s_top[threadIdx.x / 64] = top;
                __syncthreads();
                top = 0;
#pragma unroll
                for (int w = 0; w < WAVES; w++) top = max(top, s_top[w]);
            }
            const RowScale rs = row_scale<O>(top);
#pragma unroll
            for (int v = 0; v < VPT; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) h[v][i] = scaled(h[v][i], rs.inv);
            if (tid == 0) a.scales[row] = rs.scale;
        }
    }
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const uint32_t col = (v * THREADS + tid) * 8;
        const uint32_t left = a.n - min(col, a.n);
        if (left >= 8) {
            store_vec<O, 8, false>(out + (int64_t)col * O::bytes, h[v]);
        } else if constexpr (RAGGED) {
#pragma unroll
            for (int i = 0; i < 7; i++)
                if ((uint32_t)i < left) store_one<O>(out, col + i, h[v][i]);
        }
    }
}

template <typename E, typename O, bool RAGGED>
hipError_t launch_norm(const NormArg& a, uint64_t rows, hipStream_t s) {
    const auto go = [&](auto kernel, uint32_t threads) {
        constexpr uint64_t kMost = 1u << 21;  // blocks of a launch: a grid holds fewer than 2^32 threads
        const uint64_t per = threads < 256 ? 256 / threads : 1;
        for (uint64_t r0 = 0; r0 < rows; r0 += kMost * per) {
            NormArg b = a;
            b.row0 = r0, b.rows = std::min(rows - r0, kMost * per);
            CKR_LAUNCH("add_rms_norm", s, kernel<<<dim3((uint32_t)((b.rows + per - 1) / per)), std::max(threads, 256u), 0, s>>>(b));
        }
        return hipGetLastError();
    };
    // The fewest threads whose registers hold a row in at most four loads of a tensor:
    // one wave has no barrier, and blocks of four rows keep more loads on their way.
    // bfloat16 with residual to e4m3, 469 MB in all, us here / otherwise: 256 values 95 /
    // 154 (a wave a row), 425 (256 threads); 1024: 87 / 140 (256 threads); 2048: 93, and 12 /
    // 13.5 with 59 MB (256 threads); 4096: 84 / 90 (512 threads); 8192: 92 / 99 (1024
    // threads); 16384: 88 / 121 (256 threads, eight loads).  Above 32768 the 64 values of a
    // thread do not fit the 128 registers that 1024 threads leave it: 22 to 50 spill, in the
    // ragged kernel 88 to 151 (16-bit rows; 65536: 138 us).
    if (a.n <= 128) return go(add_rms_norm_kernel<E, O, 16, 1, RAGGED>, 16);
    if (a.n <= 256) return go(add_rms_norm_kernel<E, O, 32, 1, RAGGED>, 32);
    if (a.n <= 512) return go(add_rms_norm_kernel<E, O, 64, 1, RAGGED>, 64);
    if (a.n <= 1024) return go(add_rms_norm_kernel<E, O, 64, 2, RAGGED>, 64);
    if (a.n <= 2048) return go(add_rms_norm_kernel<E, O, 64, 4, RAGGED>, 64);
    if (a.n <= 4096) return go(add_rms_norm_kernel<E, O, 256, 2, RAGGED>, 256);
    if (a.n <= 8192) return go(add_rms_norm_kernel<E, O, 256, 4, RAGGED>, 256);
    if (a.n <= 16384) return go(add_rms_norm_kernel<E, O, 1024, 2, RAGGED>, 1024);
    if (a.n <= 32768) return go(add_rms_norm_kernel<E, O, 1024, 4, RAGGED>, 1024);
    return go(add_rms_norm_kernel<E, O, 1024, 8, RAGGED>, 1024);
}

template <typename E, typename O>
hipError_t launch_norm_any(const NormArg& a, uint64_t rows, hipStream_t s) {
    return a.n % 8 ? launch_norm<E, O, true>(a, rows, s) : launch_norm<E, O, false>(a, rows, s);
}
template <typename E>
hipError_t launch_norm_of(const NormArg& a, int out_dtype, uint64_t rows, hipStream_t s) {
    if (out_dtype == CKR_F8) return launch_norm_any<E, ElemF8>(a, rows, s);
    if (out_dtype == CKR_I8) return launch_norm_any<E, ElemI8>(a, rows, s);
    return launch_norm_any<E, E>(a, rows, s);
}

inline bool multiple(const void* p, uint64_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

// ---------------------------------------------------------------- argument checks
// (An axis of one entry may have any stride: it is never taken.)
int kv_check_rows(const void* p, uint64_t rows, int64_t row_stride, uint64_t heads, int64_t head_stride, uint64_t dim,
                  int es, bool written, const char* what) {
    if (!p) return err(CKR_E_INVALID, std::string("null ") + what + " pointer");
    if (rows == 1) row_stride = 0;
    if (heads == 1) head_stride = 0;
    if (row_stride < 0 || head_stride < 0) return err(CKR_E_INVALID, std::string("negative stride of the ") + what);
    if (!multiple(p, 16) || (row_stride * es) % 16 || (head_stride * es) % 16)
        return err(CKR_E_INVALID, std::string("rows of the ") + what + " must start on 16-byte boundaries");
    const unsigned __int128 last = (unsigned __int128)(rows - 1) * (uint64_t)row_stride +
                                   (unsigned __int128)(heads - 1) * (uint64_t)head_stride + dim;
    if (last > (1ull << 46)) return err(CKR_E_INVALID, std::string("strides of the ") + what + " are out of range");
    if (written && !apart(std::array<Axis, 2>{{{row_stride, rows}, {head_stride, heads}}}, dim))
        return err(CKR_E_INVALID, std::string("rows of the ") + what + " overlap");
    return check_range(p, (uint64_t)last * es, what);
}

int kv_check_cache(const ckr_kv_cache* c) {
    if (!c) return err(CKR_E_INVALID, "null cache");
    const bool four = c->dtype == CKR_F4, coded = four || c->dtype == CKR_F8 || c->dtype == CKR_I8;
    if (!coded && c->dtype != CKR_BF16 && c->dtype != CKR_F16)
        return err(CKR_E_INVALID, "a cache holds 4- or 8-bit floats, int8, bfloat16 or float16, not dtype " + std::to_string(c->dtype));
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1)))
        return err(CKR_E_INVALID, "page size " + std::to_string(c->page_size) + ": a power of two from 16 on");
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
        return err(CKR_E_INVALID, "head size " + std::to_string(c->head_dim) + ": a multiple of 16 up to 256");
    if (four && c->head_dim % kGroup)
        return err(CKR_E_INVALID, "head size " + std::to_string(c->head_dim) + ": a multiple of 32 in 4 bits");
    if (c->n_heads == 0 || c->n_heads > 65535) return err(CKR_E_INVALID, "a cache has 1 to 65535 heads");
    if (c->n_pages == 0 || c->n_pages > 0x7fffffffu) return err(CKR_E_INVALID, "a cache has 1 to 2^31 - 1 pages");
    const int es = coded ? 1 : 2;
    for (int which = 0; which < 2; which++) {
        const void* p = which ? c->d_v : c->d_k;
        const int64_t* st = which ? c->v_stride : c->k_stride;
        const char* what = which ? "cache values" : "cache keys";
        if (!p) return err(CKR_E_INVALID, std::string("null ") + what + " pointer");
        unsigned __int128 last = entries_of_row(c);
        const uint64_t shape[3] = {c->n_pages, c->n_heads, c->page_size};
        for (int i = 0; i < 3; i++) {
            if (shape[i] == 1) continue;
            if (st[i] < 0 || (st[i] * es) % 16)
                return err(CKR_E_INVALID, std::string("strides of the ") + what + " must be multiples of 16 bytes, not negative");
            last += (unsigned __int128)(shape[i] - 1) * (uint64_t)st[i];
        }
        if (!multiple(p, 16)) return err(CKR_E_INVALID, std::string(what) + " must start on a 16-byte boundary");
        if (last > (1ull << 46)) return err(CKR_E_INVALID, std::string("strides of the ") + what + " are out of range");
        int rc = check_range(p, (uint64_t)last * es, what);
        if (rc) return rc;
        if (!coded) continue;
        const void* s = which ? c->d_v_scale : c->d_k_scale;
        const int64_t* given = which ? c->v_scale_stride : c->k_scale_stride;
        const int64_t ss[2] = {c->n_pages == 1 ? 0 : given[0], c->n_heads == 1 ? 0 : given[1]};
        const char* swhat = which ? "value scales" : "key scales";
        if (!s) return err(CKR_E_INVALID, std::string("null ") + swhat + " pointer (" + (four ? "a 4" : "an 8") + "-bit cache has scales)");
        const int64_t unit = four ? 16 : 4;  // scales in 16 bytes
        if (!multiple(s, 16) || ss[0] < 0 || ss[1] < 0 || ss[0] % unit || ss[1] % unit)
            return err(CKR_E_INVALID, std::string(swhat) + " must start on 16-byte boundaries for every page and head");
        const unsigned __int128 slast = (unsigned __int128)(c->n_pages - 1) * (uint64_t)ss[0] +
                                        (unsigned __int128)(c->n_heads - 1) * (uint64_t)ss[1] + scales_of_head(c);
        if (slast > (1ull << 46)) return err(CKR_E_INVALID, std::string("strides of the ") + swhat + " are out of range");
        if ((rc = check_range(s, (uint64_t)slast * (four ? 1 : 4), swhat))) return rc;
    }
    return CKR_OK;
}

int kv_check_batch(const ckr_kv_cache* c, const ckr_kv_batch* b) {
    if (!b) return err(CKR_E_INVALID, "null batch");
    if (b->n_tokens > 0x7fffffffu || b->n_seqs > 0x7fffffffu || b->table_width > 0x7fffffffu)
        return err(CKR_E_INVALID, "a batch has at most 2^31 - 1 tokens, sequences and pages of a sequence");
    if ((uint64_t)b->n_tokens * c->n_heads > (1ull << 27)) return err(CKR_E_INVALID, "a batch has at most 2^27 rows (tokens x heads)");
    if (b->n_tokens == 0 || b->n_seqs == 0) {
        if (b->n_tokens) return err(CKR_E_INVALID, "a batch of no sequences has no tokens");
        return CKR_OK;
    }
    if (!b->d_page_table || !b->d_starts || !b->d_offsets) return err(CKR_E_INVALID, "null page table, starts or offsets pointer");
    if (!multiple(b->d_page_table, 4) || !multiple(b->d_starts, 4) || !multiple(b->d_offsets, 4))
        return err(CKR_E_INVALID, "page table, starts and offsets must be aligned to 4 bytes");
    // the table is only read, so its rows may overlap
    if (b->table_width == 0 || b->table_stride > (1ull << 40))
        return err(CKR_E_INVALID, "the page table's rows must hold table_width entries, their stride at most 2^40");
    int rc;
    const unsigned __int128 entries = (unsigned __int128)(b->n_seqs - 1) * b->table_stride + b->table_width;
    if (entries > (1ull << 46)) return err(CKR_E_INVALID, "the page table is out of range");
    if ((rc = check_range(b->d_page_table, (uint64_t)entries * 4, "page table")) ||
        (rc = check_range(b->d_starts, (uint64_t)b->n_seqs * 4, "starts")) ||
        (rc = check_range(b->d_offsets, ((uint64_t)b->n_seqs + 1) * 4, "offsets")))
        return rc;
    return CKR_OK;
}

}  // namespace ckr

using namespace ckr;

extern "C" {

int ckr_kv_write(const ckr_kv_cache* cache, const ckr_kv_batch* batch, const void* d_k, int64_t k_token_stride,
                 int64_t k_head_stride, const void* d_v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                 void* stream) {
    return rows_call<true>(cache, batch, const_cast<void*>(d_k), k_token_stride, k_head_stride, const_cast<void*>(d_v),
                           v_token_stride, v_head_stride, dtype, stream);
}

int ckr_kv_read(const ckr_kv_cache* cache, const ckr_kv_batch* batch, void* d_k, int64_t k_token_stride,
                int64_t k_head_stride, void* d_v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                void* stream) {
    return rows_call<false>(cache, batch, d_k, k_token_stride, k_head_stride, d_v, v_token_stride, v_head_stride, dtype,
                            stream);
}

int ckr_add_rms_norm(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride,
                     const void* d_weight, int w_dtype, uint64_t rows, uint32_t n, int dtype, float eps, int out_dtype,
                     uint32_t group, void* d_out, int64_t out_stride, float* d_scales, void* d_total,
                     int64_t total_stride, void* stream) {
    if (dtype != CKR_F32 && dtype != CKR_BF16 && dtype != CKR_F16)
        return err(CKR_E_INVALID, "rows are of float32, bfloat16 or float16, not dtype " + std::to_string(dtype));
    if (w_dtype != dtype && w_dtype != CKR_F32) return err(CKR_E_INVALID, "the weight is of the rows' type or float32");
    const bool coded = out_dtype == CKR_F8 || out_dtype == CKR_I8;
    if (!coded && out_dtype != dtype) return err(CKR_E_INVALID, "the output is of the rows' type, 8-bit floats or int8");
    if (n == 0 || n > 65536) return err(CKR_E_INVALID, "row length " + std::to_string(n) + ": 1 to 65536");
    if (!(eps >= 0.f) || std::isinf(eps)) return err(CKR_E_INVALID, "eps must be finite and not negative");
    if (group && (!coded || (group != 32 && group != 64 && group != 128 && group != 256) || n % group))
        return err(CKR_E_INVALID, "group " + std::to_string(group) + ": 32, 64, 128 or 256 dividing the row length, for 8-bit outputs");
    if (rows > 0x7fffffffull) return err(CKR_E_INVALID, "at most 2^31 - 1 rows");
    if (rows == 0) return CKR_OK;
    const int es = ckr_element_size(dtype), os = coded ? 1 : es;
    if (!d_x || !d_weight || !d_out || (coded && !d_scales)) return err(CKR_E_INVALID, "null rows, weight, output or scales pointer");
    const struct { const void* p; int64_t stride; int es; const char* what; } t[4] = {
        {d_x, x_stride, es, "rows"}, {d_residual, residual_stride, es, "residual"}, {d_total, total_stride, es, "total"},
        {d_out, out_stride, os, "output"}};
    int rc;
    for (const auto& q : t) {
        if (!q.p) continue;
        if (rows > 1 && (q.stride < 0 || q.stride > (1ll << 40))) return err(CKR_E_INVALID, std::string("stride of the ") + q.what + " out of range");
        if (!multiple(q.p, q.es)) return err(CKR_E_INVALID, std::string(q.what) + " must be aligned to the element size");
        if ((rc = check_range(q.p, ((rows - 1) * (uint64_t)q.stride + n) * q.es, q.what))) return rc;
    }
    if (!multiple(d_weight, ckr_element_size(w_dtype)) || !multiple(d_scales, 4))
        return err(CKR_E_INVALID, "weight and scales must be aligned to their element size");
    if ((rc = check_range(d_weight, (uint64_t)n * ckr_element_size(w_dtype), "weight")) ||
        (coded && (rc = check_range(d_scales, rows * (group ? n / group : 1) * 4, "scales"))))
        return rc;
    if ((out_stride < (int64_t)n && rows > 1) || (d_total && total_stride < (int64_t)n && rows > 1))
        return err(CKR_E_INVALID, "rows of an output overlap");
    NormArg a{};
    a.x = static_cast<const uint8_t*>(d_x), a.r = static_cast<const uint8_t*>(d_residual);
    a.w = static_cast<const uint8_t*>(d_weight), a.out = static_cast<uint8_t*>(d_out), a.scales = d_scales;
    a.total = static_cast<uint8_t*>(d_total);
    a.x_stride = x_stride, a.r_stride = residual_stride, a.out_stride = out_stride, a.total_stride = total_stride;
    a.n = n, a.group = group, a.eps = eps, a.w_f32 = w_dtype == CKR_F32;
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = dtype == CKR_F32    ? launch_norm_of<ElemF32>(a, out_dtype, rows, s)
                         : dtype == CKR_BF16 ? launch_norm_of<ElemBF16>(a, out_dtype, rows, s)
                                             : launch_norm_of<ElemF16>(a, out_dtype, rows, s);
    return hip_rc(e, "add_rms_norm");
}

}  // extern "C"
