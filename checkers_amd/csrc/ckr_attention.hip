// checkers_amd/csrc/ckr_attention.hip — attention of a chunk of new tokens over
// a paged cache (ckr_kv_attention).
#include <algorithm>
#include <cmath>
#include <string>

#include "ckr_internal.h"
#include "ckr_kv.h"

namespace ckr {

int kv_check_cache(const ckr_kv_cache* c);
int kv_check_batch(const ckr_kv_cache* c, const ckr_kv_batch* b);
int kv_check_rows(const void* p, uint64_t rows, int64_t row_stride, uint64_t heads, int64_t head_stride, uint64_t dim,
                  int es, const char* what);

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
    int64_t kst[3], vst[3], skst[2], svst[2];
    uint32_t n_pages, page_shift, dim, heads, group;  // heads: query heads
    uint32_t window;
    float scale2;  // scale * log2(e): the softmax runs in powers of two
    KvBatch b;
};

// One wave per (token, query head): 64 keys at a time, a key per lane for the
// scores, four dimensions per lane for the weighted sum of the values.
template <typename X, typename C>
__global__ void __launch_bounds__(64) attend_row_kernel(AttnArg a) {
    __shared__ float q[256];
    const uint32_t token = blockIdx.x / a.heads, head = blockIdx.x % a.heads, lane = threadIdx.x;
    uint32_t seq = 0;
    for (uint32_t base = 0; base < a.b.n_seqs; base += 64) {
        const bool here = base + lane < a.b.n_seqs && a.b.offsets[base + lane + 1] <= (int32_t)token;
        const int n = __popcll(__ballot(here));
        seq += n;
        if (n < 64) break;
    }
    const int64_t kh = head / a.group;
    for (uint32_t d = lane; d < a.dim; d += 64)
        q[d] = load_one<X>(a.q + ((int64_t)token * a.q_tok + (int64_t)head * a.q_head) * 2, d) * a.scale2;
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    if (seq < a.b.n_seqs) {
        const int64_t pos = (int64_t)a.b.starts[seq] + (int64_t)token - a.b.offsets[seq];
        const int64_t first = a.window ? max((int64_t)0, pos - (int64_t)a.window + 1) : 0;
        const int64_t end = min(pos + 1, (int64_t)a.b.width << a.page_shift);
        for (int64_t base = first & ~63ll; base < end; base += 64) {
            const int64_t j = base + lane;
            const int32_t page = j >= first && j < end ? page_of(a.b, seq, j, a.page_shift, a.n_pages) : -1;
            const int64_t slot = j & ((1ll << a.page_shift) - 1);
            float s = -INFINITY, vs = 0.f;
            if (page >= 0) {
                const uint8_t* k = a.ck + ((int64_t)page * a.kst[0] + kh * a.kst[1] + slot * a.kst[2]) * C::bytes;
                float dot = 0.f;
                for (uint32_t d = 0; d < a.dim; d += 16) {
                    float x[16];
                    load_vec<C, 16>(k + d * C::bytes, x);
#pragma unroll
                    for (int i = 0; i < 16; i++) dot = __builtin_fmaf(x[i], q[d + i], dot);
                }
                if constexpr (C::bytes == 1) {
                    dot *= a.sk[(int64_t)page * a.skst[0] + kh * a.skst[1] + slot];
                    vs = a.sv[(int64_t)page * a.svst[0] + kh * a.svst[1] + slot];
                } else {
                    vs = 1.f;
                }
                s = dot;
            }
            // a NaN score must reach the result: fmax alone would pass it over
            float top = s;
            for (int d = 32; d; d /= 2) {
                const float u = __shfl_xor(top, d);
                top = u != u || top != top ? NAN : fmaxf(top, u);
            }
            if (top == -INFINITY) continue;  // no key of these 64
            const float m2 = m != m || top != top ? NAN : fmaxf(m, top);
            const float back = m == -INFINITY ? 0.f : exp2f(m - m2);
            float p = page >= 0 ? exp2f(s - m2) : 0.f, sum = p;
            for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
            l = l * back + sum;
            m = m2;
            p = page >= 0 ? p * vs : 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] *= back;
            for (int t = 0; t < 64; t++) {
                const int32_t pg = __shfl(page, t);
                const float w = __shfl(p, t);
                if (pg < 0) continue;
                const uint8_t* v = a.cv + ((int64_t)pg * a.vst[0] + kh * a.vst[1] + ((base + t) & ((1ll << a.page_shift) - 1)) * a.vst[2]) * C::bytes;
                if (4 * lane < a.dim) {
                    if constexpr (C::bytes == 1) {
                        const f32x4 x = codes4<C>(*reinterpret_cast<const uint32_t*>(v + 4 * lane));
#pragma unroll
                        for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf(w, x[i], o[i]);
                    } else {
                        const u32x2 x = *reinterpret_cast<const u32x2*>(v + 8 * lane);
                        o[0] = __builtin_fmaf(w, lo16<C>(x.x), o[0]);
                        o[1] = __builtin_fmaf(w, hi16<C>(x.x), o[1]);
                        o[2] = __builtin_fmaf(w, lo16<C>(x.y), o[2]);
                        o[3] = __builtin_fmaf(w, hi16<C>(x.y), o[3]);
                    }
                }
            }
        }
    }
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    if (4 * lane < a.dim) {
        uint8_t* out = a.out + ((int64_t)token * a.o_tok + (int64_t)head * a.o_head + 4 * lane) * 2;
        *reinterpret_cast<u32x2*>(out) = u32x2{pack16<X>(o[0] * inv, o[1] * inv), pack16<X>(o[2] * inv, o[3] * inv)};
    }
    if (a.lse && lane == 0) a.lse[(int64_t)token * a.heads + head] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename X, typename C>
hipError_t launch_attend(const AttnArg& a, hipStream_t s) {
    const uint64_t rows = (uint64_t)a.b.n_tokens * a.heads;
    CKR_LAUNCH("kv_attention", s, attend_row_kernel<X, C><<<dim3((uint32_t)rows), 64, 0, s>>>(a));
    return hipGetLastError();
}

}  // namespace
}  // namespace ckr

using namespace ckr;

extern "C" {

uint64_t ckr_kv_attention_workspace_bytes(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t n_seqs,
                                          uint32_t n_tokens, uint32_t max_chunk, uint32_t max_context) {
    return 0;
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
    if ((rc = kv_check_rows(d_q, batch->n_tokens, q_token_stride, n_heads, q_head_stride, cache->head_dim, 2, "queries")) ||
        (rc = kv_check_rows(d_out, batch->n_tokens, out_token_stride, n_heads, out_head_stride, cache->head_dim, 2, "output")))
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
    std::copy(cache->k_stride, cache->k_stride + 3, a.kst);
    std::copy(cache->v_stride, cache->v_stride + 3, a.vst);
    std::copy(cache->k_scale_stride, cache->k_scale_stride + 2, a.skst);
    std::copy(cache->v_scale_stride, cache->v_scale_stride + 2, a.svst);
    a.n_pages = cache->n_pages, a.page_shift = (uint32_t)__builtin_ctz(cache->page_size), a.dim = cache->head_dim;
    a.heads = n_heads, a.group = n_heads / cache->n_heads, a.window = window, a.scale2 = scale * kLog2e;
    a.b = {batch->d_page_table, batch->d_starts, batch->d_offsets, (int64_t)batch->table_stride, batch->table_width,
           batch->n_seqs, batch->n_tokens};
    const hipStream_t s = (hipStream_t)stream;
    hipError_t e;
    if (dtype == CKR_BF16)
        e = cache->dtype == CKR_F8   ? launch_attend<ElemBF16, ElemF8>(a, s)
            : cache->dtype == CKR_I8 ? launch_attend<ElemBF16, ElemI8>(a, s)
                                     : launch_attend<ElemBF16, ElemBF16>(a, s);
    else
        e = cache->dtype == CKR_F8   ? launch_attend<ElemF16, ElemF8>(a, s)
            : cache->dtype == CKR_I8 ? launch_attend<ElemF16, ElemI8>(a, s)
                                     : launch_attend<ElemF16, ElemF16>(a, s);
    return e == hipSuccess ? CKR_OK : err(CKR_E_HIP, std::string("HIP error in kv_attention: ") + hipGetErrorString(e));
}

}  // extern "C"
