// checkers_amd/csrc/ckr_attention.hip — attention of a chunk of new tokens over
// a paged cache (ckr_kv_attention): how a batch is cut, the checks and the launch.
#include <cmath>
#include <string>

#include "ckr_attention.h"

namespace ckr {

int kv_check_cache(const ckr_kv_cache* c);
int kv_check_batch(const ckr_kv_cache* c, const ckr_kv_batch* b);
int kv_check_rows(const void* p, uint64_t rows, int64_t row_stride, uint64_t heads, int64_t head_stride, uint64_t dim,
                  int es, bool written, const char* what);
hipError_t attend_four(const AttnArg& a, const Cut& c, int dtype, hipStream_t s);

namespace {

int err(int code, const std::string& m) { return set_error(code, "[ckr] " + m); }

// ------------------------------------------------------------ the launch
constexpr uint64_t kSplitMin = 128;   // keys of a split at least
// Blocks of the few rows' kernel: two a CU.  (For heads of 256 its registers leave room
// for one, so there a full launch runs in two rounds.)
constexpr uint32_t kFewBlocks = 512;
// Over a cache of 4 bits three, with a tile on its way a wave (two, with two tiles: 64 sequences of 200 to 16000
// tokens 112 / 118 us, 512 of 1000 133 / 144, 40 of 50 to 3000 24 / 25; float16 queries 126 / 123); of heads of 256 two.
constexpr uint32_t kFourBlocks = 768;
// There an item (its queries, the first tiles' way, the join) costs a block as much as so many tiles, so
// that stretches with many short items are given fewer tiles (64 sequences of 200 to 16000 tokens: 126 us with
// none, 124 with 8, 112 with 16, 116 with 24; 40 of 50 to 3000: 37, 25.5, 25 and 25); in stretches from kPadFrom
// tiles on, below which a block has hardly more than one.
constexpr uint32_t kItemPad = 16, kPadFrom = 32;
uint32_t most_blocks(bool four, uint32_t dp) { return four && dp <= 128 ? kFourBlocks : kFewBlocks; }
// Its tiles of 32 keys a block at least: one a wave (one token over a thousand: 9.5 us;
// 11.0 with 8, 13.5 with 16).
constexpr uint32_t kFewTiles = 4;
// Rows of a chunk up to which it is taken, in tiles of 16 that each read the cache; us,
// few / many rows, e4m3, 8 heads of 128: 32 rows of 16 sequences over 4096 tokens 53 / 78, of one
// over 32768 42 / 79, of 64 over 1024 51 / 58; 64 rows of 64 over 1024 96 / 60, of 16
// over 4096 66 / 104.
constexpr uint32_t kFewMost = 32;
// Over 4 bits, whose tiles cost few rows half as much (e4m3's figures above; here 48 rows of 16 sequences over
// 4096 tokens 52 / 101, of one over 32768 42 / 78, of 64 over 1024 44 / 56): more rows, and more again where
// there is much to read and a tile of many rows for each sequence and head would not fill the card.  64 and 96 rows of
// 16 sequences over 4096: 60 / 98 and 65 / 101, in a window of 1024 29 / 36 and 26 / 39, of 256 24 / 21 and 16 / 25;
// of 48 over 4096 124 / 179 and 184 / 180; of one over 32768 46 / 81 and 54 / 84, over 2000 28 / 20 and 29 / 20; of 32
// over 1024 42 / 43 and 45 / 44, over 512 36 / 25 and 32 / 27; of 64 over 4096 197 / 191 and 260 / 194, in a
// window of 1024 70 / 57 and 87 / 59.
constexpr uint32_t kFourMost = 48, kFourMostLong = 96, kFourLong = 1024, kFourKeys = 1 << 17;
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
constexpr uint64_t kCounterBytes = kFourBlocks * 4;
void set_bytes(Cut& c, uint64_t rows) {
    c.part_m_bytes = (rows * 8 + 255) / 256 * 256;
    c.bytes = kCounterBytes + c.part_m_bytes + rows * c.dp * 4;
}
uint32_t few_blocks(uint64_t items, uint64_t max_context, bool four, uint32_t dp) {
    return (uint32_t)std::min<uint64_t>(items * ((max_context + 31) / 32) / kFewTiles + 1, most_blocks(four, dp));
}
// Rows of parts that a workspace holds (calls keep multiples of 32, which set_bytes rounds no further).
uint64_t rows_held(uint64_t bytes, uint32_t dp) { return bytes < kCounterBytes ? 0 : (bytes - kCounterBytes) / (8 + dp * 4); }
// workspace: its bytes; blocks and splits that it does not hold are left out, down to
// one block of few rows and no split.
Cut cut(uint32_t n_heads, uint32_t n_kv, uint32_t dim, uint32_t n_seqs, uint32_t n_tokens, uint32_t max_chunk,
        uint64_t max_context, uint64_t all_keys, uint32_t window, bool near_slots, bool four, uint64_t workspace) {
    Cut c{};
    const uint64_t group = n_heads / n_kv, rows = (uint64_t)max_chunk * group;
    c.dp = padded_dim(dim);
    uint32_t few_most = kFewMost;
    if (four) {
        const uint64_t pairs = (uint64_t)std::min(n_seqs, n_tokens) * n_kv;  // of a sequence and a head
        const uint64_t keys = window ? std::min<uint64_t>(max_context, (uint64_t)window + max_chunk) : max_context;
        few_most = keys >= kFourLong && pairs * keys >= kFourKeys && pairs < blocks_wanted(kManyRows) ? kFourMostLong : kFourMost;
    }
    const bool few = rows <= few_most && (near_slots || !four) &&
                     most_tiles(kFewRows, group, n_seqs, n_tokens) * n_kv * ((all_keys + 31) / 32 + 1 + (four ? kItemPad : 0)) < (1ull << 31);
    c.bm = few ? kFewRows : rows <= kManyMost || c.dp == 256 || !near_slots ? kManyRows : kWideRows;
    c.tiles = (uint32_t)most_tiles(c.bm, group, n_seqs, n_tokens);
    c.splits = 1;
    // the keys of a tile: a window's, and as many again as the tile has tokens
    if (window) max_context = std::min<uint64_t>(max_context, (uint64_t)window + c.bm / group + 64);
    const uint64_t items = std::max<uint64_t>((uint64_t)c.tiles * n_kv, 1);
    if (c.bm == kFewRows) {
        c.min_tiles = kFewTiles;
        c.blocks = (uint32_t)std::clamp<uint64_t>(rows_held(workspace, c.dp) / (2 * kFewRows), 1, few_blocks(items, max_context, four, c.dp));
        c.item_pad = four && items * ((max_context + 31) / 32) >= (uint64_t)c.blocks * kPadFrom ? kItemPad : 0;
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
    set_bytes(c, (uint64_t)few_blocks(items, max_context, true, c.dp) * 2 * kFewRows);
    uint64_t most = c.bytes;
    for (const uint32_t bm : {kManyRows, kWideRows}) {
        items = most_tiles(bm, group, n_seqs, n_tokens) * n_kv;
        set_bytes(c, std::min(blocks_wanted(bm), items * ((max_context + kSplitMin - 1) / kSplitMin)) * bm);
        if (max_context > kSplitMin) most = std::max(most, c.bytes);
    }
    return most;
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
    const int ces = cache->dtype == CKR_F8 || cache->dtype == CKR_I8 || cache->dtype == CKR_F4 ? 1 : 2;  // of a stride's unit
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
    const bool four = cache->dtype == CKR_F4;
    for (const int64_t* st : {a.kst, a.vst}) near_slots = near_slots && st[2] < (1ll << 26) - 16 && (cache->n_pages == 1 || st[0] < (1ll << 36));
    for (const int64_t* st : {a.skst, a.svst}) near_slots = near_slots && (!four || (a.page_shift < 29 && (cache->n_pages == 1 || st[0] < (1ll << 36))));
    const Cut c = cut(n_heads, cache->n_heads, cache->head_dim, batch->n_seqs, batch->n_tokens, batch->max_chunk,
                      std::min<uint64_t>(batch->max_context, (uint64_t)batch->table_width * cache->page_size),
                      (uint64_t)batch->table_width * cache->page_size, window, near_slots, four, workspace_bytes);
    if ((uint64_t)c.tiles * cache->n_heads * 512 > 0xffffffffull) return err(CKR_E_INVALID, "the batch is too large for one launch");
    a.tiles = c.tiles, a.splits = c.splits, a.split_len = c.split_len, a.min_tiles = c.min_tiles, a.item_pad = c.item_pad;
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
    if (four)
        e = attend_four(a, c, dtype, s);
    else if (dtype == CKR_BF16)
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
