// kvattention.hip — checks, slices and workspace of the attention over a cache; the kernels are in kvattention.hpp.
#include "kvattention.hpp"

using namespace dxh;

namespace {

// Which of the two kernels; `rows` of one sequence and key head.  The 16-row kernel decodes a tile of codes for every 16 rows, the other for
// every 128, but padded to that many rows and a tile at a time behind two barriers.  16-row against 128-row kernel, bf16 unless said:
//   up to 32 rows always; up to 96 f32 rows, whose products cost more than the codes (48 rows over 3k-8k tokens, 16 x 4 heads of
//   128: 64 and 122 us; bf16, 35 rows over 4k-8k, 16 x 8 heads: 103 and 91);
//   else where the 128-row tiles leave a third of the CUs idle and there is little work, at most 64 products of a 16-row and a 64-token tile a CU: a prompt
//   of 512 tokens, 16 / 4 heads of 128, 13.6 and 23.2; a prompt of 300, f32, 2 / 1 heads of 80, 9.7 and 25.7; but four f32 prompts of
//   2000, 8 / 2 heads of 128 (128 products a CU), 132 and 114, and eight prompts of 128, 32 / 8 heads of 128 (as many 128-row tiles as
//   CUs), 31 and 14.5; eight of 313-364, 8 heads of 256, 75 and 34.
// Tiles of tokens are those that the table has room for, as the host does not see the lengths: a table much wider than its sequences
// can send a short prompt to the kernel for many rows.
bool few_rows(const KvArgs &kv, int64_t rows, int dtype) {
    if (rows <= (dtype == DXH_F32 ? 96 : 32)) return true;
    const int64_t tiles = ((int64_t)kv.pages_per_seq * kv.page_size + 63) / 64, pairs = (int64_t)kv.batch * kv.heads;
    return product(3, pairs, (rows + kTileRows - 1) / kTileRows, value_parts(kv.dim)) <= 2 * kCUs && product(pairs, (rows + 15) / 16, tiles) <= 64 * kCUs;
}

// How many slices the tokens of a sequence are cut into, counted on the longest sequence that the cache can hold; a slice has at
// least min_tiles tiles (slice_tiles), so that short sequences use fewer.
//   Few rows (16 tiles a slice): the sequences of a batch differ in length, and 8 workgroups a CU let the card fill the gaps that
//   short ones leave (64 sequences of 1k-16k tokens: 245 us at 4, 229 at 8, 230 at 16); one sequence is cut into what runs at once,
//   two workgroups a CU (131071 tokens: 64 us at 2, 76 at 4).  16 against 8 tiles a slice: one row over 777 tokens, one launch
//   instead of two, 9.7 and 12.8 us.
//   Many rows (4 tiles; 16 for heads over 128, whose partial results are twice as long: eight prompts of 313-364 tokens, 8 heads of
//   256, 43 us uncut and 65 in two slices): only where the tiles of rows alone leave CUs idle (two prompts of 1832 and 498 tokens,
//   7 / 1 heads of 64: 82 us uncut, 39 in slices).
int choose_splits(const KvArgs &kv, int q_heads, int64_t row_tiles, bool few, int min_tiles) {
    const int64_t blocks = product(kv.batch, kv.heads, row_tiles, few ? 1 : value_parts(kv.dim)), tiles = ((int64_t)kv.pages_per_seq * kv.page_size + 63) / 64;
    int64_t want;
    if (few) want = ((kv.batch > 1 ? 8 : 2) * kCUs - 1) / blocks + 1;
    else want = blocks < 2 * kCUs ? (4 * kCUs - 1) / blocks + 1 : 1;
    want = std::min<int64_t>(want, (tiles + min_tiles - 1) / min_tiles);
    const int64_t row_bytes = product(kv.rows, q_heads, (kv.dim + 2) * 4);
    want = std::min<int64_t>(want, ((int64_t)256 << 20) / std::max<int64_t>(1, row_bytes));  // partial results of at most 256 MiB
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, 128));
}
size_t part_bytes(const KvArgs &kv, int q_heads, int splits) {
    return splits > 1 ? ((size_t)splits * kv.rows * q_heads * (kv.dim + 2) * sizeof(float) + 255) / 256 * 256 : 0;
}

int plan(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, int32_t q_heads, AttArgs &a) {
    a = AttArgs{};
    const int rc = kv_check(cache, rows, dtype, a.kv);
    if (rc != DXH_OK) return rc;
    if (q_heads < 1) return DXH_ERR_ARG;
    if (q_heads % a.kv.heads) return DXH_ERR_SHAPE;
    a.q_heads = q_heads;
    a.group = q_heads / a.kv.heads;
    a.splits = 1;
    if (kv_nothing(a.kv)) return DXH_OK;
    const int64_t most = (int64_t)a.kv.max_rows * a.group;
    if (most > INT32_MAX - kTileRows) return DXH_ERR_TOO_LARGE;
    a.tile_rows = few_rows(a.kv, most, dtype) ? 16 : kTileRows;
    a.row_tiles = (int)((most + a.tile_rows - 1) / a.tile_rows);
    a.min_tiles = a.tile_rows == 16 || a.kv.dim > 128 ? 16 : 4;
    a.splits = choose_splits(a.kv, q_heads, a.row_tiles, a.tile_rows == 16, a.min_tiles);
    const int64_t blocks = product(a.kv.batch, a.kv.heads, a.row_tiles, a.tile_rows == 16 ? 1 : value_parts(a.kv.dim), a.splits), joins = a.splits > 1 ? product(a.kv.batch, a.kv.max_rows, q_heads) : 0;
    return launch_fits(blocks, kBlock) && launch_fits(joins, kBlock) ? DXH_OK : DXH_ERR_TOO_LARGE;
}

}  // namespace

extern "C" {

int dxh_kvcache_attention_workspace_bytes(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, int32_t q_heads, size_t *bytes) {
    if (!bytes) return DXH_ERR_ARG;
    AttArgs a;
    const int rc = plan(cache, rows, dtype, q_heads, a);
    if (rc == DXH_OK) *bytes = part_bytes(a.kv, q_heads, a.splits);
    return rc;
}

int dxh_kvcache_attention(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, int32_t q_heads, const dxh_heads *q, const dxh_heads *out, float *lse,
                          float scale, int causal, int64_t window, void *workspace, size_t workspace_bytes, void *stream) {
    AttArgs a;
    int rc = plan(cache, rows, dtype, q_heads, a);
    if (rc != DXH_OK) return rc;
    if ((causal != 0 && causal != 1) || window < 0 || !__builtin_isfinite(scale * kLog2e)) return DXH_ERR_ARG;
    const bool used = !kv_nothing(a.kv);
    const int es = dtype_size(dtype);
    if ((rc = kv_heads_check(q, es, used)) != DXH_OK || (rc = kv_heads_check(out, es, used)) != DXH_OK) return rc;
    if (!aligned(lse, 4)) return DXH_ERR_ALIGN;
    if (!used) return DXH_OK;
    if (q->data == out->data) return DXH_ERR_ARG;  // a row's queries are read by several workgroups
    const size_t need = part_bytes(a.kv, q_heads, a.splits);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 256))) return DXH_ERR_WORKSPACE;
    if (kv_meets(a.kv, out->data) || kv_meets(a.kv, lse) || (lse && (lse == out->data || lse == q->data))) return DXH_ERR_ARG;
    a.q = (const char *)q->data; a.q_row = q->row_stride; a.q_head = q->head_stride;
    a.out = (char *)out->data; a.o_row = out->row_stride; a.o_head = out->head_stride;
    a.lse = lse;
    a.scale = scale * kLog2e;
    a.causal = causal;
    a.window = window > INT32_MAX ? 0 : (int)window;
    // Codes of a third more than the last-level cache are not in it from step to step, and reading them past it leaves it to what comes
    // again (8 key heads of 128, 32 query heads, 1 to 32 sequences; plain against nt loads: 268 MB 49-50 and 51-54 us, 330 MB 60-66 and
    // 60-69, 400 MB 75-82 and 71-77, 537 MB 104-110 and 91-103).  Pages of 128 keep plain loads: a tile reads half of a line of
    // values, whose other half the next tile finds in the cache (268 MB 49 and 61 us, 819 MB 149 and 170).  What counts is the
    // pages that the sequences can have, not the pool they are taken from: a server's pool is past any size.  Several tiles of
    // rows read the codes more than once.
    const int64_t pages = std::min<int64_t>(a.kv.num_pages, (int64_t)a.kv.batch * a.kv.pages_per_seq);
    a.nt = a.tile_rows == 16 && a.row_tiles == 1 && a.kv.page_size == 64 && product(2 * pages, a.kv.heads, a.kv.page_size, a.kv.dim) > ((int64_t)340 << 20);
    a.part_o = (float *)workspace;
    a.part_ml = a.part_o + (size_t)a.splits * a.kv.rows * q_heads * a.kv.dim;
    hipStream_t st = as_stream(stream);
    const bool i8 = cache->code == DXH_I8;
    return dtype == DXH_F32 ? kvattention_f32(a, i8, st) : dtype == DXH_F16 ? kvattention_f16(a, i8, st) : kvattention_bf16(a, i8, st);
}

}  // extern "C"
