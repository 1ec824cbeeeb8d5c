// C-ABI of the ragged attention: checks, then the kernel for the call's rows per kv head.
#include "attn_ragged.cuh"

using namespace b2;

namespace {
// Whether the longest sequence's rows per kv head go to the 16-row kernel. It reads the keys again for every 16 rows, but
// starts sooner and wastes less on few rows. Measured in us, 16-row kernel / 256-row kernel:
//   dim 128, 24 x 8000 keys: 16 rows 102 / 114, 20 rows 150 / 115;  4 x 16000 keys: 16 rows 51 / 57, 20 rows 83 / 57
//   dim 64,  32 x 2000 keys: 16 rows 27 / 47, 32 rows 39 / 47, 36 rows 56 / 48
// One kernel takes the whole batch, so sequences of unlike lengths lose on either side (dim 128):
//   64 sequences of two tokens over 4000 keys, a row each 166 / 246, four rows each 170 / 247
//   one of 1000 tokens over 4000 keys beside 99 single tokens over 3000, a row each: 231 / 330; over 61 000 keys: 1851 / 555
//   one of 500 tokens over 2500 keys beside 200 single tokens over 2000, four rows each: 303 / 440
bool few_rows(int heads, int kv_heads, int dim, int max_q) {
    return (int64_t)max_q * (heads / kv_heads) <= (dim == 64 ? 32 : 16);
}
}  // namespace

// The larger of the two kernels' needs, whatever max_q is: the call cannot tell how large its buffer is, and one that was
// sized for single tokens may be handed to a chunk.
extern "C" int64_t b2_attn_ragged_workspace_bytes(int heads, int kv_heads, int dim, int max_q) {
    (void)max_q;
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || (dim != 64 && dim != 128)) return 0;
    const int64_t rows = rows_workspace(dim), tiles = tiles_workspace(dim);
    return rows > tiles ? rows : tiles;
}

extern "C" int b2_attn_ragged(const b2_attn_ragged_args* p, void* stream) {
    if (!p) return fail(B2_ERR_INVALID, "attn_ragged: null arguments");
    if (p->batch < 0 || p->tokens < 0 || p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads || p->window < 0 ||
        p->key_rows < 0 || p->max_pages < 0 || p->num_pages < 0 || p->table_ld < 0)
        return fail(B2_ERR_INVALID, "attn_ragged: bad shape batch=%d tokens=%d heads=%d kv_heads=%d window=%d", p->batch,
                    p->tokens, p->heads, p->kv_heads, p->window);
    if (p->dim != 64 && p->dim != 128) return fail(B2_ERR_UNSUPPORTED, "attn_ragged: head dim %d (64 or 128)", p->dim);
    if (p->dtype != B2_F16 && p->dtype != B2_BF16)
        return fail(B2_ERR_UNSUPPORTED, "attn_ragged: dtype code %d (fp16 or bf16)", p->dtype);
    // Both are multiplied by log2(e), and scores by scale / softcap.
    if (!(p->scale > 0.f) || p->scale > 2e38f || !(p->softcap >= 0.f) || p->softcap > 2e38f ||
        (p->softcap > 0.f && p->scale / p->softcap > 2e38f))
        return fail(B2_ERR_INVALID, "attn_ragged: scale must be positive, softcap not negative, scale, softcap and scale / softcap "
                                    "at most 2e38");
    if ((int64_t)p->tokens * p->heads > (1 << 30))
        return fail(B2_ERR_UNSUPPORTED, "attn_ragged: %d tokens of %d heads in one call", p->tokens, p->heads);
    if (p->batch == 0 || p->tokens == 0) return B2_OK;
    if (!p->q || !p->out || !p->k || !p->v || !p->cu_q || !p->lengths || !p->workspace)
        return fail(B2_ERR_INVALID, "attn_ragged: null pointer");
    if (p->table && p->page_size <= 0) return fail(B2_ERR_INVALID, "attn_ragged: page size %d", p->page_size);
    if (!aligned16(p->q) || !aligned16(p->out) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->workspace) ||
        (p->sqt | p->sqh | p->sot | p->soh | p->s_page | p->s_row | p->s_head) % 8)
        return fail(B2_ERR_UNSUPPORTED, "attn_ragged: q, k, v and out must be 16-byte aligned with 16-byte strides");
    RaggedArgs a{};
    a.q = p->q;
    a.sqt = p->sqt;
    a.sqh = p->sqh;
    a.out = p->out;
    a.sot = p->sot;
    a.soh = p->soh;
    a.lse = p->lse;
    a.k = p->k;
    a.v = p->v;
    a.s_page = p->s_page;
    a.s_row = p->s_row;
    a.s_head = p->s_head;
    a.table = p->table;
    a.table_ld = p->table_ld;
    a.max_pages = p->max_pages;
    a.num_pages = p->num_pages;
    a.page_size = p->page_size;
    a.cu_q = p->cu_q;
    a.lengths = p->lengths;
    a.prefix = p->prefix;
    a.slopes = p->slopes;
    a.batch = p->batch;
    a.tokens = p->tokens;
    a.key_rows = p->key_rows;
    a.heads = p->heads;
    a.kv_heads = p->kv_heads;
    a.group = p->heads / p->kv_heads;
    a.causal = p->causal != 0;
    a.window = p->window >= (1 << 30) ? 0 : p->window;  // no position reaches that far
    a.by_group.set(a.group);
    if (a.table) a.by_page.set(a.page_size);
    a.scale = p->scale;
    a.softcap = p->softcap;
    a.cap_y = p->softcap > 0.f ? p->scale / p->softcap : 0.f;
    auto kernel = few_rows(p->heads, p->kv_heads, p->dim, p->max_q) ? attn_rows : attn_tiles;
    return kernel(a, p->dim, p->dtype == B2_BF16, p->workspace, (cudaStream_t)stream);
}
