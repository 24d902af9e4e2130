// C ABI of the 8-bit paged cache: argument checks.
#include "sb_cache.cuh"

using namespace sb;

namespace {

bool mat_ok(const SbMat& m) { return m.stride_t >= 0 && m.stride_h >= 0; }

int check_cache(const SbCacheParams* p) {
    if (!p) return SBATTN_ENULL;
    if (p->dtype != SBATTN_BF16 && p->dtype != SBATTN_F32 && p->dtype != SBATTN_F16) return SBATTN_EINVAL;
    if (p->kv_heads < 0 || p->head_dim <= 0 || p->pages < 1 || p->tokens < 0) return SBATTN_EINVAL;
    if (p->head_dim > kMaxHeadDim) return SBATTN_EUNSUPPORTED;
    if (p->row != cache_row(p->head_dim) || !page_size_ok(p->page_tokens)) return SBATTN_EINVAL;
    if (p->tokens > (1 << 30)) return SBATTN_EUNSUPPORTED;
    return SBATTN_OK;
}
int check_pages(const SbCacheParams* p) {
    if (!p->k_codes || !p->v_codes || !p->k_scale || !p->v_scale || !p->status) return SBATTN_ENULL;
    const int64_t page = (int64_t)p->kv_heads * p->page_tokens * p->row;
    if (p->k_stride < page || p->v_stride < page || p->k_scale_stride < p->kv_heads || p->v_scale_stride < p->kv_heads) return SBATTN_EINVAL;
    if ((((uintptr_t)p->k_codes | (uintptr_t)p->v_codes | (uintptr_t)p->k_stride | (uintptr_t)p->v_stride) & 15) != 0) return SBATTN_EALIGN;
    return SBATTN_OK;
}

}  // namespace

extern "C" size_t sbattn_blocks_params_size(void) { return sizeof(SbBlocksParams); }
extern "C" size_t sbattn_cache_params_size(void) { return sizeof(SbCacheParams); }

// A request with new tokens has one piece, two if it has two tokens or more, and page_tokens more tokens make one more.
extern "C" int64_t sbattn_cache_pieces(int64_t requests, int64_t tokens, int64_t page_tokens) {
    const int64_t m = requests < tokens ? requests : tokens, second = m < tokens - m ? m : tokens - m;
    return page_tokens < 1 || m < 1 ? 0 : m + second + (tokens > 2 * m ? (tokens - 2 * m) / page_tokens : 0);
}

extern "C" int sbattn_cache_blocks(const SbBlocksParams* p) {
    if (!p) return SBATTN_ENULL;
    if (p->requests < 0 || p->width < 0 || p->pages < 0 || p->tokens < 0 || p->n_pieces < 0 || !page_size_ok(p->page_tokens)) return SBATTN_EINVAL;
    if (p->requests > SBATTN_MAX_REQUESTS || p->tokens > (1 << 30) || (int64_t)p->width * p->page_tokens > (1 << 30)) return SBATTN_EUNSUPPORTED;
    if (p->table_stride < p->width || p->n_pieces < sbattn_cache_pieces(p->requests, p->tokens, p->page_tokens)) return SBATTN_EINVAL;
    if (!p->free_count || !p->free_count_out || !p->status) return SBATTN_ENULL;
    if (p->requests > 0 && (!p->lengths || !p->new_tokens || !p->lengths_out || !p->ends)) return SBATTN_ENULL;
    if ((p->requests > 0 && p->width > 0 && !p->tables) || (p->pages > 0 && !p->free_pages) || (p->tokens > 0 && !p->slots) || (p->n_pieces > 0 && !p->pieces))
        return SBATTN_ENULL;
    if (((uintptr_t)p->pieces & 15) != 0) return SBATTN_EALIGN;
    return launch_cache_blocks(*p, (cudaStream_t)p->stream) == 0 ? SBATTN_OK : SBATTN_ECUDA;
}

extern "C" int sbattn_cache_append(const SbCacheParams* p) {
    int rc = check_cache(p);
    if (rc != SBATTN_OK) return rc;
    if (p->n_pieces < 0) return SBATTN_EINVAL;
    if ((int64_t)p->n_pieces * p->kv_heads > 0x7fffffffll) return SBATTN_EUNSUPPORTED;
    if (p->n_pieces == 0 || p->kv_heads == 0 || p->tokens == 0) return SBATTN_OK;
    if ((rc = check_pages(p)) != SBATTN_OK) return rc;
    if (!p->k.ptr || !p->v.ptr || !p->pieces) return SBATTN_ENULL;
    if (!mat_ok(p->k) || !mat_ok(p->v)) return SBATTN_EINVAL;
    if (((uintptr_t)p->pieces & 15) != 0) return SBATTN_EALIGN;
    return launch_cache_append(*p, (cudaStream_t)p->stream) == 0 ? SBATTN_OK : SBATTN_ECUDA;
}

static int check_cached(const SbCacheParams* p) {
    const int rc = check_cache(p);
    if (rc != SBATTN_OK) return rc;
    if (p->heads < 0 || p->requests < 0 || p->width < 0) return SBATTN_EINVAL;
    if (p->kv_heads > 0 ? p->heads % p->kv_heads != 0 : p->heads != 0) return SBATTN_EINVAL;
    if (p->requests > SBATTN_MAX_REQUESTS || p->heads > 65535 || (int64_t)p->width * p->page_tokens > (1 << 30)) return SBATTN_EUNSUPPORTED;
    if (p->kv_heads > 0 && (int64_t)p->tokens * (p->heads / p->kv_heads) > (1ll << 30)) return SBATTN_EUNSUPPORTED;
    return SBATTN_OK;
}

extern "C" int sbattn_cached_workspace_bytes(const SbCacheParams* p, size_t* bytes) {
    const int rc = check_cached(p);
    if (rc != SBATTN_OK) return rc;
    if (bytes) *bytes = cached_workspace(*p);
    return SBATTN_OK;
}

extern "C" int sbattn_cached_fwd(const SbCacheParams* p) {
    int rc = check_cached(p);
    if (rc != SBATTN_OK) return rc;
    if (p->heads == 0 || p->tokens == 0) return SBATTN_OK;
    if (!p->q.ptr || !p->o.ptr || !p->rem.ptr) return SBATTN_ENULL;
    if (!mat_ok(p->q) || !mat_ok(p->o) || !mat_ok(p->v) || p->rem.stride_h < 0 || p->rem.stride_t < 0) return SBATTN_EINVAL;
    if (p->requests > 0 && (!p->lengths || (p->width > 0 && !p->tables))) return SBATTN_ENULL;
    if (p->table_stride < p->width || (!p->ends && p->tokens < p->requests)) return SBATTN_EINVAL;
    if ((rc = check_pages(p)) != SBATTN_OK) return rc;
    const size_t need = cached_workspace(*p);
    if (need > 0 && (!p->workspace || p->workspace_bytes < need || ((uintptr_t)p->workspace & 255) != 0)) return SBATTN_EWORKSPACE;
    return launch_cached_fwd(*p, (cudaStream_t)p->stream) == 0 ? SBATTN_OK : SBATTN_ECUDA;
}
