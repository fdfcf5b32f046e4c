// pkv_paged_api.cu -- extern "C" entry points of the paged cache: argument checks, then the launches.

#include <atomic>
#include <cmath>

#include "pkv_paged.cuh"

namespace pkv {

int paged_device_error(int32_t* flag_out, int32_t clear) {
    if (cudaMemcpyFromSymbol(flag_out, g_device_error, sizeof(int32_t)) != cudaSuccess) return PKV_ERR_CUDA;
    if (clear) {
        const int32_t zero = 0;
        if (cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int32_t)) != cudaSuccess) return PKV_ERR_CUDA;
    }
    return PKV_OK;
}

}  // namespace pkv

namespace {

// Token and list indexes are 32-bit, with room above them for what the kernels' loops add before they stop.
constexpr int64_t kMaxIndex = 0x7fff0000;

bool paged_dtype(int dt) { return dt == PKV_F32 || dt == PKV_BF16 || dt == PKV_F16; }

int check_paged_codec(const pkv_codec* c, bool tables) {
    if (!c || c->dim <= 0 || c->dim % 3 != 0) return PKV_ERR_INVALID;
    if (c->dim > 192) return PKV_ERR_UNSUPPORTED;
    const int b[3] = {c->bits_z, c->bits_r, c->bits_theta};
    for (int i = 0; i < 3; ++i)
        if (b[i] < 1 || b[i] > PKV_MAX_BITS) return PKV_ERR_INVALID;
    if (b[0] + b[1] + b[2] > 12) return PKV_ERR_UNSUPPORTED;
    if (!c->R || (tables && (!c->dec_z || !c->dec_xy))) return PKV_ERR_INVALID;
    return PKV_OK;
}

int check_pages(const pkv_pages* g, int m, bool need_codes) {
    if (!g || g->batch < 0 || g->max_pages < 0 || g->num_pages < 0 || g->kv_heads < 1 || m < 1) return PKV_ERR_INVALID;
    if (m > 64) return PKV_ERR_UNSUPPORTED;                                        // head_dim <= 192
    if (g->code_bytes != 1 && g->code_bytes != 2) return PKV_ERR_INVALID;
    const int ps = g->page_size;
    if (ps < 16 || ps > 1024 || (ps & (ps - 1))) return PKV_ERR_INVALID;
    if ((int64_t)g->max_pages * ps > kMaxIndex) return PKV_ERR_UNSUPPORTED;
    if (g->token_stride < m || g->head_stride < 0 || g->page_stride < 0) return PKV_ERR_INVALID;
    if (g->batch > 0 && g->max_pages > 0 && (!g->table || g->table_stride < g->max_pages)) return PKV_ERR_INVALID;
    if (need_codes && g->num_pages > 0 && !g->k) return PKV_ERR_INVALID;
    const int64_t cb = g->code_bytes;
    if ((g->token_stride * cb | g->head_stride * cb | g->page_stride * cb) % 16) return PKV_ERR_ALIGNMENT;
    // byte strides of a page and of a page's tokens are 32-bit factors in the kernels
    if (g->page_stride * cb > 0x7fffffff || g->token_stride * cb > 0x7fffffff / 1024) return PKV_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(g->k) | reinterpret_cast<uintptr_t>(g->v)) % 16) return PKV_ERR_ALIGNMENT;
    return PKV_OK;
}

pkv::Pages device_pages(const pkv_pages* g) {
    pkv::Pages p{};
    p.k = static_cast<const uint8_t*>(g->k);
    p.v = static_cast<const uint8_t*>(g->v);
    p.page_bs = g->page_stride * g->code_bytes;
    p.head_bs = g->head_stride * g->code_bytes;
    p.tok_bs = g->token_stride * g->code_bytes;
    p.table = g->table;
    p.table_stride = g->table_stride;
    p.num_pages = g->num_pages;
    p.Hkv = g->kv_heads;
    p.B = g->batch;
    p.max_pages = g->max_pages;
    while ((1 << p.ps_log2) < g->page_size) ++p.ps_log2;
    return p;
}

int check_paged_attn(const pkv_codec* c, const pkv_paged_attn_args* a) {
    int rc = check_paged_codec(c, true);
    if (rc) return rc;
    if (!a) return PKV_ERR_INVALID;
    rc = check_pages(&a->pages, c->dim / 3, true);
    if (rc) return rc;
    const pkv_pages& g = a->pages;
    if (g.code_bytes == 1 && c->bits_z + c->bits_r + c->bits_theta > 8) return PKV_ERR_INVALID;
    if (c->flags & PKV_CODEC_FP32_ATTN) return PKV_ERR_UNSUPPORTED;                // fp16 pairs are all there is
    if (a->q_heads < 1 || a->q_heads % g.kv_heads != 0) return PKV_ERR_INVALID;
    if (a->q_heads / g.kv_heads > 16) return PKV_ERR_UNSUPPORTED;
    if (!paged_dtype(a->q_dtype) || !paged_dtype(a->out_dtype) || !std::isfinite(a->scale)) return PKV_ERR_INVALID;
    if (a->n_selected < 0 || (a->n_selected > 0 && !a->selected)) return PKV_ERR_INVALID;
    if ((int64_t)a->n_selected * g.page_size > kMaxIndex) return PKV_ERR_UNSUPPORTED;
    if ((a->weights == nullptr) != (a->weights_out == nullptr)) return PKV_ERR_INVALID;
    if (a->weights && (a->weights_slots < 0 || a->weights_row_stride < a->weights_slots)) return PKV_ERR_INVALID;
    if (g.batch == 0) return PKV_OK;
    if (!a->q || !a->out || !a->seq_lens || (g.num_pages > 0 && !g.v)) return PKV_ERR_INVALID;
    if ((int64_t)g.batch * a->q_heads > 0xffffff) return PKV_ERR_UNSUPPORTED;
    return PKV_OK;
}

// SMs of the current device, asked for once per device.
int sm_count(int* n) {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return PKV_ERR_CUDA;
    const bool kept = dev >= 0 && dev < 64;
    *n = kept ? known[dev].load(std::memory_order_relaxed) : 0;
    if (*n) return PKV_OK;
    if (cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return PKV_ERR_CUDA;
    if (kept) known[dev].store(*n, std::memory_order_relaxed);
    return PKV_OK;
}

}  // namespace

extern "C" {

size_t pkv_paged_attn_workspace_size(const pkv_codec* c, const pkv_paged_attn_args* a) {
    int sms = 0;
    if (check_paged_attn(c, a) != PKV_OK || a->pages.batch == 0 || sm_count(&sms) != PKV_OK) return 0;
    return pkv::paged_workspace(c, a, device_pages(&a->pages), sms);
}

int pkv_paged_attn(const pkv_codec* c, const pkv_paged_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_paged_attn(c, a), sms = 0;
    if (rc) return rc;
    if (a->pages.batch == 0) return PKV_OK;
    rc = sm_count(&sms);
    if (rc) return rc;
    const pkv::Pages pg = device_pages(&a->pages);
    if (!workspace || workspace_bytes < pkv::paged_workspace(c, a, pg, sms)) return PKV_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return PKV_ERR_ALIGNMENT;
    return pkv::launch_paged_attn(c, a, pg, sms, workspace, static_cast<cudaStream_t>(stream));
}

int pkv_pages_store(const pkv_pages* pages, int32_t m, void* dst, const void* codes, int32_t n, const int32_t* start,
                    const int32_t* counts, void* stream) {
    const int rc = check_pages(pages, m, false);
    if (rc) return rc;
    if (n < 0) return PKV_ERR_INVALID;
    if (n == 0 || pages->batch == 0) return PKV_OK;
    if (!dst || !codes || !start) return PKV_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(dst) % 16 || reinterpret_cast<uintptr_t>(codes) % pages->code_bytes) return PKV_ERR_ALIGNMENT;
    return pkv::launch_pages_store(device_pages(pages), static_cast<uint8_t*>(dst), static_cast<const uint8_t*>(codes),
                                   m * pages->code_bytes, pages->code_bytes, n, start, counts, static_cast<cudaStream_t>(stream));
}

int pkv_pages_summarize(const pkv_codec* c, const pkv_pages* pages, const int32_t* seq_lens, const int32_t* start,
                        const int16_t* grid_z, const int16_t* grid_xy, int8_t* summaries, void* stream) {
    int rc = check_paged_codec(c, false), sms = 0;
    if (rc) return rc;
    rc = check_pages(pages, c->dim / 3, true);
    if (rc) return rc;
    if (pages->code_bytes == 1 && c->bits_z + c->bits_r + c->bits_theta > 8) return PKV_ERR_INVALID;
    if (pages->batch == 0 || pages->max_pages == 0) return PKV_OK;
    if (!seq_lens || !grid_z || !grid_xy || !summaries) return PKV_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(summaries) | reinterpret_cast<uintptr_t>(grid_xy)) % 16) return PKV_ERR_ALIGNMENT;
    rc = sm_count(&sms);
    if (rc) return rc;
    return pkv::launch_pages_summarize(c, device_pages(pages), pages->code_bytes, seq_lens, start, grid_z, grid_xy, summaries,
                                       sms, static_cast<cudaStream_t>(stream));
}

int pkv_pages_select(const pkv_codec* c, const pkv_pages* pages, const void* q, int32_t q_dtype, int32_t q_heads,
                     int64_t q_batch_stride, int64_t q_head_stride, const int32_t* seq_lens, const int8_t* summaries,
                     int32_t top, int32_t sinks, int32_t recent, int32_t* out, void* stream) {
    int rc = check_paged_codec(c, false), sms = 0;
    if (rc) return rc;
    rc = check_pages(pages, c->dim / 3, false);
    if (rc) return rc;
    if (q_heads < 1 || q_heads % pages->kv_heads != 0 || !paged_dtype(q_dtype)) return PKV_ERR_INVALID;
    if (q_heads / pages->kv_heads > 16) return PKV_ERR_UNSUPPORTED;
    if (top < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > top) return PKV_ERR_INVALID;
    if (top > kMaxIndex || !pkv::pages_select_fits(c->dim, q_heads / pages->kv_heads, pages->max_pages)) return PKV_ERR_UNSUPPORTED;
    if (pages->batch == 0) return PKV_OK;
    if (!q || !seq_lens || !out || (pages->num_pages > 0 && !summaries)) return PKV_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(summaries) % 16) return PKV_ERR_ALIGNMENT;
    rc = sm_count(&sms);
    if (rc) return rc;
    return pkv::launch_pages_select(c, device_pages(pages), q, q_dtype, q_heads, q_batch_stride, q_head_stride, seq_lens,
                                    summaries, top, sinks, recent, out, sms, static_cast<cudaStream_t>(stream));
}

int pkv_tokens_select(const float* weights, int32_t batch, int32_t kv_heads, int32_t slots, int64_t row_stride,
                      const int32_t* seq_lens, int32_t keep, int32_t sinks, int32_t recent, int32_t* kept,
                      float* kept_weights, void* stream) {
    if (batch < 0 || kv_heads < 1 || slots < 0 || row_stride < slots) return PKV_ERR_INVALID;
    if (keep < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > keep) return PKV_ERR_INVALID;
    if (slots > kMaxIndex || keep > kMaxIndex) return PKV_ERR_UNSUPPORTED;
    if (batch == 0) return PKV_OK;
    if (!seq_lens || !kept || !kept_weights || (slots > 0 && !weights)) return PKV_ERR_INVALID;
    int sms = 0;
    const int rc = sm_count(&sms);
    if (rc) return rc;
    return pkv::launch_tokens_select(weights, batch, kv_heads, slots, row_stride, seq_lens, keep, sinks, recent, kept,
                                     kept_weights, sms, static_cast<cudaStream_t>(stream));
}

int pkv_tokens_gather(const pkv_pages* src, int32_t m, const int32_t* kept, int32_t keep, const pkv_pages* dst, void* dst_k,
                      void* dst_v, void* stream) {
    int rc = check_pages(src, m, true);
    if (rc) return rc;
    rc = check_pages(dst, m, false);
    if (rc) return rc;
    if (src->code_bytes != dst->code_bytes || src->batch != dst->batch || src->kv_heads != dst->kv_heads || keep < 0)
        return PKV_ERR_INVALID;
    if (keep > (int64_t)dst->max_pages * dst->page_size) return PKV_ERR_INVALID;
    if (src->batch == 0 || keep == 0) return PKV_OK;
    if (!kept || !dst_k || !dst_v || (src->num_pages > 0 && !src->v)) return PKV_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(dst_k) | reinterpret_cast<uintptr_t>(dst_v)) % 16) return PKV_ERR_ALIGNMENT;
    return pkv::launch_tokens_gather(device_pages(src), device_pages(dst), static_cast<uint8_t*>(dst_k),
                                     static_cast<uint8_t*>(dst_v), m * src->code_bytes, kept, keep,
                                     static_cast<cudaStream_t>(stream));
}

}  // extern "C"
