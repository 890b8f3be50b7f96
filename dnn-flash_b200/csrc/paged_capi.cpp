// paged_capi.cpp -- argument checks and launch requests of the paged-cache entry points
// (include/odf_paged_sm100.h).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "paged_internal.h"

namespace {

using odf::set_error;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int current_device_ready(int** status, int* sm_count = nullptr) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return set_error(ODF_ERR_NO_DEVICE, "no CUDA device");
    const char* err = "";
    const int rc = odf::ensure_device_ready(device, &err);
    if (rc != ODF_OK) return set_error(rc, err);
    *status = odf::device_status_ptr(device);
    if (sm_count != nullptr) *sm_count = odf::device_sm_count(device);
    return ODF_OK;
}

// Contiguous strides when all are zero; element counts of one stride in 16-byte steps otherwise.
int resolve(const int64_t in[3], int64_t heads, int64_t tokens, int64_t feat, int64_t es, int64_t out[3],
            const char* what) {
    if (in[0] == 0 && in[1] == 0 && in[2] == 0) {
        out[2] = feat;
        out[1] = tokens * feat;
        out[0] = heads * tokens * feat;
        return ODF_OK;
    }
    for (int i = 0; i < 3; ++i) {
        if (in[i] <= 0 || in[i] > (int64_t{1} << 48) || (in[i] * es) % 16 != 0) return set_error(ODF_ERR_INVALID_ARG, what);
        out[i] = in[i];
    }
    return ODF_OK;
}

// Checks of the cache itself; `tables` adds the page table's (not read by page copies).
int view_of(const odf_paged_cache* c, bool tables, odf::PagedView* out) {
    if (c->k_pages == nullptr || c->v_pages == nullptr)
        return set_error(ODF_ERR_INVALID_ARG, "cache pointers must be non-null");
    if (c->kv_dtype != ODF_DTYPE_BF16 && c->kv_dtype != ODF_DTYPE_E4M3)
        return set_error(ODF_ERR_UNSUPPORTED, "a cache holds bf16 or e4m3");
    if (c->num_pages <= 0 || c->heads_kv <= 0 || c->page_size <= 0 || c->head_dim <= 0)
        return set_error(ODF_ERR_INVALID_ARG, "cache dimensions must be non-zero");
    if (c->head_dim != 64 && c->head_dim != 128)
        return set_error(ODF_ERR_UNSUPPORTED, "the sm_100a kernels support head_dim in {64, 128}");
    if (c->num_pages > 0x7fffffffLL || c->heads_kv > 65535 || c->page_size > 65536)
        return set_error(ODF_ERR_UNSUPPORTED, "cache dimensions beyond the kernels' limits");
    if (!aligned(c->k_pages, 16) || !aligned(c->v_pages, 16))
        return set_error(ODF_ERR_INVALID_ARG, "cache pointers must be 16-byte aligned");
    const int64_t es = c->kv_dtype == ODF_DTYPE_BF16 ? 2 : 1;
    const char* bad = "cache strides must be positive multiples of 16 bytes (or all zero for contiguous)";
    int64_t ks[3], vs[3];
    int rc = resolve(c->k_strides, c->heads_kv, c->page_size, c->head_dim, es, ks, bad);
    if (rc == ODF_OK) rc = resolve(c->v_strides, c->heads_kv, c->page_size, c->head_dim, es, vs, bad);
    if (rc != ODF_OK) return rc;
    if (c->kv_dtype == ODF_DTYPE_BF16 && (c->k_scale != nullptr || c->v_scale != nullptr))
        return set_error(ODF_ERR_INVALID_ARG, "scales belong to an e4m3 cache");
    if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return set_error(ODF_ERR_INVALID_ARG, "scales must be 4-byte aligned");
    std::memset(out, 0, sizeof(*out));
    out->k = static_cast<uint8_t*>(c->k_pages);
    out->v = static_cast<uint8_t*>(c->v_pages);
    out->k_page = ks[0] * es;
    out->k_head = ks[1] * es;
    out->k_slot = ks[2] * es;
    out->v_page = vs[0] * es;
    out->v_head = vs[1] * es;
    out->v_slot = vs[2] * es;
    out->num_pages = static_cast<int32_t>(c->num_pages);
    out->page_size = static_cast<int32_t>(c->page_size);
    out->heads_kv = static_cast<int32_t>(c->heads_kv);
    out->fd_page = odf::make_fastdiv(static_cast<uint32_t>(c->page_size));
    out->k_scale = c->k_scale;
    out->v_scale = c->v_scale;
    if (!tables) return ODF_OK;
    if (c->page_table == nullptr || c->max_pages <= 0)
        return set_error(ODF_ERR_INVALID_ARG, "a page table of at least one page per sequence is needed");
    if (!aligned(c->page_table, 4)) return set_error(ODF_ERR_INVALID_ARG, "the page table must be 4-byte aligned");
    if (c->table_stride < 0 || (c->table_stride != 0 && c->table_stride < c->max_pages))
        return set_error(ODF_ERR_INVALID_ARG, "table_stride must be 0 or at least max_pages");
    if (c->max_pages > 0x7fffffffLL / c->page_size)
        return set_error(ODF_ERR_UNSUPPORTED, "max_pages * page_size must be below 2^31");
    out->table = c->page_table;
    out->table_stride = c->table_stride != 0 ? c->table_stride : c->max_pages;
    out->max_pages = static_cast<int32_t>(c->max_pages);
    return ODF_OK;
}

// Ids of page copies, in order: inside the cache, no page written twice, none both read and written.  A few
// pairs are compared with one another, many by a byte per page of the cache.
int check_pairs(const int32_t* ids, int64_t n_pairs, int64_t num_pages) {
    constexpr int64_t kFew = 32;
    const char* twice = "a page is written twice";
    const char* read = "a written page is also read";
    std::vector<uint8_t> role;  // 1 = read, 2 = written
    if (n_pairs > kFew) {
        try {
            role.resize(static_cast<size_t>(num_pages), 0);
        } catch (const std::exception&) {
            return set_error(ODF_ERR_UNSUPPORTED, "out of host memory");
        }
    }
    for (int64_t i = 0; i < 2 * n_pairs; ++i) {
        const int32_t id = ids[i];
        if (id < 0 || id >= num_pages) return set_error(ODF_ERR_INVALID_ARG, "a page id is outside the cache");
        if (n_pairs > kFew) {
            if ((i & 1) && role[id] == 2) return set_error(ODF_ERR_INVALID_ARG, twice);
            role[id] |= (i & 1) ? 2 : 1;
            if (role[id] == 3) return set_error(ODF_ERR_INVALID_ARG, read);
        } else {
            for (int64_t j = 0; j < i; ++j) {
                if (ids[j] != id || (~i & ~j & 1)) continue;
                return set_error(ODF_ERR_INVALID_ARG, (i & j & 1) ? twice : read);
            }
        }
    }
    return ODF_OK;
}

// Joins a page's rows into runs of consecutive bytes.
void page_runs(int64_t heads, int64_t slots, int64_t row, int64_t head_stride, int64_t slot_stride, int which,
               odf::CopyArgs* a) {
    // the axis with the smaller stride is the inner one
    int64_t n_in = slots, s_in = slot_stride, n_out = heads, s_out = head_stride;
    if (n_in == 1 || (n_out > 1 && s_out < s_in)) {
        std::swap(n_in, n_out);
        std::swap(s_in, s_out);
    }
    int64_t run = row;
    if (n_in == 1 || s_in == run) {
        run *= n_in;
        n_in = 1;
        if (n_out == 1 || s_out == run) {
            run *= n_out;
            n_out = 1;
        }
    }
    a->run_bytes[which] = run;
    a->inner[which] = static_cast<int32_t>(n_in);
    a->inner_stride[which] = s_in;
    a->outer[which] = static_cast<int32_t>(n_out);
    a->outer_stride[which] = s_out;
}

}  // namespace

extern "C" {

size_t odf_paged_decode_workspace_size(const odf_decode_params* p) {
    if (p == nullptr) return 0;
    return odf::decode_workspace_bytes(static_cast<int32_t>(p->cache.head_dim));
}

int odf_paged_decode_sm100(const odf_decode_params* p, void* stream) {
    if (p == nullptr) return set_error(ODF_ERR_INVALID_ARG, "params must be non-null");
    if (p->q == nullptr || p->o == nullptr || p->lens == nullptr)
        return set_error(ODF_ERR_INVALID_ARG, "attention input/output pointers must be non-null");
    if (p->batch <= 0 || p->heads_q <= 0) return set_error(ODF_ERR_INVALID_ARG, "attention dimensions must be non-zero");
    odf::DecodeArgs a;
    std::memset(&a, 0, sizeof(a));
    int rc = view_of(&p->cache, true, &a.c);
    if (rc != ODF_OK) return rc;
    if (p->heads_q % p->cache.heads_kv != 0)
        return set_error(ODF_ERR_INVALID_ARG, "heads_q must be a multiple of heads_kv");
    if (p->batch > 0x7fffff || p->heads_q > 65535 || p->batch * p->heads_q > 0x7fffffffLL)
        return set_error(ODF_ERR_UNSUPPORTED, "batch or heads beyond the kernel's limits");
    // the kernel counts rows of the cache in 16-byte units of 32 bits
    for (int which = 0; which < 2; ++which) {
        const double reach = static_cast<double>(which ? a.c.v_page : a.c.k_page) * (a.c.num_pages - 1) +
                             static_cast<double>(which ? a.c.v_head : a.c.k_head) * (a.c.heads_kv - 1) +
                             static_cast<double>(which ? a.c.v_slot : a.c.k_slot) * (a.c.page_size - 1) + 256.0;
        if (reach > 16.0 * 4294967295.0)
            return set_error(ODF_ERR_UNSUPPORTED, "K or V pages of one layer span more than 64 GB");
    }
    if (p->o_dtype != ODF_DTYPE_F32 && p->o_dtype != ODF_DTYPE_BF16)
        return set_error(ODF_ERR_UNSUPPORTED, "output dtype must be f32 or bf16");
    if (!std::isfinite(p->scale)) return set_error(ODF_ERR_INVALID_ARG, "scale must be finite");
    if (!(p->softcap >= 0.0f) || !std::isfinite(p->softcap))
        return set_error(ODF_ERR_INVALID_ARG, "softcap must be finite and >= 0");
    if (p->window < 0 || p->sinks < 0) return set_error(ODF_ERR_INVALID_ARG, "window and sinks must be >= 0");
    if (p->bias_kind != ODF_BIAS_NONE && p->bias_kind != ODF_BIAS_ALIBI)
        return set_error(ODF_ERR_UNSUPPORTED, "only BiasKind::None and AlibiGenerated run in the decode kernel");
    if (p->bias_kind == ODF_BIAS_ALIBI && p->alibi_slopes != nullptr && p->heads_q > ODF_MAX_EXPLICIT_SLOPES)
        return set_error(ODF_ERR_UNSUPPORTED, "explicit ALiBi slopes are limited to 256 heads (use generated slopes)");
    if (!aligned(p->q, 16) || !aligned(p->o, 16)) return set_error(ODF_ERR_INVALID_ARG, "device pointers must be 16-byte aligned");
    if (!aligned(p->lens, 4) || !aligned(p->lse, 4))
        return set_error(ODF_ERR_INVALID_ARG, "lens and lse must be 4-byte aligned");
    const int64_t D = p->cache.head_dim;
    const int64_t oes = p->o_dtype == ODF_DTYPE_BF16 ? 2 : 4;
    const bool q_dense = p->q_strides[0] == 0 && p->q_strides[1] == 0;
    const bool o_dense = p->o_strides[0] == 0 && p->o_strides[1] == 0;
    a.q_b = q_dense ? p->heads_q * D : p->q_strides[0];
    a.q_h = q_dense ? D : p->q_strides[1];
    a.o_b = o_dense ? p->heads_q * D : p->o_strides[0];
    a.o_h = o_dense ? D : p->o_strides[1];
    if (a.q_b <= 0 || a.q_h <= 0 || a.o_b <= 0 || a.o_h <= 0 || a.q_b % 8 || a.q_h % 8 || (a.o_b * oes) % 16 ||
        (a.o_h * oes) % 16)
        return set_error(ODF_ERR_INVALID_ARG, "q and o strides must be positive multiples of 16 bytes (or all zero for contiguous)");
    a.batch = static_cast<int32_t>(p->batch);
    a.heads_q = static_cast<int32_t>(p->heads_q);
    a.group = static_cast<int32_t>(p->heads_q / p->cache.heads_kv);
    a.window = static_cast<int32_t>(std::min<int64_t>(p->window, 0x7fffffff));
    a.sinks = static_cast<int32_t>(std::min<int64_t>(p->sinks, 0x7fffffff));
    if (!odf::decode_work_fits(a, static_cast<int32_t>(D), p->cache.kv_dtype))
        return set_error(ODF_ERR_UNSUPPORTED, "batch x kv-heads x the page table's room is beyond the kernel's 32 bits");
    if (p->workspace == nullptr || p->workspace_bytes < odf_paged_decode_workspace_size(p))
        return set_error(ODF_ERR_INVALID_ARG, "the workspace is smaller than odf_paged_decode_workspace_size() bytes");
    if (!aligned(p->workspace, 16)) return set_error(ODF_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
    int sm_count = 0;
    rc = current_device_ready(&a.c.status, &sm_count);
    if (rc != ODF_OK) return rc;
    a.q = p->q;
    a.o = p->o;
    a.lse = p->lse;
    a.lens = p->lens;
    a.o_bf16 = p->o_dtype == ODF_DTYPE_BF16;
    a.scale = p->scale;
    a.softcap = p->softcap;
    a.inv_softcap = p->softcap > 0.0f ? 1.0f / p->softcap : 0.0f;
    a.has_alibi = p->bias_kind == ODF_BIAS_ALIBI;
    if (a.has_alibi) {
        if (p->alibi_slopes != nullptr) {
            std::copy(p->alibi_slopes, p->alibi_slopes + p->heads_q, a.alibi_slopes);
        } else if (p->heads_q <= ODF_MAX_EXPLICIT_SLOPES) {
            for (int64_t h = 0; h < p->heads_q; ++h) a.alibi_slopes[h] = odf::generated_alibi_slope(h, p->heads_q);
        } else {
            a.alibi_generated = 1;
        }
    }
    a.workspace = p->workspace;
    a.sm_count = sm_count;
    const char* err = "";
    rc = odf::launch_paged_decode(a, static_cast<int32_t>(D), p->cache.kv_dtype, static_cast<cudaStream_t>(stream), &err);
    return rc == ODF_OK ? ODF_OK : set_error(rc, err);
}

int odf_paged_append_sm100(const odf_append_params* p, void* stream) {
    if (p == nullptr) return set_error(ODF_ERR_INVALID_ARG, "params must be non-null");
    if (p->k == nullptr || p->v == nullptr || p->starts == nullptr)
        return set_error(ODF_ERR_INVALID_ARG, "k, v and starts must be non-null");
    if (p->batch <= 0 || p->tokens <= 0) return set_error(ODF_ERR_INVALID_ARG, "batch and tokens must be non-zero");
    odf::AppendArgs a;
    std::memset(&a, 0, sizeof(a));
    int rc = view_of(&p->cache, true, &a.c);
    if (rc != ODF_OK) return rc;
    if (p->batch > 0x7fffff || p->tokens > 0x7fffffffLL || p->batch * p->tokens > (int64_t{1} << 40))
        return set_error(ODF_ERR_UNSUPPORTED, "batch or tokens beyond the kernel's limits");
    if (!aligned(p->k, 16) || !aligned(p->v, 16)) return set_error(ODF_ERR_INVALID_ARG, "device pointers must be 16-byte aligned");
    if (!aligned(p->starts, 4) || !aligned(p->counts, 4))
        return set_error(ODF_ERR_INVALID_ARG, "starts and counts must be 4-byte aligned");
    int64_t ks[3], vs[3];
    const char* bad = "k and v strides must be positive multiples of 16 bytes (or all zero for contiguous)";
    rc = resolve(p->k_strides, p->cache.heads_kv, p->tokens, p->cache.head_dim, 2, ks, bad);
    if (rc == ODF_OK) rc = resolve(p->v_strides, p->cache.heads_kv, p->tokens, p->cache.head_dim, 2, vs, bad);
    if (rc != ODF_OK) return rc;
    int sm_count = 0;
    rc = current_device_ready(&a.c.status, &sm_count);
    if (rc != ODF_OK) return rc;
    a.k = p->k;
    a.v = p->v;
    a.k_b = ks[0];
    a.k_h = ks[1];
    a.k_t = ks[2];
    a.v_b = vs[0];
    a.v_h = vs[1];
    a.v_t = vs[2];
    a.starts = p->starts;
    a.counts = p->counts;
    a.batch = static_cast<int32_t>(p->batch);
    a.tokens = static_cast<int32_t>(p->tokens);
    a.sm_count = sm_count;
    const char* err = "";
    rc = odf::launch_paged_append(a, static_cast<int32_t>(p->cache.head_dim), p->cache.kv_dtype,
                                  static_cast<cudaStream_t>(stream), &err);
    return rc == ODF_OK ? ODF_OK : set_error(rc, err);
}

int odf_page_copy_sm100(const odf_page_copy_params* p, void* stream) {
    if (p == nullptr) return set_error(ODF_ERR_INVALID_ARG, "params must be non-null");
    odf::PagedView c;
    int rc = view_of(&p->cache, false, &c);
    if (rc != ODF_OK) return rc;
    if (p->layers <= 0 || p->layers > 65535) return set_error(ODF_ERR_INVALID_ARG, "layers must be in [1, 65535]");
    if (p->n_pairs < 0 || (p->n_pairs > 0 && p->pairs == nullptr))
        return set_error(ODF_ERR_INVALID_ARG, "pairs must be non-null");
    if (p->n_pairs > p->cache.num_pages) return set_error(ODF_ERR_INVALID_ARG, "a page is written twice");
    const int64_t es = p->cache.kv_dtype == ODF_DTYPE_BF16 ? 2 : 1;
    if (p->layers > 1) {
        for (int64_t s : {p->k_layer_stride, p->v_layer_stride})
            if (s <= 0 || s > (int64_t{1} << 48) || (s * es) % 16 != 0)
                return set_error(ODF_ERR_INVALID_ARG, "layer strides must be positive multiples of 16 bytes");
    }
    rc = check_pairs(p->pairs, p->n_pairs, p->cache.num_pages);
    if (rc != ODF_OK || p->n_pairs == 0) return rc;
    int* status = nullptr;
    rc = current_device_ready(&status);
    if (rc != ODF_OK) return rc;
    odf::CopyArgs a;
    std::memset(&a, 0, sizeof(a));
    a.base[0] = c.k;
    a.base[1] = c.v;
    a.page[0] = c.k_page;
    a.page[1] = c.v_page;
    a.layer[0] = p->layers > 1 ? p->k_layer_stride * es : 0;
    a.layer[1] = p->layers > 1 ? p->v_layer_stride * es : 0;
    const int64_t row = p->cache.head_dim * es;
    page_runs(p->cache.heads_kv, p->cache.page_size, row, c.k_head, c.k_slot, 0, &a);
    page_runs(p->cache.heads_kv, p->cache.page_size, row, c.v_head, c.v_slot, 1, &a);
    a.layers = static_cast<int32_t>(p->layers);
    a.pairs = p->pairs;
    a.n_pairs = p->n_pairs;
    const char* err = "";
    rc = odf::launch_page_copy(a, static_cast<cudaStream_t>(stream), &err);
    return rc == ODF_OK ? ODF_OK : set_error(rc, err);
}

}  // extern "C"
