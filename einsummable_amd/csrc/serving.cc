// Argument checks and device handling of the serving operators (include/es_km.h).  Everything a
// kernel's own bounds checks cannot turn into a dropped row is refused here.
#include "serving.h"

#include "ir.h"
#include "kernel_manager.h"

#include <string>

namespace es
{

device_scope_t::device_scope_t(int device)
{
    int current = -1;
    if (hipGetDevice(&current) == hipSuccess && current != device) {
        hipError_t const err = hipSetDevice(device);
        if (err != hipSuccess) {
            throw km_error(km_status::device,
                           std::string("hipSetDevice: ") + hipGetErrorString(err));
        }
        previous_ = current;
    }
}

device_scope_t::~device_scope_t()
{
    if (previous_ >= 0) (void)hipSetDevice(previous_);
}

namespace
{

void need(bool ok, char const* what)
{
    if (!ok) throw ir_error(what);
}

bool aligned(void const* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

uint64_t size_of(int dtype) { return dtype == ES_KM_F16 ? 2 : 4; }

bool served(int dtype) { return dtype == ES_KM_F16 || dtype == ES_KM_F32; }

// no address of the kernels passes 2^62 bytes
constexpr uint64_t STRIDE_MAX = 1ull << 40;

}  // namespace

int check_cache(es_km_kv_cache_t const* c, bool with_buffers)
{
    need(c != nullptr, "kv cache: null descriptor");
    need(c->dtype >= 0 && c->dtype <= 3, "kv cache: bad dtype");
    need(c->n_kv_heads >= 1 && c->n_heads >= 1 && c->n_heads <= 65536 &&
             c->n_heads % c->n_kv_heads == 0,
         "kv cache: n_heads has to be a multiple of n_kv_heads");
    need(c->head_dim >= 1, "kv cache: bad head_dim");
    need(c->page_size >= 1 && c->page_size <= (1 << 20), "kv cache: bad page_size");
    if (!served(c->dtype)) return ES_KM_UNSUPPORTED;
    if (c->head_dim % 8 != 0 || c->head_dim > 256) return ES_KM_UNSUPPORTED;
    uint64_t const e = size_of(c->dtype);
    need(c->n_pages >= 1 && c->n_pages <= 0x7fffffffull, "kv cache: bad n_pages");
    need(c->page_stride < STRIDE_MAX && c->token_stride < STRIDE_MAX &&
             c->head_stride < STRIDE_MAX,
         "kv cache: stride beyond 2^40 elements");
    need(c->page_stride * e % 16 == 0 && c->token_stride * e % 16 == 0 &&
             c->head_stride * e % 16 == 0,
         "kv cache: strides have to be multiples of 16 bytes");
    if (with_buffers) {
        need(c->k && c->v, "kv cache: null buffer");
        need(aligned(c->k, 16) && aligned(c->v, 16), "kv cache: buffers have to be 16-byte aligned");
    }
    return ES_KM_OK;
}

int check_batch(es_km_kv_batch_t const* b, bool with_buffers)
{
    need(b != nullptr, "kv batch: null descriptor");
    need(b->n_seqs >= 0 && b->n_seqs <= (1 << 20), "kv batch: n_seqs beyond 0 .. 2^20");
    need(b->n_tokens >= 0 && b->n_tokens <= (1 << 22), "kv batch: n_tokens beyond 0 .. 2^22");
    need(b->max_pages >= 1, "kv batch: bad max_pages");
    need(b->table_stride >= uint64_t(b->max_pages) || b->n_seqs <= 1,
         "kv batch: table_stride below max_pages");
    need(b->table_stride < STRIDE_MAX, "kv batch: stride beyond 2^40 elements");
    if (with_buffers && b->n_seqs > 0 && b->n_tokens > 0) {
        need(b->offsets && b->lens && b->page_table, "kv batch: null buffer");
        need(aligned(b->offsets, 4) && aligned(b->lens, 4) && aligned(b->page_table, 4),
             "kv batch: arrays have to be 4-byte aligned");
    }
    return ES_KM_OK;
}

namespace
{

// positions are int32 in the kernels, and so are the products of a page's number and its size
void check_reach(es_km_kv_cache_t const& c, es_km_kv_batch_t const& b)
{
    need(uint64_t(b.max_pages) * uint64_t(c.page_size) <= (1ull << 30),
         "kv batch: max_pages * page_size beyond 2^30 positions");
}

void check_rows(void const* p, uint64_t stride, uint64_t width, uint64_t e, int n_tokens,
                std::string const& what)
{
    if (n_tokens == 0) return;
    need(p != nullptr, (what + ": null buffer").c_str());
    need(aligned(p, 16), (what + ": has to be 16-byte aligned").c_str());
    need(stride < STRIDE_MAX, (what + ": stride beyond 2^40 elements").c_str());
    need(n_tokens == 1 || (stride >= width && stride * e % 16 == 0),
         (what + ": its stride has to hold a row and be a multiple of 16 bytes").c_str());
}

}  // namespace

int check_kv_append(kv_append_args_t const& a)
{
    if (int const rc = check_cache(&a.cache, true)) return rc;
    if (int const rc = check_batch(&a.batch, true)) return rc;
    check_reach(a.cache, a.batch);
    uint64_t const e = size_of(a.cache.dtype);
    uint64_t const d = uint64_t(a.cache.head_dim);
    int const      n = a.batch.n_tokens;
    need((a.q == nullptr) == (a.q_out == nullptr), "kv_append: q and q_out go together");
    if (a.q) {
        check_rows(a.q, a.q_stride, uint64_t(a.cache.n_heads) * d, e, n, "kv_append: q");
        check_rows(a.q_out, a.q_out_stride, uint64_t(a.cache.n_heads) * d, e, n,
                   "kv_append: q_out");
        need(a.q != a.q_out || a.q_stride == a.q_out_stride || n <= 1,
             "kv_append: q_out on top of q needs q's stride");
    }
    check_rows(a.k, a.k_stride, uint64_t(a.cache.n_kv_heads) * d, e, n, "kv_append: k");
    check_rows(a.v, a.v_stride, uint64_t(a.cache.n_kv_heads) * d, e, n, "kv_append: v");
    need(a.rope >= ES_KM_ROPE_NONE && a.rope <= ES_KM_ROPE_HALVES, "kv_append: bad rope");
    if (a.rope == ES_KM_ROPE_NONE) {
        need(a.freqs == nullptr, "kv_append: frequencies without a rotation");
    } else {
        need(a.freqs != nullptr && a.n_pos >= 1, "kv_append: a rotation needs frequencies");
        need(aligned(a.freqs, 8), "kv_append: frequencies have to be 8-byte aligned");
        need(a.n_pos <= (1ull << 31), "kv_append: n_pos beyond 2^31");
    }
    return ES_KM_OK;
}

int check_attention(attention_args_t const& a)
{
    if (int const rc = check_cache(&a.cache, true)) return rc;
    if (int const rc = check_batch(&a.batch, true)) return rc;
    check_reach(a.cache, a.batch);
    uint64_t const e = size_of(a.cache.dtype);
    uint64_t const width = uint64_t(a.cache.n_heads) * uint64_t(a.cache.head_dim);
    need(a.shared <= (1ull << 30), "prefix_attention: shared beyond 2^30 positions");
    need(a.scale == a.scale && a.scale - a.scale == 0.0f, "prefix_attention: scale is not finite");
    check_rows(a.q, a.q_stride, width, e, a.batch.n_tokens, "prefix_attention: q");
    check_rows(a.out, a.out_stride, width, e, a.batch.n_tokens, "prefix_attention: out");
    need(a.q != a.out || a.batch.n_tokens == 0, "prefix_attention: out on top of q");
    return ES_KM_OK;
}

int check_int4_weight(es_km_int4_weight_t const* w, bool with_buffers)
{
    need(w != nullptr, "int4 weight: null descriptor");
    need(w->dtype >= 0 && w->dtype <= 3, "int4 weight: bad dtype");
    need(w->n >= 1 && w->k >= 1 && w->group >= 1, "int4 weight: empty");
    if (!served(w->dtype)) return ES_KM_UNSUPPORTED;
    if (w->k % 32 != 0 || w->group % 32 != 0 || w->k > (1u << 20) || w->n > (1u << 26)) {
        return ES_KM_UNSUPPORTED;
    }
    uint64_t const groups = (w->k + w->group - 1) / w->group;
    need(w->n == 1 || (w->w_stride >= w->k / 2 && w->scale_stride >= groups),
         "int4 weight: a stride below its row");
    need(w->w_stride % 16 == 0 && w->w_stride < STRIDE_MAX && w->scale_stride < STRIDE_MAX,
         "int4 weight: w_stride has to be a multiple of 16 bytes");
    if (with_buffers) {
        need(w->w && w->scales, "int4 weight: null buffer");
        need(aligned(w->w, 16), "int4 weight: w has to be 16-byte aligned");
        need(aligned(w->scales, size_of(w->dtype)), "int4 weight: scales are not aligned");
    }
    return ES_KM_OK;
}

int check_int4_linear(int4_args_t const& a)
{
    if (int const rc = check_int4_weight(&a.w, true)) return rc;
    need(a.m <= 65536, "int4_linear: more than 65536 tokens");
    uint64_t const e = size_of(a.w.dtype);
    check_rows(a.x, a.x_stride, a.w.k, e, int(a.m), "int4_linear: x");
    if (a.m > 0) {
        need(a.y != nullptr, "int4_linear: null output");
        need(aligned(a.y, e), "int4_linear: y is not aligned");
        need(a.m == 1 || (a.y_stride >= a.w.n && a.y_stride < STRIDE_MAX),
             "int4_linear: y's stride has to hold a row");
        need(a.x != a.y, "int4_linear: y on top of x");
    }
    return ES_KM_OK;
}

}  // namespace es
