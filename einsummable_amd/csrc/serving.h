// The operators of a decoder layer's token-by-token step: appending to a paged cache of keys
// and values, attention over it, products with 4-bit weights.  Checked host entries (they
// throw ir_error / km_error and only enqueue work) over kernels in kv_append.hip,
// prefix_attention.hip and int4_linear.hip.
#pragma once
#include "../../include/es_km.h"

#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace es
{

// Makes `device` current for the scope of a launch.  A stream belongs to a device; launching
// on it while another device is current is an error of the HIP runtime.
class device_scope_t
{
public:
    explicit device_scope_t(int device);
    ~device_scope_t();
    device_scope_t(device_scope_t const&) = delete;
    device_scope_t& operator=(device_scope_t const&) = delete;

private:
    int previous_ = -1;
};

// `device` < 0: check the arguments only (what a call without a handle gets to see).
// All of them return an ES_KM_* status: ES_KM_UNSUPPORTED for a valid descriptor that has no
// kernel (the reason in *why), ES_KM_OK otherwise.
struct kv_append_args_t {
    es_km_kv_cache_t cache;
    es_km_kv_batch_t batch;
    void const *     q, *k, *v;
    void*            q_out;
    uint64_t         q_stride, k_stride, v_stride, q_out_stride;  // elements between tokens
    int              rope;
    float const*     freqs;
    uint64_t         n_pos;
};

int check_cache(es_km_kv_cache_t const* cache, bool with_buffers);
int check_batch(es_km_kv_batch_t const* batch, bool with_buffers);

int check_kv_append(kv_append_args_t const& a);
void launch_kv_append(kv_append_args_t const& a, hipStream_t stream);

struct attention_args_t {
    es_km_kv_cache_t cache;
    es_km_kv_batch_t batch;
    uint64_t         shared;  // positions every sequence of the batch has in common
    float            scale;
    void const*      q;
    void*            out;
    uint64_t         q_stride, out_stride;
};

// How one call is cut into workgroups; a function of the sizes the host knows.
struct attention_plan_t {
    uint32_t shared = 0;         // positions treated as shared
    uint32_t prefix_rows = 0;    // rows per tile, shared positions
    uint32_t prefix_tiles = 0;   // row tiles over all tokens of the batch
    uint32_t prefix_splits = 0;  // cuts of the shared positions
    uint32_t prefix_chunk = 0;   // positions per cut
    uint32_t own_rows = 0;       // rows per tile, the sequences' own positions
    uint32_t shares = 0;         // parts of the own positions of the whole batch
    uint32_t own_slots = 0;      // upper bound of (row tile, part) pairs of the own positions
    uint64_t own_base = 0;       // rows of partial results before the own positions'
    uint64_t part_rows = 0;      // rows of partial results
    uint64_t workspace_bytes = 0;
};

int              check_attention(attention_args_t const& a);
attention_plan_t plan_attention(es_km_kv_cache_t const& c, int n_seqs, int n_tokens,
                                uint64_t shared);
void launch_attention(attention_args_t const& a, attention_plan_t const& p, void* workspace,
                      hipStream_t stream);

struct int4_args_t {
    es_km_int4_weight_t w;
    uint64_t            m;
    void const*         x;
    void*               y;
    uint64_t            x_stride, y_stride;  // elements between tokens
};

int      check_int4_weight(es_km_int4_weight_t const* w, bool with_buffers);
int      check_int4_linear(int4_args_t const& a);
uint64_t int4_workspace(es_km_int4_weight_t const& w, uint64_t m);
void     launch_int4_linear(int4_args_t const& a, void* workspace, hipStream_t stream);

}  // namespace es
