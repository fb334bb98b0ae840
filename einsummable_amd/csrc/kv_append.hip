// es_km_kv_append: the new tokens' queries and keys rotated by their positions, keys and values
// written into the cache's pages.
//
//   token i of sequence s:  pos = lens[s] - (offsets[s+1] - i)
//   z_j = x_a(j) + i x_b(j) times (cos, sin)[pos][j]:  a' = a c - b s,  b' = a s + b c
//   pairs: (a, b) = (2j, 2j+1);  halves: (a, b) = (j, j + d/2)
//
// Bound by memory: 2 * (H + 2 KV) * d * size bytes per token and the rows of the frequency
// table; a step of a few tokens is bound by the launch and three dependent loads (offsets,
// page, store).  The elements of a token are independent of its position until the rotation,
// so a thread asks for them before it looks for the sequence, and what it looked up (position,
// page, its column of the frequencies) serves the same column of several heads.  Prompts of 7877
// tokens, 391 MB: 77 us, 5.1 TB/s, the rate of a copy; 64 tokens: 3.4 us.
#include "kernel_manager.h"
#include "serving.h"
#include "serving_device.h"

namespace es
{

namespace
{

struct append_dev_t {
    char const *   q, *k, *v;
    char *         q_out, *kc, *vc;
    float const*   freqs;
    int const*     offsets;
    int const*     lens;
    int const*     table;
    uint64_t       table_stride;
    uint64_t       page_stride, token_stride, head_stride;          // cache, elements
    uint64_t       q_stride, k_stride, v_stride, q_out_stride;  // elements
    uint64_t       n_pages;
    int64_t        n_pos;
    int            n_seqs, n_tokens, max_pages, page_size;
    int            h_q, h_kv, d;
    int            units;     // threads that serve one head: d / 2 / VP
    int            per_pass;  // heads per pass of the workgroup
};

template <typename T, int N>
struct __attribute__((aligned(sizeof(T) * N < 16 ? sizeof(T) * N : 16))) pack_t {
    T x[N];
};

// The 2 * VP elements of a head that column u owns: one group, or one in each half.
template <typename T, int VP, int ROPE>
struct column_t {
    static constexpr bool APART = ROPE == ES_KM_ROPE_HALVES;
    static constexpr int  GROUPS = APART ? 2 : 1;
    static constexpr int  N = 2 * VP / GROUPS;
    pack_t<T, N>          g[GROUPS];

    static __device__ int at(int group, int u, int d) { return group * (d / 2) + u * N; }
    __device__ void       load(T const* head, int u, int d)
    {
#pragma unroll
        for (int i = 0; i != GROUPS; ++i) {
            g[i] = *reinterpret_cast<pack_t<T, N> const*>(head + at(i, u, d));
        }
    }
    __device__ void store(T* head, int u, int d) const
    {
#pragma unroll
        for (int i = 0; i != GROUPS; ++i) {
            *reinterpret_cast<pack_t<T, N>*>(head + at(i, u, d)) = g[i];
        }
    }
    __device__ T& re(int e) { return APART ? g[0].x[e] : g[0].x[2 * e]; }
    __device__ T& im(int e) { return APART ? g[GROUPS - 1].x[e] : g[0].x[2 * e + 1]; }
};

// VP pairs per thread, heads taken UNR at a time.
template <typename T, int VP, int ROPE, int UNR>
__global__ __launch_bounds__(256) void kv_append_kernel(append_dev_t a)
{
    int const token = int(blockIdx.x);
    int const tid = int(threadIdx.x);
    int const hl = tid / a.units;       // head within a pass
    int const u = tid - hl * a.units;   // column
    bool const mine = hl < a.per_pass;
    int const heads = (a.q ? a.h_q : 0) + 2 * a.h_kv;
    int const h0 = int(blockIdx.y) * a.per_pass * UNR + hl;
    int const h_q = a.q ? a.h_q : 0;

    column_t<T, VP, ROPE> x[UNR];
#pragma unroll
    for (int i = 0; i != UNR; ++i) {
        int const h = h0 + i * a.per_pass;
        if (!mine || h >= heads) continue;
        T const* src;
        if (h < h_q) {
            src = reinterpret_cast<T const*>(a.q) + uint64_t(token) * a.q_stride + uint64_t(h) * a.d;
        } else if (h < h_q + a.h_kv) {
            src = reinterpret_cast<T const*>(a.k) + uint64_t(token) * a.k_stride +
                  uint64_t(h - h_q) * a.d;
        } else {
            src = reinterpret_cast<T const*>(a.v) + uint64_t(token) * a.v_stride +
                  uint64_t(h - h_q - a.h_kv) * a.d;
        }
        x[i].load(src, u, a.d);
    }

    int       first, end;
    int const s = find_sequence(a.offsets, a.n_seqs, token, &first, &end);
    if (s < 0) return;
    int const pos = a.lens[s] - (end - token);
    if (pos < 0 || (ROPE != ES_KM_ROPE_NONE && pos >= a.n_pos)) return;
    int const pi = pos / a.page_size;
    int const page = pi < a.max_pages ? a.table[uint64_t(s) * a.table_stride + uint64_t(pi)] : -1;
    bool const  stored = page >= 0 && uint64_t(page) < a.n_pages;
    uint64_t const row = uint64_t(stored ? page : 0) * a.page_stride +
                         uint64_t(pos - pi * a.page_size) * a.token_stride;
    float c[VP], sn[VP];
    if (ROPE != ES_KM_ROPE_NONE && mine) {
        float const* f = a.freqs + (uint64_t(pos) * uint64_t(a.d / 2) + uint64_t(u) * VP) * 2;
#pragma unroll
        for (int e = 0; e != VP; ++e) {
            float2_t const cs = *reinterpret_cast<float2_t const*>(f + 2 * e);
            c[e] = cs.x;
            sn[e] = cs.y;
        }
    }
#pragma unroll
    for (int i = 0; i != UNR; ++i) {
        int const h = h0 + i * a.per_pass;
        if (!mine || h >= heads) continue;
        bool const value = h >= h_q + a.h_kv;
        if (h >= h_q && !stored) continue;
        T* dst;
        if (h < h_q) {
            dst = reinterpret_cast<T*>(a.q_out) + uint64_t(token) * a.q_out_stride +
                  uint64_t(h) * a.d;
        } else if (!value) {
            dst = reinterpret_cast<T*>(a.kc) + row + uint64_t(h - h_q) * a.head_stride;
        } else {
            dst = reinterpret_cast<T*>(a.vc) + row + uint64_t(h - h_q - a.h_kv) * a.head_stride;
        }
        if (ROPE != ES_KM_ROPE_NONE && !value) {
#pragma unroll
            for (int e = 0; e != VP; ++e) {
                float const re = float(x[i].re(e)), im = float(x[i].im(e));
                x[i].re(e) = T(re * c[e] - im * sn[e]);
                x[i].im(e) = T(re * sn[e] + im * c[e]);
            }
        }
        x[i].store(dst, u, a.d);
    }
}

template <typename T, int VP, int ROPE>
void launch_one(append_dev_t const& a, hipStream_t stream)
{
    int const heads = (a.q ? a.h_q : 0) + 2 * a.h_kv;
    // Four heads to a thread where tokens alone fill the device (two workgroups per compute unit):
    // 7877 tokens 77 us, 100 us with one; 64 tokens 4.1 us, 3.3 us with one.
    constexpr int UNR = 4;
    if (a.n_tokens >= 512) {
        dim3 const grid(uint32_t(a.n_tokens),
                        uint32_t((heads + a.per_pass * UNR - 1) / (a.per_pass * UNR)));
        kv_append_kernel<T, VP, ROPE, UNR><<<grid, 256, 0, stream>>>(a);
    } else {
        dim3 const grid(uint32_t(a.n_tokens), uint32_t((heads + a.per_pass - 1) / a.per_pass));
        kv_append_kernel<T, VP, ROPE, 1><<<grid, 256, 0, stream>>>(a);
    }
}

template <typename T, int VP>
void launch_rope(append_dev_t& a, int rope, hipStream_t stream)
{
    a.units = a.d / 2 / VP;
    a.per_pass = 256 / a.units;
    if (rope == ES_KM_ROPE_PAIRS) {
        launch_one<T, VP, ES_KM_ROPE_PAIRS>(a, stream);
    } else if (rope == ES_KM_ROPE_HALVES) {
        launch_one<T, VP, ES_KM_ROPE_HALVES>(a, stream);
    } else {
        launch_one<T, VP, ES_KM_ROPE_NONE>(a, stream);
    }
}

}  // namespace

void launch_kv_append(kv_append_args_t const& g, hipStream_t stream)
{
    append_dev_t a;
    a.q = static_cast<char const*>(g.q);
    a.k = static_cast<char const*>(g.k);
    a.v = static_cast<char const*>(g.v);
    a.q_out = static_cast<char*>(g.q_out);
    a.kc = static_cast<char*>(g.cache.k);
    a.vc = static_cast<char*>(g.cache.v);
    a.freqs = g.freqs;
    a.offsets = g.batch.offsets;
    a.lens = g.batch.lens;
    a.table = g.batch.page_table;
    a.table_stride = g.batch.table_stride;
    a.page_stride = g.cache.page_stride;
    a.token_stride = g.cache.token_stride;
    a.head_stride = g.cache.head_stride;
    a.q_stride = g.q_stride;
    a.k_stride = g.k_stride;
    a.v_stride = g.v_stride;
    a.q_out_stride = g.q_out_stride;
    a.n_pages = g.cache.n_pages;
    a.n_pos = int64_t(g.n_pos);
    a.n_seqs = g.batch.n_seqs;
    a.max_pages = g.batch.max_pages;
    a.page_size = g.cache.page_size;
    a.h_q = g.cache.n_heads;
    a.h_kv = g.cache.n_kv_heads;
    a.d = g.cache.head_dim;
    a.n_tokens = g.batch.n_tokens;
    if (a.n_tokens == 0 || a.n_seqs == 0) return;
    if (g.cache.dtype == ES_KM_F16) {
        launch_rope<_Float16, 4>(a, g.rope, stream);
    } else {
        launch_rope<float, 4>(a, g.rope, stream);
    }
    hipError_t const err = hipGetLastError();
    if (err != hipSuccess) {
        throw km_error(km_status::device,
                       std::string("kv_append launch: ") + hipGetErrorString(err));
    }
}

}  // namespace es
