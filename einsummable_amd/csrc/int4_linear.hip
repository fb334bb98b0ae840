// es_km_int4_linear: y[i, n] = sum over groups G of scale[n, G] sum_{k in G} (q[n,k] - z[n,G]) x[i,k]
// for a few tokens i.
//
// Bound by the weight's n * k / 2 bytes: each byte is read once per 64 rows of x.  A workgroup
// owns 16 columns n and all of k, its wavefronts take the 128-wide steps of k in turn and join
// their fp32 sums through LDS in a fixed order.  The product X W^T goes through
// v_mfma_f32_16x16x32_f16 even for one token (rows of the tile that hold no token are zero):
// a lane's share of the B operand is eight consecutive k of one n, one dword of the weight as
// it lies in memory, and the matrix unit does the multiplying and adding while the vector unit
// has only the unpacking left.
//
// Unpacking: (w & 0x000f000f) | 0x64006400 is the pair (1024 + q0, 1024 + q4) in f16; minus
// (1024 + z) it is exact.  The nibbles come out in the order 0 4 1 5 2 6 3 7, so x is put in that
// order too.  A lane loads 16 bytes, 32 consecutive k.  Groups of a multiple of 128 take them as
// they are (instruction j contracts the k = 32 g + 8 j + e of the step, all of one group);
// smaller groups have the four dwords of the four lane groups transposed (two
// v_permlane32_swap, two v_permlane16_swap), after which instruction j holds 32 consecutive k.
//
// f32 activations: int4_split_kernel writes each row as three f16 rows, h1 + h2 2^-11 + h3 2^-22
// of x / 2^e with 2^e from the row's largest magnitude.  Each part rounds to 11 bits what the
// one before left, 33 bits in all, more than the 24 of x; an element 2^29 below the row's
// largest still has its full precision.  The parts are rows of the same product.
#include "kernel_manager.h"
#include "serving.h"
#include "serving_device.h"

#include <algorithm>

namespace es
{

namespace
{

struct int4_dev_t {
    uint8_t const* w;
    void const*    scales;
    uint8_t const* zeros;
    _Float16 const* x;       // rows of f16
    int const*     x_exp;  // per token, f32 activations only: x is the parts' sum times 2^this
    void*          y;
    uint64_t       n, k;
    uint64_t       w_stride, scale_stride, x_stride, y_stride;
    uint32_t       group_magic;  // ceil(2^32 / (group / 32))
    uint32_t       m;            // tokens
    uint32_t       tokens_per_chunk;
};

template <typename T>
__device__ inline float scale_at(int4_dev_t const& a, uint64_t at)
{
    return float(static_cast<T const*>(a.scales)[at]);
}

// eight nibbles as (q - z) in the order 0 4 1 5 2 6 3 7; zz = (1024 + z, 1024 + z)
__device__ inline half8_t unpack(uint32_t w, half2_t zz)
{
    union {
        uint32_t u[4];
        half2_t  p[4];
        half8_t  v;
    } r;
#pragma unroll
    for (int i = 0; i != 4; ++i) {
        r.u[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
        r.p[i] = r.p[i] - zz;
    }
    return r.v;
}

__device__ inline half8_t in_nibble_order(u32x4_t x)
{
    union {
        uint32_t u[4];
        half8_t  v;
    } r;
    r.u[0] = __builtin_amdgcn_perm(x[2], x[0], 0x05040100u);
    r.u[1] = __builtin_amdgcn_perm(x[2], x[0], 0x07060302u);
    r.u[2] = __builtin_amdgcn_perm(x[3], x[1], 0x05040100u);
    r.u[3] = __builtin_amdgcn_perm(x[3], x[1], 0x07060302u);
    return r.v;
}

__device__ inline u32x4_t transpose_groups(u32x4_t v)
{
    auto const a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
    auto const b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    auto const c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto const d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4_t{c[0], c[1], d[0], d[1]};
}

// T: dtype of scales and y; PARTS: rows of x per token; MT: 16-row tiles of x; WK: wavefronts;
// WIDE: groups are multiples of 128
template <typename T, int PARTS, int MT, int WK, bool WIDE>
__global__ __launch_bounds__(64 * WK) void int4_kernel(int4_dev_t a)
{
    __shared__ float sums[WK][MT * 16][17];
    int const lane = int(threadIdx.x) & 63;
    int const w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    int const g = lane >> 4, c = lane & 15;
    uint64_t const n0 = uint64_t(blockIdx.x) * 16;
    uint64_t const n = min(n0 + uint64_t(c), a.n - 1);
    uint32_t const token0 = blockIdx.y * a.tokens_per_chunk;
    uint32_t const rows = min(a.m - token0, a.tokens_per_chunk) * PARTS;
    _Float16 const* const x0 = a.x + uint64_t(token0) * PARTS * a.x_stride;
    uint8_t const* const  wrow = a.w + n * a.w_stride + uint64_t(g) * 16;
    int const steps = int((a.k + 127) / 128);

    float4_t acc[MT];
#pragma unroll
    for (int t = 0; t != MT; ++t) acc[t] = float4_t{0, 0, 0, 0};

    constexpr int U = MT == 1 ? 4 : MT == 2 ? 2 : 1;  // steps in flight
    for (int st0 = w; st0 < steps; st0 += WK * U) {
        u32x4_t wv[U];
        u32x4_t xv[U][4][MT];
        float   sc[U][WIDE ? 1 : 4];
        half2_t zz[U][WIDE ? 1 : 4];
#pragma unroll
        for (int u = 0; u != U; ++u) {
            int const st = st0 + u * WK;
            bool const in = uint64_t(st) * 128 + uint64_t(g) * 32 < a.k;
            // a lane without k reads nothing; its x is zero
            wv[u] = in ? *reinterpret_cast<u32x4_t const*>(wrow + uint64_t(st) * 64) : u32x4_t{};
#pragma unroll
            for (int j = 0; j != (WIDE ? 1 : 4); ++j) {
                uint32_t const blk = uint32_t(st) * 4 + uint32_t(j);
                bool const     live = uint64_t(blk) * 32 < a.k;
                uint64_t const at = n * a.scale_stride +
                                    uint64_t(live ? __umulhi(blk, a.group_magic) : 0);
                // groups of 32 have a magic of 2^32, which 32 bits do not hold
                uint64_t const real = a.group_magic ? at : n * a.scale_stride + (live ? blk : 0);
                sc[u][j] = live ? scale_at<T>(a, real) : 0.0f;
                _Float16 const z = a.zeros ? _Float16(float(a.zeros[real])) : _Float16(8);
                zz[u][j] = half2_t{_Float16(1024), _Float16(1024)} + half2_t{z, z};
            }
        }
#pragma unroll
        for (int u = 0; u != U; ++u) {
            int const st = st0 + u * WK;
#pragma unroll
            for (int j = 0; j != 4; ++j) {
                uint64_t const k0 = uint64_t(st) * 128 +
                                    uint64_t(WIDE ? g * 32 + j * 8 : j * 32 + g * 8);
#pragma unroll
                for (int t = 0; t != MT; ++t) {
                    uint32_t const r = uint32_t(t * 16 + c);
                    xv[u][j][t] = r < rows && k0 < a.k
                                      ? *reinterpret_cast<u32x4_t const*>(x0 + r * a.x_stride + k0)
                                      : u32x4_t{};
                }
            }
        }
#pragma unroll
        for (int u = 0; u != U; ++u) {
            u32x4_t const wt = WIDE ? wv[u] : transpose_groups(wv[u]);
            float4_t      part[MT];
#pragma unroll
            for (int t = 0; t != MT; ++t) part[t] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j != 4; ++j) {
                half8_t const b = unpack(wt[j], zz[u][WIDE ? 0 : j]);
#pragma unroll
                for (int t = 0; t != MT; ++t) {
                    part[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(in_nibble_order(xv[u][j][t]), b,
                                                                    part[t], 0, 0, 0);
                    if (!WIDE || j == 3) {
                        acc[t] += part[t] * sc[u][WIDE ? 0 : j];
                        part[t] = float4_t{0, 0, 0, 0};
                    }
                }
            }
        }
    }
    // results: row 4 g + r, column c
#pragma unroll
    for (int t = 0; t != MT; ++t) {
#pragma unroll
        for (int r = 0; r != 4; ++r) sums[w][t * 16 + 4 * g + r][c] = acc[t][r];
    }
    __syncthreads();
    uint32_t const tokens = rows / PARTS;
    for (uint32_t i = threadIdx.x; i < tokens * 16; i += 64 * WK) {
        uint32_t const t = i / 16, col = i % 16;
        float          v = 0;
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p) {
            float s = 0;
#pragma unroll
            for (int q = 0; q != WK; ++q) s += sums[q][t * PARTS + p][col];
            v = v * 0x1p-11f + s;
        }
        if (PARTS > 1) v = __builtin_ldexpf(v, a.x_exp[token0 + t]);
        if (n0 + col < a.n) {
            static_cast<T*>(a.y)[uint64_t(token0 + t) * a.y_stride + n0 + col] = T(v);
        }
    }
}

// One workgroup per token: the row's largest finite magnitude, then the three parts.
__global__ __launch_bounds__(256) void int4_split_kernel(float const* x, uint64_t x_stride,
                                                         uint64_t k, _Float16* parts, int* exps)
{
    __shared__ float top[4];
    float const* const row = x + uint64_t(blockIdx.x) * x_stride;
    float              m = 0;
    for (uint64_t i = threadIdx.x * 4; i < k; i += 1024) {
        float4_t const v = *reinterpret_cast<float4_t const*>(row + i);
#pragma unroll
        for (int e = 0; e != 4; ++e) {
            float const f = __builtin_fabsf(v[e]);
            if (f <= 3.4028234664e38f) m = fmaxf(m, f);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    // m = f * 2^e with f in [0.5, 1): the largest element goes to [2^14, 2^15)
    int const e = m > 0 ? __builtin_amdgcn_frexp_expf(m) - 15 : 0;
    if (threadIdx.x == 0) exps[blockIdx.x] = e;
    _Float16* const out = parts + uint64_t(blockIdx.x) * 3 * k;
    for (uint64_t i = threadIdx.x * 4; i < k; i += 1024) {
        float4_t const v = *reinterpret_cast<float4_t const*>(row + i);
        half4_t        h[3];
#pragma unroll
        for (int q = 0; q != 4; ++q) {
            bool const fin = __builtin_fabsf(v[q]) <= 3.4028234664e38f;
            float      r = fin ? __builtin_ldexpf(v[q], -e) : v[q];
#pragma unroll
            for (int p = 0; p != 3; ++p) {
                h[p][q] = _Float16(r);
                r = fin ? (r - float(h[p][q])) * 2048.0f : 0.0f;
            }
        }
#pragma unroll
        for (int p = 0; p != 3; ++p) *reinterpret_cast<half4_t*>(out + p * k + i) = h[p];
    }
}

template <typename T, int PARTS, int MT, int WK>
void launch_group(int4_dev_t const& a, bool wide, hipStream_t stream)
{
    dim3 const grid(uint32_t((a.n + 15) / 16),
                    uint32_t((a.m + a.tokens_per_chunk - 1) / a.tokens_per_chunk));
    if (wide) {
        int4_kernel<T, PARTS, MT, WK, true><<<grid, 64 * WK, 0, stream>>>(a);
    } else {
        int4_kernel<T, PARTS, MT, WK, false><<<grid, 64 * WK, 0, stream>>>(a);
    }
}

template <typename T, int PARTS>
void launch_rows(int4_dev_t& a, bool wide, hipStream_t stream)
{
    uint64_t const rows = uint64_t(a.m) * PARTS;
    if (rows <= 16) {
        a.tokens_per_chunk = 16 / PARTS;
        launch_group<T, PARTS, 1, 8>(a, wide, stream);
    } else if (rows <= 32) {
        a.tokens_per_chunk = 32 / PARTS;
        launch_group<T, PARTS, 2, 8>(a, wide, stream);
    } else {
        a.tokens_per_chunk = 64 / PARTS;
        launch_group<T, PARTS, 4, 8>(a, wide, stream);
    }
}

}  // namespace

uint64_t int4_workspace(es_km_int4_weight_t const& w, uint64_t m)
{
    if (w.dtype != ES_KM_F32) return 0;
    return (m * 3 * w.k * 2 + 255) / 256 * 256 + m * 4;
}

void launch_int4_linear(int4_args_t const& g, void* workspace, hipStream_t stream)
{
    if (g.m == 0 || g.w.n == 0) return;
    int4_dev_t a;
    a.w = static_cast<uint8_t const*>(g.w.w);
    a.scales = g.w.scales;
    a.zeros = g.w.zeros;
    a.y = g.y;
    a.n = g.w.n;
    a.k = g.w.k;
    a.w_stride = g.w.w_stride;
    a.scale_stride = g.w.scale_stride;
    a.y_stride = g.y_stride;
    a.m = uint32_t(g.m);
    // blocks of 32 k to a group; k <= 2^20 keeps block * blocks below 2^32, where the product
    // with the magic number divides exactly
    uint64_t const blocks = std::min(g.w.group, g.w.k) / 32;
    a.group_magic = uint32_t((0x100000000ull + blocks - 1) / blocks);  // 0 for one block
    bool const wide = g.w.group % 128 == 0 || g.w.group >= g.w.k;
    if (g.w.dtype == ES_KM_F16) {
        a.x = static_cast<_Float16 const*>(g.x);
        a.x_stride = g.x_stride;
        a.x_exp = nullptr;
        launch_rows<_Float16, 1>(a, wide, stream);
    } else {
        _Float16* const parts = static_cast<_Float16*>(workspace);
        int* const      exps = reinterpret_cast<int*>(static_cast<char*>(workspace) +
                                                 (g.m * 3 * g.w.k * 2 + 255) / 256 * 256);
        int4_split_kernel<<<uint32_t(g.m), 256, 0, stream>>>(static_cast<float const*>(g.x),
                                                            g.x_stride, g.w.k, parts, exps);
        a.x = parts;
        a.x_stride = g.w.k;
        a.x_exp = exps;
        launch_rows<float, 3>(a, wide, stream);
    }
    hipError_t const err = hipGetLastError();
    if (err != hipSuccess) {
        throw km_error(km_status::device,
                       std::string("int4_linear launch: ") + hipGetErrorString(err));
    }
}

}  // namespace es
