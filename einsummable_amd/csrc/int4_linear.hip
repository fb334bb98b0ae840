// es_km_int4_linear: y[i, n] = sum over groups G of scale[n, G] sum_{k in G} (q[n,k] - z[n,G]) x[i,k]
// for a few tokens i.
//
// Bound by the weight's n * k / 2 bytes: each byte is read once per 64 rows of x.  A workgroup
// owns 16 or 32 columns n and all of k; its wavefronts take runs of 128-wide steps of k and join
// their fp32 sums through LDS in a fixed order.  The product X W^T goes through
// v_mfma_f32_16x16x32_f16 even for one token: a lane's share of the B operand is eight consecutive
// k of one n, one dword of the weight as it lies in memory, and the matrix unit does the
// multiplying and adding while the vector unit has only the unpacking left.  One token, 4096 x 11008:
// 8.5 us, 2.8 TB/s (a read reaches 5 to 6); f32, 5 tokens, 4096 x 32000: 22 us, 3.3 TB/s.
//
// Unpacking: (w & 0x000f000f) | 0x64006400 is the pair (1024 + q0, 1024 + q4) in f16; minus
// (1024 + z) it is exact.  (The bits w & 0x000f000f alone are q 2^-24, and the zero point can be a
// second product; but products of subnormal factors were summed less exactly, f32 results were off
// by 1e-5, and the time was the same.)  The nibbles come out in the order 0 4 1 5 2 6 3 7, so x is
// put in that order too.
// A lane holds 16 bytes, 32 consecutive k.  Groups of a multiple of 128 take them as they are
// (instruction j contracts the k = 32 g + 8 j + e of the step, all of one group); smaller groups
// have the four dwords of the four lane groups transposed (two v_permlane32_swap, two
// v_permlane16_swap), after which instruction j holds 32 consecutive k.
//
// Loads: in the products' layout sixteen neighbouring lanes belong to sixteen rows, and a load
// asks for 64 separate stretches of 16 bytes; what a load costs went by their number.  So four
// neighbouring lanes load 64 bytes of one row, and LDS brings the values to the lanes of the
// products (16 tokens, 11008 x 4096: 18.9 us without, 13.2 us with it).  Scales of up to four
// steps come in one load, a step per lane group.
//
// Few rows of x: the rows of the 16-row tile are independent, so any row may stand in those that
// hold no token.  With up to four (eight) rows, the four (two) lanes of one row load the
// fragments of one (two) of the step's instructions each and pass them on within the quad.
//
// f32 activations: int4_split_kernel writes each row as three f16 rows, h1 + h2 2^-11 + h3 2^-22
// of x / 2^e with 2^e from the row's largest magnitude.  Each part rounds to 11 bits what the
// one before left, 33 bits in all, more than the 24 of x; an element 2^29 below the row's
// largest still has its full precision.  The parts are rows of the same product.
#include "kernel_manager.h"
#include "serving.h"
#include "serving_device.h"

#include <algorithm>
#include <type_traits>

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
    uint32_t       group_magic;  // number of a group from a count of steps or blocks
    uint32_t       m;            // tokens
    uint32_t       tokens_per_chunk;
};

// eight nibbles as q - z in the order 0 4 1 5 2 6 3 7; zz = (1024 + z, 1024 + z)
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

__device__ inline u32x4_t in_nibble_order(u32x4_t x)
{
    return u32x4_t{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u),
                   __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                   __builtin_amdgcn_perm(x[3], x[1], 0x05040100u),
                   __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}

// each lane's x from lane QUAD >> (2 * its place) & 3 of its quad
template <int QUAD>
__device__ inline u32x4_t from_quad(u32x4_t x)
{
    u32x4_t r;
#pragma unroll
    for (int i = 0; i != 4; ++i) {
        r[i] = uint32_t(__builtin_amdgcn_mov_dpp(int(x[i]), QUAD, 0xf, 0xf, true));
    }
    return r;
}

__device__ inline u32x4_t transpose_groups(u32x4_t v)
{
    auto const a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
    auto const b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    auto const c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto const d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4_t{c[0], c[1], d[0], d[1]};
}

// From one value per lane group (g = lane / 16) for each of U steps: step u's for all lane groups.
// U = 4: group g holds step g's; U = 2: step g % 2's; U = 1: all the same.
template <int U>
__device__ inline void spread(uint32_t v, uint32_t* r)
{
    if constexpr (U == 1) {
        r[0] = v;
    } else if constexpr (U == 2) {
        auto const a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        r[0] = a[0];
        r[1] = a[1];
    } else {
        auto const     a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        uint32_t const lo = a[0], hi = a[1];
        auto const     b = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
        auto const     c = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
        r[0] = b[0];
        r[1] = b[1];
        r[2] = c[0];
        r[3] = c[1];
    }
}

// The zero points of weights without any.
__device__ __align__(16) uint8_t const int4_eights[16] = {8, 8, 8, 8, 8, 8, 8, 8,
                                                          8, 8, 8, 8, 8, 8, 8, 8};

// The scales and zero points of a step of 128 k, as they lie in memory until they are used (taking
// them apart earlier would wait for them).  GROUPS: groups to a step, 1 also for groups of several
// steps; 0: groups that do not divide or make up steps, looked up per 32 k.
template <typename T, int GROUPS>
struct step_scales_t {
    static constexpr int N = GROUPS ? 1 : 4;            // loads for a step
    static constexpr int S = GROUPS ? GROUPS : 1;       // scales to a load
    static constexpr int W = (S * int(sizeof(T)) + 3) / 4;  // words to a load
    uint32_t scales[N][W];
    uint32_t zeros[N];

    // the i-th load, from a row's scales and zero points; no alignment but the elements'
    __device__ void load(int i, T const* s, uint8_t const* z, uint32_t at, uint32_t z_at)
    {
        scales[i][W - 1] = 0;
        __builtin_memcpy(scales[i], s + at, S * sizeof(T));
        zeros[i] = 0;
        __builtin_memcpy(&zeros[i], z + z_at, S);
    }
    // of group j of the step
    __device__ float scale(int j) const
    {
        if constexpr (sizeof(T) == 4) {
            return __builtin_bit_cast(float, GROUPS ? scales[0][j % W] : scales[j % N][0]);
        } else {
            uint32_t const u = GROUPS ? scales[0][j / 2 % W] >> (16 * (j % 2)) : scales[j % N][0];
            return float(__builtin_bit_cast(_Float16, uint16_t(u)));
        }
    }
    __device__ uint32_t zero(int j) const
    {
        return GROUPS ? zeros[0] >> (8 * j) & 0xff : zeros[j % N];
    }
};

// A wavefront's LDS.
template <int MT, int NT, int XL>
struct int4_wave_t {
    union {
        struct {
            u32x4_t w[128];
            u32x4_t x[XL == 4 ? 256 : 1];
        };
        float sums[MT * 4 * XL][NT * 16 + 1];
    };
};

// Where 16 bytes of row r of x lie among the row's: eight lanes that write two rows each and
// sixteen that read sixteen rows all meet different banks.
__device__ inline int x_swizzle(int r) { return (r & 1) * 8 + (r & 2) * 2 + r / 4; }

__device__ inline void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// T: dtype of scales and y; PARTS: rows of x per token; MT: 16-row tiles of x; NT: 16-column tiles
// of a workgroup; XL: loads for a step of a row tile (1: up to four rows, 2: eight, 4: sixteen);
// WK: wavefronts; GROUPS as above
template <typename T, int PARTS, int MT, int NT, int XL, int WK, int GROUPS>
__global__ __launch_bounds__(64 * WK, WK == 16 || (MT * NT < 4 && GROUPS) ? 4 : 2) void int4_kernel(int4_dev_t a)
{
    constexpr int  SPREAD = 4 / XL;  // rows of the matrix product per row of x
    constexpr bool WIDE = GROUPS == 1;
    __shared__ int4_wave_t<MT, NT, XL> lds[WK];
    int const lane = int(threadIdx.x) & 63;
    int const w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    int const g = lane >> 4, c = lane & 15;  // as operands and results of products
    int const q = lane >> 3, e = lane & 7;   // as loaded: eight lanes read 128 bytes of a row
    uint64_t const n0 = uint64_t(blockIdx.x) * (16 * NT);
    uint32_t const token0 = blockIdx.y * a.tokens_per_chunk;
    uint32_t const rows = min(a.m - token0, a.tokens_per_chunk) * PARTS;
    uint32_t const k = uint32_t(a.k);

    uint8_t const* wrow[NT][2];  // rows q and q + 8 of the tile
    T const*       srow[NT];
    uint8_t const* zrow[NT];
#pragma unroll
    for (int i = 0; i != NT; ++i) {
#pragma unroll
        for (int r = 0; r != 2; ++r) {
            wrow[i][r] = a.w + min(n0 + uint64_t(i * 16 + r * 8 + q), a.n - 1) * a.w_stride;
        }
        uint64_t const n = min(n0 + uint64_t(i * 16 + c), a.n - 1);
        srow[i] = static_cast<T const*>(a.scales) + n * a.scale_stride;
        zrow[i] = a.zeros ? a.zeros + n * a.scale_stride : int4_eights;
    }
    constexpr int   XR = XL == 4 ? 2 : 1;
    _Float16 const* xrow[MT][XR];
#pragma unroll
    for (int t = 0; t != MT; ++t) {
#pragma unroll
        for (int i = 0; i != XR; ++i) {
            uint32_t const r = min(uint32_t(t * 16 + (XL == 4 ? i * 8 + q : c / SPREAD)), rows - 1);
            xrow[t][i] = a.x + (uint64_t(token0) * PARTS + r) * a.x_stride;
        }
    }
    // k within a step of what load l brings this lane
    auto k_of = [&](int l) {
        if (XL == 4) return uint32_t(l / 2 * 64 + e * 8);
        int const j = l * SPREAD + c % SPREAD;
        return uint32_t(WIDE ? g * 32 + j * 8 : j * 32 + g * 8);
    };

    int4_wave_t<MT, NT, XL>& mine = lds[w];
    float4_t                 acc[MT][NT];
#pragma unroll
    for (int t = 0; t != MT; ++t) {
#pragma unroll
        for (int i = 0; i != NT; ++i) acc[t][i] = float4_t{0, 0, 0, 0};
    }

    uint32_t const z_mask = a.zeros ? ~0u : 0;
    int const      steps = int((k + 127) / 128), whole = int(k / 128);
    // two steps are 128 bytes of a row
    int const pairs = (steps + 1) / 2;
    int const begin = pairs * w / WK * 2, end = min(steps, pairs * (w + 1) / WK * 2);

    // Up to U steps from st0 on, steps at stop and behind it left out.  PARTIAL: the row ends within
    // the step.
    auto batch = [&](int st0, int stop, auto uu, auto partial) {
        constexpr int  U = decltype(uu)::value;
        constexpr bool PARTIAL = decltype(partial)::value;
        // a partial step need not have all its groups
        constexpr int       G = PARTIAL && GROUPS > 1 ? 0 : GROUPS;
        constexpr int       PIECES = step_scales_t<T, G>::N;
        u32x4_t             wv[U][NT];
        // more than a tile of x at a time leaves no registers for the x of several steps
        constexpr int XU = MT == 1 ? U : 1;
        u32x4_t       xv[XU][MT][XL];
        step_scales_t<T, G> sc[NT];
        // Loads without a condition, all on their way before the first is waited for: steps behind
        // the last and k behind the row stand for what is there.
#pragma unroll
        for (int u = 0; u != U; u += 2) {
            uint32_t const st = uint32_t(min(st0 + u + e / 4, stop - 1));
            uint32_t const in = uint32_t(e % 4) * 16;
            uint32_t const at = st * 64 + (PARTIAL && st * 128 + in * 2 >= k ? 0 : in);
#pragma unroll
            for (int r = 0; r != 2; ++r) {
#pragma unroll
                for (int i = 0; i != NT; ++i) {
                    wv[u + r][i] = *reinterpret_cast<u32x4_t const*>(wrow[i][r] + at);
                }
            }
        }
        // one load for all U steps, a step per lane group
        uint32_t const st_g = uint32_t(min(st0 + g % U, stop - 1));
#pragma unroll
        for (int j = 0; j != PIECES; ++j) {
            uint32_t at = st_g * G;
            if (G <= 1) {
                uint32_t const at_k = G ? st_g : min(st_g * 4 + uint32_t(j), k / 32 - 1);
                at = a.group_magic ? __umulhi(at_k, a.group_magic) : at_k;
            }
#pragma unroll
            for (int i = 0; i != NT; ++i) sc[i].load(j, srow[i], zrow[i], at, at & z_mask);
        }
        auto load_x = [&](int u) {
            uint32_t const k0 = uint32_t(min(st0 + u, stop - 1)) * 128;
#pragma unroll
            for (int t = 0; t != MT; ++t) {
#pragma unroll
                for (int l = 0; l != XL; ++l) {
                    uint32_t at = k0 + k_of(l);
                    if (PARTIAL) at = at < k ? at : 0;
                    xv[u % XU][t][l] =
                        *reinterpret_cast<u32x4_t const*>(xrow[t][l % XR] + at);
                }
            }
        };
#pragma unroll
        for (int u = 0; u != XU; ++u) load_x(u);
        __builtin_amdgcn_sched_barrier(0);
        step_scales_t<T, G> su[U][NT];
#pragma unroll
        for (int i = 0; i != NT; ++i) {
#pragma unroll
            for (int j = 0; j != PIECES; ++j) {
                uint32_t r[U];
#pragma unroll
                for (int v = 0; v != step_scales_t<T, G>::W; ++v) {
                    spread<U>(sc[i].scales[j][v], r);
#pragma unroll
                    for (int u = 0; u != U; ++u) su[u][i].scales[j][v] = r[u];
                }
                spread<U>(sc[i].zeros[j], r);
#pragma unroll
                for (int u = 0; u != U; ++u) su[u][i].zeros[j] = r[u];
            }
        }
#pragma unroll
        for (int u = 0; u != U; ++u) {
            uint32_t const st = uint32_t(st0 + u);
            if (int(st) >= stop) break;
            if (XU == 1 && u > 0) load_x(u);
            if (PARTIAL) {
#pragma unroll
                for (int l = 0; l != XL; ++l) {
                    bool const in = st * 128 + k_of(l) < k;
#pragma unroll
                    for (int t = 0; t != MT; ++t) {
                        xv[u % XU][t][l] = in ? xv[u % XU][t][l] : u32x4_t{0, 0, 0, 0};
                    }
                }
            }
            // from the lanes that loaded to the lanes of the products, through LDS; the order of a
            // row's 16 bytes there keeps either side free of bank conflicts
            u32x4_t xs[MT][XL];
#pragma unroll
            for (int t = 0; t != MT; ++t) {
#pragma unroll
                for (int l = 0; l != XL; ++l) xs[t][l] = in_nibble_order(xv[u % XU][t][l]);
                if constexpr (XL == 4) {
                    wave_sync();
#pragma unroll
                    for (int l = 0; l != 4; ++l) {
                        int const r = l % 2 * 8 + q;
                        mine.x[r * 16 + ((l / 2 * 8 + e) ^ x_swizzle(r))] = xs[t][l];
                    }
                    wave_sync();
#pragma unroll
                    for (int j = 0; j != 4; ++j) {
                        int const s = WIDE ? g * 4 + j : j * 4 + g;
                        xs[t][j] = mine.x[c * 16 + (s ^ x_swizzle(c))];
                    }
                }
            }
            if (u % 2 == 0) {
#pragma unroll
                for (int i = 0; i != NT; ++i) {
                    wave_sync();
#pragma unroll
                    for (int r = 0; r != 2; ++r) {
                        mine.w[(r * 8 + q) * 8 + (e ^ (r * 4 + q / 2))] = wv[u + r][i];
                    }
                    wave_sync();
#pragma unroll
                    for (int r = 0; r != 2; ++r) {
                        wv[u + r][i] = mine.w[c * 8 + ((r * 4 + g) ^ c / 2)];
                    }
                }
            }
            u32x4_t wt[NT];
#pragma unroll
            for (int i = 0; i != NT; ++i) {
                wt[i] = WIDE ? wv[u][i] : transpose_groups(wv[u][i]);
            }
            float4_t part[MT][NT];
            half2_t  z[NT];
            auto const product = [&](auto jj) {
                constexpr int j = decltype(jj)::value;
                // the first and the last product of a group (of what a step has of it)
                constexpr int EACH = G ? 4 / (G ? G : 1) : 1;
                constexpr bool first = j % EACH == 0, last = j % EACH == EACH - 1;
                // groups that the row does not have
                if (PARTIAL && !WIDE && st * 128 + uint32_t(j) * 32 >= k) return;
#pragma unroll
                for (int i = 0; i != NT; ++i) {
                    if (first) {
                        uint32_t const zero = su[u][i].zero(j / EACH) * 0x10001u + 0x64006400u;
                        z[i] = __builtin_bit_cast(half2_t, zero);
                    }
                    half8_t const q = unpack(wt[i][j], z[i]);
#pragma unroll
                    for (int t = 0; t != MT; ++t) {
                        u32x4_t f = xs[t][j / SPREAD];
                        if constexpr (XL == 1) f = from_quad<j * 0x55>(f);
                        if constexpr (XL == 2) f = from_quad<j % 2 ? 0xf5 : 0xa0>(f);
                        half8_t const x = __builtin_bit_cast(half8_t, f);
                        if (first) part[t][i] = float4_t{0, 0, 0, 0};
                        part[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q, part[t][i], 0, 0,
                                                                           0);
                        if (last) {
                            float const s = su[u][i].scale(j / EACH);
#pragma unroll
                            for (int r = 0; r < 4; r += SPREAD) acc[t][i][r] += part[t][i][r] * s;
                        }
                    }
                }
            };
            product(std::integral_constant<int, 0>{});
            product(std::integral_constant<int, 1>{});
            product(std::integral_constant<int, 2>{});
            product(std::integral_constant<int, 3>{});
        }
    };
    constexpr int U = MT * XL * NT <= 2 ? 4 : 2;  // steps in flight
    for (int st = begin; st < min(end, whole); st += U) {
        batch(st, min(end, whole), std::integral_constant<int, U>{}, std::false_type{});
    }
    if (begin < end && end > whole) {
        batch(whole, end, std::integral_constant<int, 2>{}, std::true_type{});
    }
    wave_sync();
    // results: row 4 g + r, column c
#pragma unroll
    for (int t = 0; t != MT; ++t) {
#pragma unroll
        for (int i = 0; i != NT; ++i) {
#pragma unroll
            for (int r = 0; r < 4; r += SPREAD) {
                mine.sums[(t * 16 + 4 * g + r) / SPREAD][i * 16 + c] = acc[t][i][r];
            }
        }
    }
    __syncthreads();
    uint32_t const tokens = rows / PARTS;
    for (uint32_t i = threadIdx.x; i < tokens * (16 * NT); i += 64 * WK) {
        uint32_t const t = i / (16 * NT), col = i % (16 * NT);
        float          v = 0;
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p) {
            float s = 0;
#pragma unroll
            for (int q = 0; q != WK; ++q) s += lds[q].sums[t * PARTS + p][col];
            v = v * 0x1p-11f + s;
        }
        if (PARTS > 1) v = __builtin_ldexpf(v, a.x_exp[token0 + t]);
        if (n0 + col < a.n) {
            static_cast<T*>(a.y)[uint64_t(token0 + t) * a.y_stride + n0 + col] = T(v);
        }
    }
}

// One workgroup per token: the row's largest finite magnitude, then the three parts.
__global__ __launch_bounds__(1024) void int4_split_kernel(float const* x, uint64_t x_stride,
                                                          uint64_t k, _Float16* parts, int* exps)
{
    __shared__ float top[16];
    float const* const row = x + uint64_t(blockIdx.x) * x_stride;
    constexpr float    HUGEST = 3.4028234664e38f;
    auto const         at = [&](uint64_t i) { return *reinterpret_cast<float4_t const*>(row + i); };
    // rows of up to 4096 are read once
    float4_t const zero = {0, 0, 0, 0};
    float4_t const mine = threadIdx.x * 4 < k ? at(threadIdx.x * 4) : zero;
    float4_t       v = mine;
    float          m = 0;
    for (uint64_t i = threadIdx.x * 4;;) {
#pragma unroll
        for (int e = 0; e != 4; ++e) {
            float const f = __builtin_fabsf(v[e]);
            m = fmaxf(m, f <= HUGEST ? f : 0.0f);
        }
        i += 4096;
        if (i >= k) break;
        v = at(i);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i != 16; ++i) m = fmaxf(m, top[i]);
    // m = f * 2^e with f in [0.5, 1): the largest element goes to [2^14, 2^15)
    int const e = m > 0 ? __builtin_amdgcn_frexp_expf(m) - 15 : 0;
    if (threadIdx.x == 0) exps[blockIdx.x] = e;
    _Float16* const out = parts + uint64_t(blockIdx.x) * 3 * k;
    for (uint64_t i = threadIdx.x * 4; i < k; i += 4096) {
        v = i < 4096 ? mine : at(i);
        half4_t h[3];
#pragma unroll
        for (int q = 0; q != 4; ++q) {
            bool const fin = __builtin_fabsf(v[q]) <= HUGEST;
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

template <typename T, int PARTS, int MT, int NT, int XL, int WK>
void launch_groups(int4_dev_t a, uint64_t group, hipStream_t stream)
{
    dim3 const grid(uint32_t((a.n + 16 * NT - 1) / (16 * NT)),
                    uint32_t((a.m + a.tokens_per_chunk - 1) / a.tokens_per_chunk));
    // A group's number is its 32 k's or its step's number divided by their count in a group, as a
    // product with ceil(2^32 / count); 0 stands for a count of one.  Exact, as number * count is
    // below 2^32 (k <= 2^20).
    auto const magic = [&](uint64_t per) {
        uint64_t const count = std::min(group, (a.k + per - 1) / per * per) / per;
        a.group_magic = uint32_t((0x100000000ull + count - 1) / count);
    };
    if (group % 128 == 0 || group >= a.k) {
        group = (group + 127) / 128 * 128;
        magic(128);
        int4_kernel<T, PARTS, MT, NT, XL, WK, 1><<<grid, 64 * WK, 0, stream>>>(a);
        return;
    }
    magic(32);
    if (group == 32) {
        int4_kernel<T, PARTS, MT, NT, XL, WK, 4><<<grid, 64 * WK, 0, stream>>>(a);
    } else if (group == 64) {
        int4_kernel<T, PARTS, MT, NT, XL, WK, 2><<<grid, 64 * WK, 0, stream>>>(a);
    } else {
        int4_kernel<T, PARTS, MT, NT, XL, WK, 0><<<grid, 64 * WK, 0, stream>>>(a);
    }
}

template <typename T, int PARTS, int MT, int XL>
void launch_columns(int4_dev_t const& a, uint64_t group, hipStream_t stream)
{
    uint64_t const tiles = (a.n + 15) / 16 * ((a.m + a.tokens_per_chunk - 1) / a.tokens_per_chunk);
    // Up to a tile per compute unit, sixteen wavefronts share its k (16 tokens, 11008 x 4096: 13.1 us
    // with either count; one token, 4096 x 4096: 4.9 us, 5.1 with eight).  From four tiles per
    // compute unit on, two tiles share their x (f32, 5 tokens, 4096 x 32000: 26 us, 40 us one by
    // one; one token, 4096 x 11008, 2.7 tiles: 8.4 us one by one, 8.8 us in twos).
    if (tiles >= 1024) {
        launch_groups<T, PARTS, MT, 2, XL, 8>(a, group, stream);
        return;
    }
    // (64 rows of x leave sixteen wavefronts no registers)
    if constexpr (MT <= 2) {
        if (tiles <= 256) {
            launch_groups<T, PARTS, MT, 1, XL, 16>(a, group, stream);
            return;
        }
    }
    launch_groups<T, PARTS, MT, 1, XL, 8>(a, group, stream);
}

template <typename T, int PARTS>
void launch_rows(int4_dev_t& a, uint64_t group, hipStream_t stream)
{
    uint64_t const rows = uint64_t(a.m) * PARTS;
    a.tokens_per_chunk = (rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64) /
                         PARTS;
    if (rows <= 4) {
        launch_columns<T, PARTS, 1, 1>(a, group, stream);
    } else if (rows <= 8) {
        launch_columns<T, PARTS, 1, 2>(a, group, stream);
    } else if (rows <= 16) {
        launch_columns<T, PARTS, 1, 4>(a, group, stream);
    } else if (rows <= 32) {
        launch_columns<T, PARTS, 2, 4>(a, group, stream);
    } else {
        launch_columns<T, PARTS, 4, 4>(a, group, stream);
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
    if (g.w.dtype == ES_KM_F16) {
        a.x = static_cast<_Float16 const*>(g.x);
        a.x_stride = g.x_stride;
        a.x_exp = nullptr;
        launch_rows<_Float16, 1>(a, g.w.group, stream);
    } else {
        _Float16* const parts = static_cast<_Float16*>(workspace);
        int* const      exps = reinterpret_cast<int*>(static_cast<char*>(workspace) +
                                                 (g.m * 3 * g.w.k * 2 + 255) / 256 * 256);
        int4_split_kernel<<<uint32_t(g.m), 1024, 0, stream>>>(static_cast<float const*>(g.x),
                                                            g.x_stride, g.w.k, parts, exps);
        a.x = parts;
        a.x_stride = g.w.k;
        a.x_exp = exps;
        launch_rows<float, 3>(a, g.w.group, stream);
    }
    hipError_t const err = hipGetLastError();
    if (err != hipSuccess) {
        throw km_error(km_status::device,
                       std::string("int4_linear launch: ") + hipGetErrorString(err));
    }
}

}  // namespace es
