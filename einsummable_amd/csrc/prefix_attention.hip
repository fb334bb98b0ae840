// es_km_prefix_attention: attention of a batch's new tokens over a paged cache, the positions
// that all sequences share read once for many rows.
//
// A row is a query: token i, head h.  The rows that read one key head (h' = h / G) are dealt
// with in tiles of 16, the keys in steps of KS (32 in f16, 16 in f32), one pass with a running
// maximum m and sum l per row:
//
//   S^T = K Q^T             rows are keys, columns are the tile's queries
//   m' = max(m, max_j S), p_j = 2^(S_j - m'), l' = l 2^(m - m') + sum_j p_j
//   O^T = O^T 2^(m - m') + V^T P^T
//
// Both products are taken transposed because of what the matrix instructions' registers hold:
// lane (g, c), g = lane / 16, c = lane % 16, gets column c of a result, so a query's maximum,
// sum and scaling live in the lanes of its own column, and the four (f32) or eight (f16) scores
// a lane gets are exactly the slice of P^T it has to supply to the second product -- for the
// keys 16 t + 4 g + r, which is then the order the lane reads the rows of V in (a sum over keys
// has no preferred order).  Neither K nor V nor P passes through LDS.  A lane's rows of V are
// consecutive elements of 4 or 8 keys; in f16 they are transposed in registers (v_perm_b32).
//
// A workgroup is four wavefronts that take the steps of its keys in turn and join their m, l
// and O at the end through LDS.  Work is cut over the keys: "prefix" workgroups take the rows
// of the whole batch against a cut of the shared positions, the others the rows of one sequence
// against a cut of its own positions.  How many cuts a sequence gets follows from the lengths
// in device memory (every workgroup adds them up for itself: the host knows only the number of
// sequences and tokens, and a captured graph must see the lengths of the day).  Each cut leaves
// O, m, l in fp32 in the workspace; attention_join_kernel adds them in a fixed order, so
// results do not depend on timing.  A row whose keys were all in one workgroup is stored
// directly.
#include "kernel_manager.h"
#include "serving.h"
#include "serving_device.h"

#include <algorithm>

namespace es
{

namespace
{

constexpr int ROWS = 16;     // queries per tile
constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;

struct attention_dev_t {
    char const* q;
    char*       out;
    char const *k, *v;
    int const * offsets, *lens, *table;
    uint64_t    table_stride;
    uint64_t    page_stride, token_stride, head_stride;  // elements
    uint64_t    q_stride, out_stride;
    uint64_t    n_pages;
    int         n_seqs, n_tokens, max_pages, page_size;
    int         h_kv, group, d;
    int         shared;
    float       scale;  // of the scores, times log2(e)
    int         prefix_tiles, prefix_splits, prefix_chunk;
    int         split_target;
    int         items;
    float*      part_o;     // [slot][key head][16][D]
    float*      part_ml;    // [slot][key head][16][2]
    int*        part_meta;  // [token][4]: slot of its tile's first cut, cuts, first token, -
};

constexpr float NEG_INF = -__builtin_huge_valf();

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ inline long long wave_sum(long long v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// The lane that owns a row's column also knows where the row ends up.
struct rows_t {
    int  token = -1;  // of this lane's column (-1: no such row)
    int  head = 0;
    int  limit = 0x7fffffff;  // its last position
    int  least = 0x7fffffff;  // the least limit of the tile's rows
};

template <typename T, int D>
struct core_t;

// ---- f16: steps of 32 keys, v_mfma_f32_16x16x32_f16
template <int D>
struct core_t<_Float16, D> {
    static constexpr int KS = 32;     // keys per step
    static constexpr int KL = 8;      // keys whose scores a lane holds
    static constexpr int DV = D / 16; // elements of a row of V per lane
    static constexpr int QC = D / 32;

    half8_t q[QC];
    half8_t k[2][QC];
    union vrow_t {
        uint32_t u[DV / 2];
        _Float16 h[DV];
    } v[KL];

    static __device__ int key_of(int j, int g) { return 16 * (j >> 2) + 4 * g + (j & 3); }

    __device__ void load_q(_Float16 const* row, int g, int d)
    {
#pragma unroll
        for (int c = 0; c != QC; ++c) {
            int const e = c * 32 + g * 8;
            q[c] = row && e < d ? *reinterpret_cast<half8_t const*>(row + e) : half8_t{};
        }
    }
    // element offsets of the two keys this lane loads of K, the eight of V
    __device__ void load(_Float16 const* kb, _Float16 const* vb, int64_t const* off, int c, int g,
                         int d)
    {
#pragma unroll
        for (int t = 0; t != 2; ++t) {
            int64_t const o = off[16 * t + c];
            _Float16 const* p = kb + (o < 0 ? 0 : o);
#pragma unroll
            for (int i = 0; i != QC; ++i) {
                int const e = i * 32 + g * 8;
                k[t][i] = e < d ? *reinterpret_cast<half8_t const*>(p + e) : half8_t{};
            }
        }
#pragma unroll
        for (int j = 0; j != KL; ++j) {
            int64_t const o = off[key_of(j, g)];
            _Float16 const* p = vb + (o < 0 ? 0 : o) + c * DV;
            constexpr int N = DV < 8 ? DV : 8;  // d is a multiple of 8
#pragma unroll
            for (int e = 0; e != DV; e += N) {
                if (c * DV + e < d) {
                    __builtin_memcpy(&v[j].h[e], __builtin_assume_aligned(p + e, N * 2), N * 2);
                } else {
#pragma unroll
                    for (int i = 0; i != N; ++i) v[j].h[e + i] = 0;
                }
            }
        }
    }
    __device__ void drop_key(int j)
    {
#pragma unroll
        for (int i = 0; i != DV / 2; ++i) v[j].u[i] = 0;
    }
    __device__ bool not_finite(int j) const
    {
        bool bad = false;
#pragma unroll
        for (int i = 0; i != DV / 2; ++i) {
            bad |= (v[j].u[i] & 0x7c00u) == 0x7c00u || (v[j].u[i] & 0x7c000000u) == 0x7c000000u;
        }
        return bad;
    }
    __device__ void scores(float* s) const
    {
#pragma unroll
        for (int t = 0; t != 2; ++t) {
            float4_t a = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i != QC; ++i) {
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][i], q[i], a, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r != 4; ++r) s[4 * t + r] = a[r];
        }
    }
    // o[t] += V^T P^T for the elements i * DV + t of the head, i the result's row.  With ONLY:
    // for the lanes with `take`, and with the keys whose bit is missing in `seen` as zeros.
    template <bool ONLY>
    __device__ void values(float const* p, float4_t* o, uint32_t seen, bool take) const
    {
        half8_t b;
#pragma unroll
        for (int j = 0; j != KL; ++j) b[j] = _Float16(p[j]);
#pragma unroll
        for (int t = 0; t != DV; ++t) {
            union {
                uint32_t u[4];
                half8_t  h;
            } a;
            uint32_t const sel = t & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
            for (int i = 0; i != 4; ++i) {
                uint32_t lo = v[2 * i].u[t / 2], hi = v[2 * i + 1].u[t / 2];
                if (ONLY) {
                    lo = seen >> (2 * i) & 1 ? lo : 0;
                    hi = seen >> (2 * i + 1) & 1 ? hi : 0;
                }
                a.u[i] = __builtin_amdgcn_perm(hi, lo, sel);
            }
            if (ONLY) {
                float4_t const x =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b, float4_t{0, 0, 0, 0}, 0, 0, 0);
                if (take) o[t] += x;
            } else {
                o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b, o[t], 0, 0, 0);
            }
        }
    }
};

// ---- f32: steps of 16 keys, v_mfma_f32_16x16x4_f32; chunk c of a row of K is taken in the order
// that lets a lane load 16 bytes: matrix instruction e contracts the elements 16 c + 4 g + e
template <int D>
struct core_t<float, D> {
    static constexpr int KS = 16;
    static constexpr int KL = 4;
    static constexpr int DV = D / 16;
    static constexpr int QC = D / 16;

    float4_t q[QC];
    float4_t k[QC];
    float    v[KL][DV];

    static __device__ int key_of(int j, int g) { return 4 * g + j; }

    __device__ void load_q(float const* row, int g, int d)
    {
#pragma unroll
        for (int c = 0; c != QC; ++c) {
            int const e = c * 16 + g * 4;
            q[c] = row && e < d ? *reinterpret_cast<float4_t const*>(row + e) : float4_t{};
        }
    }
    __device__ void load(float const* kb, float const* vb, int64_t const* off, int c, int g, int d)
    {
        int64_t const ok = off[c];
        float const*  p = kb + (ok < 0 ? 0 : ok);
#pragma unroll
        for (int i = 0; i != QC; ++i) {
            int const e = i * 16 + g * 4;
            k[i] = e < d ? *reinterpret_cast<float4_t const*>(p + e) : float4_t{};
        }
#pragma unroll
        for (int j = 0; j != KL; ++j) {
            int64_t const o = off[key_of(j, g)];
            float const*  pv = vb + (o < 0 ? 0 : o) + c * DV;
#pragma unroll
            for (int e = 0; e != DV; e += 4) {
                float4_t const x = c * DV + e < d ? *reinterpret_cast<float4_t const*>(pv + e)
                                                  : float4_t{};
#pragma unroll
                for (int i = 0; i != 4; ++i) v[j][e + i] = x[i];
            }
        }
    }
    __device__ void drop_key(int j)
    {
#pragma unroll
        for (int i = 0; i != DV; ++i) v[j][i] = 0;
    }
    __device__ bool not_finite(int j) const
    {
        bool bad = false;
#pragma unroll
        for (int i = 0; i != DV; ++i) {
            bad |= (__builtin_bit_cast(uint32_t, v[j][i]) & 0x7f800000u) == 0x7f800000u;
        }
        return bad;
    }
    __device__ void scores(float* s) const
    {
        float4_t a = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i != QC; ++i) {
#pragma unroll
            for (int e = 0; e != 4; ++e) {
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i][e], q[i][e], a, 0, 0, 0);
            }
        }
#pragma unroll
        for (int r = 0; r != 4; ++r) s[r] = a[r];
    }
    template <bool ONLY>
    __device__ void values(float const* p, float4_t* o, uint32_t seen, bool take) const
    {
#pragma unroll
        for (int t = 0; t != DV; ++t) {
            float4_t x = ONLY ? float4_t{0, 0, 0, 0} : o[t];
#pragma unroll
            for (int j = 0; j != KL; ++j) {
                float const e = !ONLY || (seen >> j & 1) ? v[j][t] : 0.0f;
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(e, p[j], x, 0, 0, 0);
            }
            if (!ONLY) {
                o[t] = x;
            } else if (take) {
                o[t] += x;
            }
        }
    }
};

template <typename T, int D>
struct shared_t {
    static constexpr int DJ = D < 128 ? D : 128;  // elements joined at a time
    int64_t off[WAVES][32];
    float   m[WAVES][ROWS], l[WAVES][ROWS];
    float   o[WAVES][ROWS][DJ + 4];
    long long total[WAVES];
    int     before[WAVES];
    int     found[4];  // sequence, item within it, first slot, cuts
    int     limit[ROWS];
};

// The keys lo <= position < hi of one table row against the tile's rows; steps w, w + WAVES, ...
template <typename T, int D>
__device__ void attend(attention_dev_t const& a, shared_t<T, D>& sh, rows_t const& row,
                       int const* __restrict__ table, int kvh, int lo, int hi, float4_t* o,
                       float& m, float& l)
{
    typedef core_t<T, D> core;
    constexpr int        KS = core::KS, KL = core::KL, DV = core::DV;
    int const            lane = int(threadIdx.x) & 63, w = int(threadIdx.x) >> 6;
    int const            g = lane >> 4, c = lane & 15;
    T const* const       kb = reinterpret_cast<T const*>(a.k) + uint64_t(kvh) * a.head_stride;
    T const* const       vb = reinterpret_cast<T const*>(a.v) + uint64_t(kvh) * a.head_stride;
    core                 x;
    x.load_q(row.token < 0 ? nullptr
                           : reinterpret_cast<T const*>(a.q) + uint64_t(row.token) * a.q_stride +
                                 uint64_t(row.head) * uint64_t(a.d),
             g, a.d);
    int64_t* const off = sh.off[w];
    for (int base = (lo / KS + w) * KS; base < hi; base += WAVES * KS) {
        // where the step's keys lie; -1: not among them, or no such page
        int     pos = base + (lane & (KS - 1));
        int64_t at = -1;
        if (pos >= lo && pos < hi) {
            int const pi = pos / a.page_size;
            int const page = table[pi];
            if (page >= 0 && uint64_t(page) < a.n_pages) {
                at = int64_t(uint64_t(page) * a.page_stride +
                             uint64_t(pos - pi * a.page_size) * a.token_stride);
            }
        }
        bool const holes = __any(at < 0);
        __builtin_amdgcn_wave_barrier();
        if (lane < KS) off[lane] = at;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        x.load(kb, vb, off, c, g, a.d);
        float s[KL];
        x.scores(s);
        bool const edge = holes || base + KS - 1 > row.least;
        uint32_t   masked = 0;
        if (edge) {
#pragma unroll
            for (int j = 0; j != KL; ++j) {
                int const  key = core::key_of(j, g);
                bool const hole = off[key] < 0;
                if (hole) x.drop_key(j);
                if (hole || base + key > row.limit) masked |= 1u << j;
            }
        }
        float top = NEG_INF;
#pragma unroll
        for (int j = 0; j != KL; ++j) {
            s[j] = masked >> j & 1 ? NEG_INF : s[j] * a.scale;
            top = fmaxf(top, s[j]);
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        float const mn = fmaxf(m, top);
        // nothing seen yet: any finite reference will do
        float const ref = mn == NEG_INF ? 0.0f : mn;
        float const fade = exp2_fast(m - ref);
        float       sum = 0;
#pragma unroll
        for (int j = 0; j != KL; ++j) {
            s[j] = exp2_fast(s[j] - ref);
            sum += s[j];
        }
        l = l * fade + sum;
        m = mn;
#pragma unroll
        for (int t = 0; t != DV; ++t) o[t] *= fade;
        // Zero times an infinity or NaN is no zero: where a row may not see a key whose values
        // are not finite, the rows are taken one by one, each with the keys it sees.
        bool careful = false;
        if (edge) {
            bool bad = false;
#pragma unroll
            for (int j = 0; j != KL; ++j) bad |= x.not_finite(j);
            careful = __any(bad);
        }
        if (!careful) {
            x.template values<false>(s, o, 0, true);
        } else {
            for (int r = 0; r != ROWS; ++r) {
                int const limit = __shfl(row.limit, r);
                uint32_t  seen = 0;
#pragma unroll
                for (int j = 0; j != KL; ++j) {
                    if (base + core::key_of(j, g) <= limit) seen |= 1u << j;
                }
                x.template values<true>(s, o, seen, c == r);
            }
        }
    }
    // the four lanes of a column hold sums over different keys
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
}

template <typename T, int D>
__global__ __launch_bounds__(THREADS) void attention_kernel(attention_dev_t a)
{
    __shared__ shared_t<T, D> sh;
    int const tid = int(threadIdx.x), lane = tid & 63, w = tid >> 6;
    int const c = lane & 15, g = lane >> 4;
    int const kvh = int(blockIdx.x) % a.h_kv;
    int const unit = int(blockIdx.x) / a.h_kv;
    int const prefix_units = a.prefix_tiles * a.prefix_splits;
    int const reach = a.max_pages * a.page_size;  // positions that a table row has pages for

    rows_t     row;
    int        lo, hi, slot;
    int const* table = a.table;
    bool       direct = false;
    if (unit < prefix_units) {
        int const tile = unit % a.prefix_tiles;
        int const split = unit / a.prefix_tiles;
        slot = unit;
        lo = split * a.prefix_chunk;
        hi = min(min(lo + a.prefix_chunk, a.shared), reach);
        int const r0 = tile * ROWS;
        int const t0 = r0 / a.group;
        int const t1 = min((r0 + ROWS - 1) / a.group, a.n_tokens - 1);
        if (tid < ROWS) sh.limit[tid] = -2;
        __syncthreads();
        // each thread puts down the positions of the tile's tokens in its sequences
        for (int s = tid; s < a.n_seqs; s += THREADS) {
            int const b = a.offsets[s], e = a.offsets[s + 1];
            if (b > t1 || e <= t0) continue;
            int const len = a.lens[s];
            for (int t = max(b, t0); t <= min(e - 1, t1); ++t) {
                sh.limit[t - t0] = max(len - (e - t), -1);
            }
        }
        __syncthreads();
        int const r = r0 + c;
        int const t = r / a.group;
        if (t <= t1 && sh.limit[t - t0] != -2) {
            row.token = t;
            row.head = kvh * a.group + r - t * a.group;
            row.limit = sh.limit[t - t0];
        }
    } else {
        // The cuts of all sequences, numbered through: tiles_s * splits_s each, where a cut holds
        // `chunk` steps.  A thread adds up a run of sequences.
        constexpr int KS = core_t<T, D>::KS;
        int const     item = unit - prefix_units;
        int const     run = (a.n_seqs + THREADS - 1) / THREADS;
        int const     s0 = min(tid * run, a.n_seqs), s1 = min(s0 + run, a.n_seqs);
        if (tid == 0) sh.found[0] = -1;
        long long total = 0;
        auto tiles_steps = [&](int s, int& tiles, int& steps) {
            int const b = max(a.offsets[s], 0), e = min(a.offsets[s + 1], a.n_tokens);
            int const len = min(a.lens[s], reach);
            tiles = e > b ? ((e - b) * a.group + ROWS - 1) / ROWS : 0;
            steps = len > a.shared ? (len + KS - 1) / KS - a.shared / KS : 0;
        };
        int tiles = 0, steps = 0;
        for (int s = s0; s < s1; ++s) {
            tiles_steps(s, tiles, steps);
            total += (long long)tiles * steps;
        }
        long long const ws = wave_sum(total);
        if (lane == 0) sh.total[w] = ws;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int i = 0; i != WAVES; ++i) all += sh.total[i];
        // at least one step per wavefront
        int chunk = 0x3fffffff;
        if (a.split_target > 0) {
            long long const per = (all + a.split_target - 1) / a.split_target;
            chunk = int(max((long long)WAVES, (per + WAVES - 1) / WAVES * WAVES));
        }
        int mine = 0;
        for (int s = s0; s < s1; ++s) {
            if (run > 1) tiles_steps(s, tiles, steps);
            mine += tiles * max(1, (steps + chunk - 1) / chunk);
        }
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            int const up = __shfl_up(incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 63) sh.before[w] = incl;
        __syncthreads();
        int start = incl - mine;
#pragma unroll
        for (int i = 0; i != WAVES; ++i) start += i < w ? sh.before[i] : 0;
        if (item >= start && item < start + mine) {
            for (int s = s0; s < s1; ++s) {
                if (run > 1) tiles_steps(s, tiles, steps);
                int const splits = max(1, (steps + chunk - 1) / chunk);
                if (item < start + tiles * splits) {
                    sh.found[0] = s;
                    sh.found[1] = item - start;
                    sh.found[2] = start;
                    sh.found[3] = splits;
                    break;
                }
                start += tiles * splits;
            }
        }
        __syncthreads();
        int const s = sh.found[0];
        if (s < 0) return;
        int const splits = sh.found[3];
        int const tile = sh.found[1] / splits, split = sh.found[1] - tile * splits;
        int const b = max(a.offsets[s], 0), e = min(a.offsets[s + 1], a.n_tokens);
        int const true_end = a.offsets[s + 1];
        int const full = a.lens[s];
        int const len = min(full, reach);
        slot = prefix_units + item;
        direct = splits == 1 && prefix_units == 0;
        table = a.table + uint64_t(s) * a.table_stride;
        int const r0 = tile * ROWS;
        int const r = r0 + c;
        int const t = b + r / a.group;
        if (t < e) {
            row.token = t;
            row.head = kvh * a.group + r % a.group;
            row.limit = max(full - (true_end - t), -1);
        }
        int const last = min(e - 1, b + (r0 + ROWS - 1) / a.group);
        if (split == 0 && kvh == 0) {
            int const first = b + r0 / a.group;
            if (first + tid <= last) {
                int* const meta = a.part_meta + 4 * (first + tid);
                meta[0] = slot - tile * splits;  // of the sequence's first tile
                meta[1] = direct ? 0 : splits;
                meta[2] = b;
            }
        }
        // positions of this cut, up to the last one that a row of the tile sees
        int const step0 = a.shared / KS + (splits == 1 ? 0 : split * chunk);
        lo = max(a.shared, step0 * KS);
        hi = splits == 1 ? len : min(len, (step0 + chunk) * KS);
        hi = min(hi, full - (true_end - last) + 1);
    }
    int least = row.limit;
#pragma unroll
    for (int i = 1; i != 16; i <<= 1) least = min(least, __shfl_xor(least, i));
    row.least = least;

    constexpr int DV = core_t<T, D>::DV;
    float4_t      o[DV];
#pragma unroll
    for (int t = 0; t != DV; ++t) o[t] = float4_t{0, 0, 0, 0};
    float m = NEG_INF, l = 0;
    if (lo < hi) attend<T, D>(a, sh, row, table, kvh, lo, hi, o, m, l);

    // join the wavefronts
    if (g == 0) {
        sh.m[w][c] = m;
        sh.l[w][c] = l;
    }
    __syncthreads();
    float top = NEG_INF;
#pragma unroll
    for (int i = 0; i != WAVES; ++i) top = fmaxf(top, sh.m[i][c]);
    float const mine = exp2_fast(m - (top == NEG_INF ? 0.0f : top));
    float*      part = a.part_o + (uint64_t(slot) * uint64_t(a.h_kv) + uint64_t(kvh)) * ROWS * D;
    constexpr int DJ = shared_t<T, D>::DJ;
    constexpr int TPR = THREADS / ROWS;  // threads that store a row
    constexpr int PER = DJ / TPR;
    int const     orow = tid / TPR, oe = tid % TPR * PER;
    // the row that this thread stores, from the lane that knows it
    int const   otoken = __shfl(row.token, orow);
    int const   ohead = __shfl(row.head, orow);
    float const otop = __shfl(top, orow);
    float       sum = 0;
#pragma unroll
    for (int i = 0; i != WAVES; ++i) {
        float const mi = sh.m[i][orow];
        sum += sh.l[i][orow] * exp2_fast(mi - (otop == NEG_INF ? 0.0f : otop));
    }
#pragma unroll
    for (int h = 0; h != D / DJ; ++h) {
        if (h) __syncthreads();
        // O^T: this lane has the elements (4 g + r) * DV + t of its column's row
#pragma unroll
        for (int r = 0; r != 4; ++r) {
            int const e = (4 * g + r) * DV;
            if (D > DJ && e / DJ != h) continue;
#pragma unroll
            for (int t = 0; t != DV; ++t) sh.o[w][c][e - h * DJ + t] = o[t][r] * mine;
        }
        __syncthreads();
        if (otoken >= 0) {
            float y[PER];
#pragma unroll
            for (int e = 0; e != PER; ++e) {
                y[e] = 0;
#pragma unroll
                for (int i = 0; i != WAVES; ++i) y[e] += sh.o[i][orow][oe + e];
            }
            if (direct) {
                T* const dst = reinterpret_cast<T*>(a.out) + uint64_t(otoken) * a.out_stride +
                               uint64_t(ohead) * uint64_t(a.d) + h * DJ + oe;
                float const inv = otop == NEG_INF ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int e = 0; e != PER; ++e) {
                    if (h * DJ + oe + e < a.d) dst[e] = T(otop == NEG_INF ? 0.0f : y[e] * inv);
                }
            } else {
                float* const dst = part + orow * D + h * DJ + oe;
#pragma unroll
                for (int e = 0; e != PER; e += 4) {
                    *reinterpret_cast<float4_t*>(dst + e) =
                        float4_t{y[e], y[e + 1], y[e + 2], y[e + 3]};
                }
            }
        }
    }
    if (!direct && otoken >= 0 && oe == 0) {
        float* const ml = a.part_ml +
                          ((uint64_t(slot) * uint64_t(a.h_kv) + uint64_t(kvh)) * ROWS + orow) * 2;
        ml[0] = otop;
        ml[1] = sum;
    }
}

// One wavefront per row: the maxima and sums of its cuts decide their weights, then the cuts'
// O are added in order.
template <typename T, int D>
__global__ __launch_bounds__(THREADS) void attention_join_kernel(attention_dev_t a)
{
    int const lane = int(threadIdx.x) & 63, w = int(threadIdx.x) >> 6;
    int const heads = a.h_kv * a.group;
    int const id = int(blockIdx.x) * WAVES + w;
    int const token = id / heads, head = id - token * heads;
    if (token >= a.n_tokens) return;
    if (token < a.offsets[0] || token >= a.offsets[a.n_seqs]) return;
    int const* const meta = a.part_meta + 4 * token;
    int const        splits = min(meta[1], a.items), b = meta[2];
    if (splits <= 0) return;
    int const kvh = head / a.group, hg = head - kvh * a.group;
    int const prow = token * a.group + hg, srow = (token - b) * a.group + hg;
    int const pslot = prow / ROWS;
    int const sslot = meta[0] + srow / ROWS * splits;
    int const parts = a.prefix_splits + splits;
    int const slots = a.prefix_tiles * a.prefix_splits + a.items;
    auto      place = [&](int i) -> int64_t {
        int const pre = i < a.prefix_splits;
        int const slot = pre ? pslot + i * a.prefix_tiles : sslot + i - a.prefix_splits;
        int const r = pre ? prow % ROWS : srow % ROWS;
        // stays inside the workspace whatever the device arrays held
        int const in = min(max(slot, 0), slots - 1);
        return (int64_t(in) * a.h_kv + kvh) * ROWS + r;
    };
    float top = NEG_INF;
    for (int i = lane; i < parts; i += 64) top = fmaxf(top, a.part_ml[place(i) * 2]);
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    constexpr int PER = D / 64;
    float         y[PER], sum = 0;
#pragma unroll
    for (int e = 0; e != PER; ++e) y[e] = 0;
    if (top != NEG_INF) {
        for (int i = 0; i != parts; ++i) {
            int64_t const at = place(i);
            float const   m = a.part_ml[at * 2];
            if (m == NEG_INF) continue;  // a cut without keys for this row
            float const f = exp2_fast(m - top);
            sum += a.part_ml[at * 2 + 1] * f;
#pragma unroll
            for (int e = 0; e != PER; ++e) y[e] += a.part_o[at * D + lane * PER + e] * f;
        }
    }
    T* const    dst = reinterpret_cast<T*>(a.out) + uint64_t(token) * a.out_stride +
                   uint64_t(head) * uint64_t(a.d) + lane * PER;
    float const inv = top == NEG_INF ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e != PER; ++e) {
        if (lane * PER + e < a.d) dst[e] = T(top == NEG_INF ? 0.0f : y[e] * inv);
    }
}

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }

template <typename T, int D>
void launch_dim(attention_dev_t const& a, hipStream_t stream)
{
    uint64_t const units = uint64_t(a.prefix_tiles) * a.prefix_splits + a.items;
    attention_kernel<T, D><<<uint32_t(units * a.h_kv), THREADS, 0, stream>>>(a);
    if (a.prefix_splits != 0 || a.split_target != 0) {
        uint64_t const rows = uint64_t(a.n_tokens) * a.h_kv * a.group;
        attention_join_kernel<T, D><<<uint32_t((rows + WAVES - 1) / WAVES), THREADS, 0, stream>>>(a);
    }
}

template <typename T>
void launch_type(attention_dev_t const& a, hipStream_t stream)
{
    int const D = padded_dim(a.d);
    if (D == 64) {
        launch_dim<T, 64>(a, stream);
    } else if (D == 128) {
        launch_dim<T, 128>(a, stream);
    } else {
        launch_dim<T, 256>(a, stream);
    }
}

}  // namespace

attention_plan_t plan_attention(es_km_kv_cache_t const& c, int n_seqs, int n_tokens,
                                uint64_t shared)
{
    attention_plan_t p;
    if (n_seqs == 0 || n_tokens == 0) return p;
    uint64_t const kv = uint64_t(c.n_kv_heads), group = uint64_t(c.n_heads / c.n_kv_heads);
    uint64_t const rows = uint64_t(n_tokens) * group;
    if (shared > 0) {
        uint64_t const tiles = (rows + ROWS - 1) / ROWS;
        uint64_t const want = (512 + tiles * kv - 1) / (tiles * kv);
        uint64_t const most = (shared + 255) / 256;
        uint64_t const splits = std::max<uint64_t>(1, std::min(want, most));
        uint64_t const chunk = ((shared + splits - 1) / splits + 31) / 32 * 32;
        p.prefix_tiles = uint32_t(tiles);
        p.prefix_chunk = uint32_t(chunk);
        p.prefix_splits = uint32_t((shared + chunk - 1) / chunk);
    }
    // sum over the sequences with tokens of ceil(tokens * group / ROWS)
    uint64_t const tiles = uint64_t(std::min(n_seqs, n_tokens)) + rows / ROWS;
    uint64_t const fill = 1024 / kv;
    uint64_t const target =
        tiles * kv >= 8192 ? 0 : std::max(fill > tiles ? fill - tiles : 0, (tiles + 1) / 2);
    p.split_target = uint32_t(target);
    p.items = uint32_t(tiles + target);
    uint64_t const slots = (uint64_t(p.prefix_tiles) * p.prefix_splits + p.items) * kv * ROWS;
    p.workspace_bytes = up256(slots * uint64_t(padded_dim(c.head_dim)) * 4) + up256(slots * 8) +
                        up256(uint64_t(n_tokens) * 16);
    return p;
}

void launch_attention(attention_args_t const& g, attention_plan_t const& p, void* workspace,
                      hipStream_t stream)
{
    attention_dev_t a;
    if (g.batch.n_tokens == 0 || g.batch.n_seqs == 0) return;
    a.q = static_cast<char const*>(g.q);
    a.out = static_cast<char*>(g.out);
    a.k = static_cast<char const*>(g.cache.k);
    a.v = static_cast<char const*>(g.cache.v);
    a.offsets = g.batch.offsets;
    a.lens = g.batch.lens;
    a.table = g.batch.page_table;
    a.table_stride = g.batch.table_stride;
    a.page_stride = g.cache.page_stride;
    a.token_stride = g.cache.token_stride;
    a.head_stride = g.cache.head_stride;
    a.q_stride = g.q_stride;
    a.out_stride = g.out_stride;
    a.n_pages = g.cache.n_pages;
    a.n_seqs = g.batch.n_seqs;
    a.n_tokens = g.batch.n_tokens;
    a.max_pages = g.batch.max_pages;
    a.page_size = g.cache.page_size;
    a.h_kv = g.cache.n_kv_heads;
    a.group = g.cache.n_heads / g.cache.n_kv_heads;
    a.d = g.cache.head_dim;
    a.shared = int(g.shared);
    a.scale = g.scale * 1.44269504088896340736f;
    a.prefix_tiles = int(p.prefix_tiles);
    a.prefix_splits = int(p.prefix_splits);
    a.prefix_chunk = int(p.prefix_chunk);
    a.split_target = int(p.split_target);
    a.items = int(p.items);
    uint64_t const slots = (uint64_t(p.prefix_tiles) * p.prefix_splits + p.items) *
                           uint64_t(a.h_kv) * ROWS;
    char* const    ws = static_cast<char*>(workspace);
    a.part_o = reinterpret_cast<float*>(ws);
    uint64_t const o_bytes = up256(slots * uint64_t(padded_dim(a.d)) * 4);
    a.part_ml = reinterpret_cast<float*>(ws + o_bytes);
    a.part_meta = reinterpret_cast<int*>(ws + o_bytes + up256(slots * 8));
    if (g.cache.dtype == ES_KM_F16) {
        launch_type<_Float16>(a, stream);
    } else {
        launch_type<float>(a, stream);
    }
    hipError_t const err = hipGetLastError();
    if (err != hipSuccess) {
        throw km_error(km_status::device,
                       std::string("prefix_attention launch: ") + hipGetErrorString(err));
    }
}

}  // namespace es
