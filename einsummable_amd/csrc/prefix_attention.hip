// es_km_prefix_attention: attention of a batch's new tokens over a paged cache, the positions
// that all sequences share read once for many rows.
//
// A row is a query: token i, head h.  The rows that read one key head (h' = h / G) are dealt
// with in tiles of 16, the keys in steps of 16 or 32, one pass with a running
// maximum m and sum l per row:
//
//   S^T = K Q^T             rows are keys, columns are the tile's queries
//   m' = max(m, max_j S), p_j = 2^(S_j - m'), l' = l 2^(m - m') + sum_j p_j
//   O^T = O^T 2^(m - m') + V^T P^T
//
// Both products are taken transposed because of what the matrix instructions' registers hold:
// lane (g, c), g = lane / 16, c = lane % 16, gets column c of a result, so a query's maximum,
// sum and scaling live in the lanes of its own column, and the four scores a lane gets of
// sixteen keys are exactly the slice of P^T it has to supply to the second product -- for the
// keys 4 g + r, which is then the order the lane reads the rows of V in (a sum over keys has no
// preferred order).  P passes through no memory.
//
// Two kinds of workgroups.  attention_few_kernel, for decoding, bound by the bytes of K and V: tiles
// of 16 rows; the four wavefronts of a workgroup take the steps of its keys in turn, straight from
// global memory into registers (K and V are used once; in f16 a lane's four rows of V are transposed
// there, v_perm_b32), and join their m, l and O at the end through LDS.  125 MB in 32 us, 3.9 TB/s.
// attention_many_kernel, for the shared positions of a batch and for prompts, bound by the issue and
// latency of its steps: each wavefront has 16 or 32 rows of its own and all of them go through the
// same tiles of keys, staged in LDS.  30 GFLOP of prompts in 69 us, 0.44 PFLOP/s.
// attention_mixed_kernel has workgroups of both kinds.
//
// Work is cut over the keys: "prefix" workgroups take the rows of the whole batch against a cut
// of the shared positions, the others the rows of one sequence against a cut of its own
// positions.  How many cuts a sequence gets follows from the lengths in device memory (every
// workgroup adds them up for itself: the host knows only the number of sequences and tokens, and
// a captured graph must see the lengths of the day).  Each cut leaves O, m, l in fp32 in the
// workspace; attention_join_kernel adds them in a fixed order, so results do not depend on
// timing.  A row whose keys were all in one workgroup is stored directly.
#include "kernel_manager.h"
#include "serving.h"
#include "serving_device.h"

#include <algorithm>
#include <type_traits>

namespace es
{

namespace
{

constexpr int THREADS = 256;
constexpr int FEW = 16;
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
    float       scale;   // of the scores, times log2(e); positive
    float       q_sign;  // -1, 0 or 1, multiplied into q: the sign of the caller's scale
    uint32_t    page_magic, page_shift;
    int         prefix_tiles, prefix_splits, prefix_chunk, prefix_rows;
    int         shares;     // parts that the own positions of the whole batch are cut into
    int         grain;      // steps per unit of work of the few-row kernel
    int         own_slots, own_rows;
    int         parts;      // what this launch does: 1 prefix, 2 own positions, 3 both
    int         direct;     // there are no shared positions to join with
    float*      part_o;     // [row of a slot][D]: the prefix's slots, then the own ones
    float*      part_ml;    // [row of a slot][2]
    int4*       part_meta;  // [token * group + head of the group], see piece(); null: no join
    int64_t     own_base;   // rows before the own positions' slots
};

constexpr float NEG_INF = -__builtin_huge_valf();

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ inline bool finite(float x) { return x - x == 0.0f; }

// y, scaled by a weight that is positive but may have underflowed: infinities stay what they are.
__device__ inline float scaled(float y, float by) { return finite(y) ? y * by : y; }

// f16 products take a weight p as two numbers, the f16 next to p and the f16 next to what that
// leaves: 22 bits of it, where one f16 has 11 and cost results of f16 half a step of their own.  So
// that small weights have them too, weights are taken relative to 2^-WEIGHT_LIFT of their row's
// reference: what is lost of each is below 2^-32 of the largest.  It costs the kernel of many rows the
// second product's matrix instructions once more and about sixty others in a step of 32 keys
// (prompts 55 us with one f16, 69 us), the one of few rows, which waits for memory, nothing.
constexpr int WEIGHT_LIFT = 7;

__device__ inline void split_weights(float2_t p, half2_t& high, half2_t& low)
{
    high = __builtin_convertvector(p, half2_t);
    low = __builtin_convertvector(p - __builtin_convertvector(high, float2_t), half2_t);
}

// A number that is the same in all lanes, of which the compiler is not to make two loops.
__device__ inline int opaque(int v)
{
    asm volatile("" : "+s"(v));
    return v;
}

// Inclusive sums over the 64 lanes.
__device__ inline int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);  // row_bcast:31
    return v;
}

// The largest of 64 numbers that are not negative, in lane 63.
__device__ inline int wave_max(int v)
{
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true));
    return max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true));
}

// Maximum and sum over the four lanes that share a column (lane % 16).
__device__ inline float column_max(float x)
{
    uint32_t u = __builtin_bit_cast(uint32_t, x);
    auto     r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    // by way of variables: a bit cast of r[1] itself reads r[0]
    uint32_t lo = r[0], hi = r[1];
    u = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, lo),
                                           __builtin_bit_cast(float, hi)));
    r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    lo = r[0];
    hi = r[1];
    return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

__device__ inline float column_sum(float x)
{
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// pos / page_size, exact below 2^30 positions
__device__ inline int page_of(attention_dev_t const& a, int pos)
{
    return int((uint64_t(uint32_t(pos)) * a.page_magic) >> a.page_shift);
}

// Element offset of a position's entry for key head 0; -1: no such page.
__device__ inline int64_t entry_of(attention_dev_t const& a, int page, int row)
{
    if (page < 0 || uint64_t(page) >= a.n_pages) return -1;
    return int64_t(uint64_t(page) * a.page_stride + uint64_t(row) * a.token_stride);
}

// What a workgroup works at: the positions lo <= p < hi of a page table's row, and a tile of rows,
// which are either rows of the whole batch or of one sequence.
struct work_t {
    int        lo, hi;
    int const* table;
    int64_t    part;    // first row of its slot
    bool       direct;
    bool       whole;   // rows of the whole batch, positions in limit[]
    int        r0;      // first row, counted from token b
    int        b, e;    // tokens
    int        end, len;  // of the sequence: its last token + 1, positions
};

// The row that a lane deals with.
struct row_t {
    int token = -1;  // -1: no such row
    int head = 0;
    int limit = 0x7fffffff;  // its last position
};

// Row i of the tile, all but its limit.
__device__ inline row_t row_of(attention_dev_t const& a, work_t const& k, int kvh, int i)
{
    row_t     row;
    int const r = k.r0 + i;
    int const j = r / a.group;
    int const t = k.b + j;
    if (t >= k.e) return row;
    row.token = t;
    row.head = kvh * a.group + r - j * a.group;
    return row;
}

__device__ inline void set_limit(attention_dev_t const& a, work_t const& k, int const* limit,
                                 row_t& row)
{
    if (row.token < 0) return;
    if (!k.whole) {
        row.limit = max(k.len - (k.end - row.token), -1);
        return;
    }
    int const at = limit[row.token - k.r0 / a.group];
    if (at == -2) {
        row.token = -1;  // of no sequence
    } else {
        row.limit = at;
    }
}

// Workgroups go to the eight XCDs in turn, so with the key heads innermost every XCD gets the same
// heads of all units: equal work however long the sequences are, and tiles that read the same keys
// share an L2.
__device__ inline void unit_of_block(attention_dev_t const& a, int block, int& unit, int& kvh)
{
    kvh = block % a.h_kv;
    unit = block / a.h_kv;
}

// The sequence through whose row of the page table the shared positions are read: one that has
// tokens and maps them all, the first if it does; if none does, the longest, beyond which no row sees
// any.  (An idle sequence's row holds anything, and that of one that ends inside the prefix too from
// there on.)  All lanes take part.
__device__ inline int prefix_sequence(attention_dev_t const& a)
{
    int const need = min(a.shared, a.max_pages * a.page_size);
    auto      length = [&](int s) {
        bool const any = min(a.offsets[s + 1], a.n_tokens) > max(a.offsets[s], 0);
        return any ? a.lens[s] : -1;
    };
    if (length(0) >= need) return 0;
    int const lane = int(threadIdx.x) & 63;
    int       best = -1, at = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
        int const      len = s0 + lane < a.n_seqs ? length(s0 + lane) : -1;
        uint64_t const all = __ballot(len >= need);
        if (all) return s0 + __ffsll((unsigned long long)all) - 1;
        at = len > best ? s0 + lane : at;
        best = max(best, len);
    }
    int const longest = __builtin_amdgcn_readlane(wave_max(max(best, 0)), 63);
    uint64_t const which = __ballot(best == longest);
    return which ? __builtin_amdgcn_readlane(at, __ffsll((unsigned long long)which) - 1) : 0;
}

// A prefix workgroup: a tile of the batch's rows against a cut of the shared positions.
template <int ROWS>
__device__ inline void deal_prefix(attention_dev_t const& a, int unit, int kvh, work_t& k)
{
    int const tile = unit % a.prefix_tiles;
    int const split = unit / a.prefix_tiles;
    k.part = (int64_t(unit) * a.h_kv + kvh) * ROWS;
    k.lo = split * a.prefix_chunk;
    k.hi = min(min(k.lo + a.prefix_chunk, a.shared), a.max_pages * a.page_size);
    k.table = a.table + uint64_t(prefix_sequence(a)) * a.table_stride;
    k.direct = false;
    k.whole = true;
    k.r0 = tile * ROWS;
    k.b = 0;
    k.e = min((k.r0 + ROWS - 1) / a.group + 1, a.n_tokens);
    k.end = k.len = 0;
}

// Puts down the positions of the tile's tokens in their sequences (-2: of none); `limit` holds
// ROWS ints.  Ends with a barrier.
template <int ROWS>
__device__ inline void prefix_limits(attention_dev_t const& a, work_t const& k, int* limit)
{
    int const tid = int(threadIdx.x), t0 = k.r0 / a.group;
    for (int i = tid; i < ROWS; i += THREADS) limit[i] = -2;
    __syncthreads();
    for (int s = tid; s < a.n_seqs; s += THREADS) {
        int const b = a.offsets[s], e = a.offsets[s + 1];
        int const len = a.lens[s];
        for (int t = max(b, t0); t < min(e, k.e); ++t) limit[t - t0] = max(len - (e - t), -1);
    }
    __syncthreads();
}

// ---- the sequences' own positions
//
// Work is counted in units: a tile of rows (ROWS queries of one sequence) times `grain` steps of
// KS positions, at least one per tile.  A tile is cut into pieces of `each` units, so that the
// batch has about `shares` of them, and what is left over; a piece to a workgroup.  The whole
// pieces are numbered first, the rests behind them: workgroups start in this order, so the short
// ones fill the gaps at the end.  All of it follows from the lengths in device memory, and every
// workgroup works it out for itself: up to 64 sequences a wavefront does, one per lane; more are
// dealt to the threads in runs.
struct deal_t {
    int sums[3][WAVES];
    int found[8];
};

struct sequence_t {
    int s, b, e, len;
    int per;            // units per tile
    int whole0, rest0;  // number of its first whole piece, of its first rest
};

// Tiles of a sequence and units per tile.
template <int ROWS, int KS>
__device__ inline void measure(attention_dev_t const& a, int b, int e, int len, int& tiles, int& per)
{
    int const first = max(b, 0), last = min(e, a.n_tokens);
    int const reach = min(len, a.max_pages * a.page_size);
    int const steps = reach > a.shared ? (reach + KS - 1) / KS - a.shared / KS : 0;
    tiles = last > first ? ((last - first) * a.group + ROWS - 1) / ROWS : 0;
    per = max(1, (steps + a.grain - 1) / a.grain);
}

// Units per piece.  With few rows a multiple of four steps: one for each wavefront that takes them
// in turn.
template <int ROWS>
__device__ inline int units_per_piece(attention_dev_t const& a, int total)
{
    if (a.shares == 0) return 0x3fffffff;
    int const each = max(1, (total + a.shares - 1) / a.shares);
    return ROWS == FEW && a.grain % WAVES ? (each + WAVES - 1) / WAVES * WAVES : each;
}

// The piece that `item` numbers; false: there is none.  The same in all lanes.
template <int ROWS, int KS>
__device__ inline bool piece(attention_dev_t const& a, deal_t& sh, int kvh, int item, work_t& k)
{
    if (item >= a.own_slots) return false;
    int const  tid = int(threadIdx.x), lane = tid & 63, w = tid >> 6;
    sequence_t q;
    int        each, wholes;  // units per piece, whole pieces in all
    if (a.n_seqs <= 64) {
        int sb = 0, se = 0, slen = 0, tiles = 0, per = 1;
        if (lane < a.n_seqs) {
            sb = a.offsets[lane];
            se = a.offsets[lane + 1];
            slen = a.lens[lane];
            measure<ROWS, KS>(a, sb, se, slen, tiles, per);
        }
        each = units_per_piece<ROWS>(a, __builtin_amdgcn_readlane(wave_scan(tiles * per), 63));
        if (ROWS != FEW) {
            // The least size of which the batch has at most `shares` pieces, rests included, so
            // that all run at once and there are fewer to join (prompts: 87 us with the rests on
            // top of `shares`, 69 us).  More tiles than that: several rounds anyway.
            int const count = __builtin_amdgcn_readlane(wave_scan(tiles), 63);
            int       most = __builtin_amdgcn_readlane(wave_max(tiles > 0 ? per : 0), 63);
            if (count <= a.shares) {
                while (each < most) {
                    int const mid = (each + most) / 2;
                    int const pieces = tiles * ((per + mid - 1) / mid);
                    if (__builtin_amdgcn_readlane(wave_scan(pieces), 63) <= a.shares) {
                        most = mid;
                    } else {
                        each = mid + 1;
                    }
                }
            }
        }
        int const whole = tiles * (per / each), rest = tiles * (per % each != 0);
        int const whole_n = wave_scan(whole), rest_n = wave_scan(rest);
        wholes = __builtin_amdgcn_readlane(whole_n, 63);
        int const      at = item < wholes ? item : item - wholes;
        int const      mine = item < wholes ? whole : rest;
        int const      start = (item < wholes ? whole_n : rest_n) - mine;
        uint64_t const here = __ballot(at >= start && at < start + mine);
        if (here == 0) return false;
        int const s = __ffsll((unsigned long long)here) - 1;
        q.s = s;
        q.b = __builtin_amdgcn_readlane(sb, s);
        q.e = __builtin_amdgcn_readlane(se, s);
        q.len = __builtin_amdgcn_readlane(slen, s);
        q.per = __builtin_amdgcn_readlane(per, s);
        q.whole0 = __builtin_amdgcn_readlane(whole_n - whole, s);
        q.rest0 = __builtin_amdgcn_readlane(rest_n - rest, s);
    } else {
        int const run = (a.n_seqs + THREADS - 1) / THREADS;
        int const s0 = min(tid * run, a.n_seqs), s1 = min(s0 + run, a.n_seqs);
        int       b = 0, e = 0, len = 0, tiles = 0, per = 1, units = 0;
        auto      read = [&](int s) {
            b = a.offsets[s];
            e = a.offsets[s + 1];
            len = a.lens[s];
            measure<ROWS, KS>(a, b, e, len, tiles, per);
        };
        for (int s = s0; s < s1; ++s) {
            read(s);
            units += tiles * per;
        }
        units = wave_scan(units);
        if (lane == 63) sh.sums[0][w] = units;
        if (tid == 0) sh.found[0] = -1;
        __syncthreads();
        each = units_per_piece<ROWS>(a, sh.sums[0][0] + sh.sums[0][1] + sh.sums[0][2] + sh.sums[0][3]);
        int whole = 0, rest = 0;
        for (int s = s0; s < s1; ++s) {
            if (run > 1) read(s);
            whole += tiles * (per / each);
            rest += tiles * (per % each != 0);
        }
        int const whole_n = wave_scan(whole), rest_n = wave_scan(rest);
        if (lane == 63) {
            sh.sums[1][w] = whole_n;
            sh.sums[2][w] = rest_n;
        }
        __syncthreads();
        int whole0 = whole_n - whole, rest0 = rest_n - rest;
        wholes = 0;
#pragma unroll
        for (int i = 0; i != WAVES; ++i) {
            whole0 += i < w ? sh.sums[1][i] : 0;
            rest0 += i < w ? sh.sums[2][i] : 0;
            wholes += sh.sums[1][i];
        }
        int const at = item < wholes ? item : item - wholes;
        int const start = item < wholes ? whole0 : rest0, mine = item < wholes ? whole : rest;
        if (at >= start && at < start + mine) {
            for (int s = s0; s < s1; ++s) {
                if (run > 1) read(s);
                int const n = tiles * (per / each), r = tiles * (per % each != 0);
                if (at < (item < wholes ? whole0 + n : rest0 + r)) {
                    sh.found[0] = s;
                    sh.found[1] = b;
                    sh.found[2] = e;
                    sh.found[3] = len;
                    sh.found[4] = per;
                    sh.found[5] = whole0;
                    sh.found[6] = rest0;
                    break;
                }
                whole0 += n;
                rest0 += r;
            }
        }
        __syncthreads();
        q.s = __builtin_amdgcn_readfirstlane(sh.found[0]);
        if (q.s < 0) return false;
        q.b = __builtin_amdgcn_readfirstlane(sh.found[1]);
        q.e = __builtin_amdgcn_readfirstlane(sh.found[2]);
        q.len = __builtin_amdgcn_readfirstlane(sh.found[3]);
        q.per = __builtin_amdgcn_readfirstlane(sh.found[4]);
        q.whole0 = __builtin_amdgcn_readfirstlane(sh.found[5]);
        q.rest0 = __builtin_amdgcn_readfirstlane(sh.found[6]);
        wholes = __builtin_amdgcn_readfirstlane(wholes);
        each = __builtin_amdgcn_readfirstlane(each);
    }
    int const n = q.per / each, rest = q.per - n * each;
    int       tile, at;
    if (item < wholes) {
        tile = (item - q.whole0) / n;
        at = (item - q.whole0 - tile * n) * each;
    } else {
        tile = item - wholes - q.rest0;
        at = n * each;
    }
    k.b = max(q.b, 0);
    k.e = min(q.e, a.n_tokens);
    k.end = q.e;
    k.len = q.len;
    k.whole = false;
    k.part = a.own_base + (int64_t(item) * a.h_kv + kvh) * ROWS;
    int const parts = n + (rest != 0);
    k.direct = parts == 1 && a.direct;
    k.table = a.table + uint64_t(q.s) * a.table_stride;
    k.r0 = tile * ROWS;
    if (at == 0 && kvh == 0 && a.part_meta) {
        // where the rows' partial results are: from x on y of them, then z (or none); w the row
        for (int i = tid; i < ROWS; i += THREADS) {
            int const r = k.r0 + i, t = k.b + r / a.group;
            if (t < k.e) {
                a.part_meta[k.b * a.group + r] =
                    int4{q.whole0 + tile * n, k.direct ? -1 : n,
                         rest ? wholes + q.rest0 + tile : -1, i};
            }
        }
    }
    int const last = min(k.e - 1, k.b + (k.r0 + ROWS - 1) / a.group);
    // positions, up to the last one that a row of the tile sees
    int const step0 = a.shared / KS + at * a.grain;
    k.lo = max(a.shared, step0 * KS);
    k.hi = min(min(k.len, a.max_pages * a.page_size), (step0 + min(each, q.per - at) * a.grain) * KS);
    k.hi = min(k.hi, k.len - (k.end - last) + 1);
    return true;
}

// Keys and values that hardly any other workgroup reads, as f16 sequences of few rows are one tile:
// not kept in the caches (32 heads of keys, 32 tokens, a launch of their own: 49.2 us, 47.8 us with
// it; in one launch with the shared positions 58 to 61 us either way).  In f32 every tile has sixteen
// rows, and long ones read the same keys many times.
template <typename V>
__device__ inline V read_once(void const* p)
{
    return __builtin_nontemporal_load(static_cast<V const*>(p));
}

template <typename T, int D>
struct core_t;

// ---- f16: steps of 16 keys, v_mfma_f32_16x16x32_f16 for the scores, v_mfma_f32_16x16x16_f16 for
// the values.  Steps of 32 keys would use the matrix unit twice as well, which nothing here waits
// for, and hold twice the registers: two workgroups per compute unit instead of four.
template <int D>
struct core_t<_Float16, D> {
    static constexpr int KS = 16;     // keys per step
    static constexpr int KL = 4;      // keys whose scores a lane holds
    static constexpr int DV = D / 16; // elements of a row of V per lane
    static constexpr int QC = D / 32;
    static constexpr int LIFT = WEIGHT_LIFT;

    half8_t k[QC];
    struct vrow_t {
        uint32_t u[DV / 2];
    } v[KL];

    static __device__ int key_of(int j, int g) { return 4 * g + j; }

    // PAD: d is below D.  Loads are unconditional (a branch around each would make it wait for
    // the one before); elements beyond d come from the row's start and are zeroed.  The queries
    // wait in LDS, lane by lane: every step reads them once.
    typedef half8_t query_t;
    template <bool PAD>
    static __device__ void load_q(query_t (*q)[64], int lane, _Float16 const* row, int g, int d,
                                  float sign)
    {
#pragma unroll
        for (int c = 0; c != QC; ++c) {
            int const  e = c * 32 + g * 8;
            bool const in = !PAD || e < d;
            half8_t const x = *reinterpret_cast<half8_t const*>(row + (in ? e : 0)) * _Float16(sign);
            q[c][lane] = PAD && !in ? half8_t{} : x;
        }
    }
    // element offsets of the key this lane loads of K, the four of V; negative ones (no such
    // entry) read the cache's first, to be masked by the caller
    template <bool PAD>
    __device__ void load_k(_Float16 const* kb, int64_t const* off, int c, int g, int d)
    {
        _Float16 const* p = kb + max(off[c], int64_t(0));
#pragma unroll
        for (int i = 0; i != QC; ++i) {
            int const e = i * 32 + g * 8;
            k[i] = read_once<half8_t>(p + (!PAD || e < d ? e : 0));
        }
    }
    template <bool PAD>
    __device__ void load_v(_Float16 const* vb, int64_t const* off, int c, int g, int d)
    {
        int64_t ov[KL];
#pragma unroll
        for (int j = 0; j != KL; ++j) ov[j] = off[key_of(j, g)];
        constexpr int N = DV < 8 ? DV : 8;  // d is a multiple of 8
        typedef uint32_t vec_t __attribute__((ext_vector_type(N / 2)));
#pragma unroll
        for (int j = 0; j != KL; ++j) {
            _Float16 const* p = vb + max(ov[j], int64_t(0));
#pragma unroll
            for (int e = 0; e != DV; e += N) {
                bool const  in = !PAD || c * DV + e < d;
                vec_t const x = read_once<vec_t>(p + (in ? c * DV + e : 0));
#pragma unroll
                for (int i = 0; i != N / 2; ++i) v[j].u[e / 2 + i] = x[i];
            }
        }
    }
    // zeros beyond d, once the loads are there
    template <bool PAD>
    __device__ void trim_k(int g, int d)
    {
        if (!PAD) return;
#pragma unroll
        for (int i = 0; i != QC; ++i) {
            if (i * 32 + g * 8 >= d) k[i] = half8_t{};
        }
    }
    template <bool PAD>
    __device__ void trim_v(int c, int d)
    {
        if (!PAD) return;
#pragma unroll
        for (int j = 0; j != KL; ++j) {
#pragma unroll
            for (int i = 0; i != DV / 2; ++i) v[j].u[i] = c * DV + 2 * i < d ? v[j].u[i] : 0;
        }
    }
    // zeros for what is not finite; true: there was some
    __device__ bool clean_key(int j)
    {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i != DV / 2; ++i) {
            uint32_t const u = v[j].u[i];
            uint32_t const cut = ((u & 0x7c00u) == 0x7c00u ? 0xffffu : 0) |
                                 ((u & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0);
            v[j].u[i] = u & ~cut;
            bad |= cut;
        }
        return bad != 0;
    }
    __device__ void scores(float* s, query_t const (*q)[64], int lane) const
    {
        float4_t a = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i != QC; ++i) {
            a = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[i], q[i][lane], a, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r != 4; ++r) s[r] = a[r];
    }
    // o[t] += V^T P^T for the elements i * DV + t of the head, i the result's row
    __device__ void values(float const* p, float4_t* o) const
    {
        union {
            half2_t pair[2];
            half4_t h;
        } high, low;
#pragma unroll
        for (int j = 0; j != KL; j += 2) {
            split_weights(float2_t{p[j], p[j + 1]}, high.pair[j / 2], low.pair[j / 2]);
        }
#pragma unroll
        for (int t = 0; t != DV; ++t) {
            union {
                uint32_t u[2];
                half4_t  h;
            } a;
            uint32_t const sel = t & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
            for (int i = 0; i != 2; ++i) {
                a.u[i] = __builtin_amdgcn_perm(v[2 * i + 1].u[t / 2], v[2 * i].u[t / 2], sel);
            }
            o[t] = __builtin_amdgcn_mfma_f32_16x16x16f16(a.h, high.h, o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x16f16(a.h, low.h, o[t], 0, 0, 0);
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
    static constexpr int LIFT = 0;

    float4_t k[QC];
    float    v[KL][DV];

    static __device__ int key_of(int j, int g) { return 4 * g + j; }

    typedef float4_t query_t;
    template <bool PAD>
    static __device__ void load_q(query_t (*q)[64], int lane, float const* row, int g, int d,
                                  float sign)
    {
#pragma unroll
        for (int c = 0; c != QC; ++c) {
            int const  e = c * 16 + g * 4;
            bool const in = !PAD || e < d;
            float4_t const x = *reinterpret_cast<float4_t const*>(row + (in ? e : 0)) * sign;
            q[c][lane] = PAD && !in ? float4_t{} : x;
        }
    }
    template <bool PAD>
    __device__ void load_k(float const* kb, int64_t const* off, int c, int g, int d)
    {
        int64_t const ok = off[c];
        float const*  p = kb + max(ok, int64_t(0));
#pragma unroll
        for (int i = 0; i != QC; ++i) {
            int const e = i * 16 + g * 4;
            k[i] = *reinterpret_cast<float4_t const*>(p + (!PAD || e < d ? e : 0));
        }
    }
    template <bool PAD>
    __device__ void load_v(float const* vb, int64_t const* off, int c, int g, int d)
    {
        int64_t ov[KL];
#pragma unroll
        for (int j = 0; j != KL; ++j) ov[j] = off[key_of(j, g)];
#pragma unroll
        for (int j = 0; j != KL; ++j) {
            float const* pv = vb + max(ov[j], int64_t(0));
#pragma unroll
            for (int e = 0; e != DV; e += 4) {
                bool const     in = !PAD || c * DV + e < d;
                float4_t const x = *reinterpret_cast<float4_t const*>(pv + (in ? c * DV + e : 0));
#pragma unroll
                for (int i = 0; i != 4; ++i) v[j][e + i] = x[i];
            }
        }
    }
    template <bool PAD>
    __device__ void trim_k(int g, int d)
    {
        if (!PAD) return;
#pragma unroll
        for (int i = 0; i != QC; ++i) {
            if (i * 16 + g * 4 >= d) k[i] = float4_t{};
        }
    }
    template <bool PAD>
    __device__ void trim_v(int c, int d)
    {
        if (!PAD) return;
#pragma unroll
        for (int j = 0; j != KL; ++j) {
#pragma unroll
            for (int e = 0; e != DV; ++e) v[j][e] = c * DV + e < d ? v[j][e] : 0.0f;
        }
    }
    __device__ bool clean_key(int j)
    {
        bool bad = false;
#pragma unroll
        for (int e = 0; e != DV; ++e) {
            bool const fine = finite(v[j][e]);
            v[j][e] = fine ? v[j][e] : 0.0f;
            bad |= !fine;
        }
        return bad;
    }
    __device__ void scores(float* s, query_t const (*q)[64], int lane) const
    {
        float4_t a = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i != QC; ++i) {
            float4_t const x = q[i][lane];
#pragma unroll
            for (int e = 0; e != 4; ++e) {
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i][e], x[e], a, 0, 0, 0);
            }
        }
#pragma unroll
        for (int r = 0; r != 4; ++r) s[r] = a[r];
    }
    __device__ void values(float const* p, float4_t* o) const
    {
#pragma unroll
        for (int t = 0; t != DV; ++t) {
#pragma unroll
            for (int j = 0; j != KL; ++j) {
                o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j][t], p[j], o[t], 0, 0, 0);
            }
        }
    }
};

// The sum of a row's weights in a part, with the reference m (l: their sum, zero also where none was
// added).  A softmax over scores that are all -inf is NaN, over no score the caller wants zeros: where
// m is -inf and l zero, -1 says that the row saw a key all the same.  (NaN scores leave m alone and
// make l NaN.)  All lanes take part: they look for the part's first position with a page together.
__device__ inline float sum_of(attention_dev_t const& a, work_t const& k, int limit, float m, float l)
{
    bool const none = m == NEG_INF && l == 0.0f && limit >= k.lo;
    if (!__any(none)) return l;
    int const lane = int(threadIdx.x) & 63;
    for (int base = k.lo; base < k.hi; base += 64) {
        int const      pos = min(base + lane, k.hi - 1);
        uint64_t const there = __ballot(entry_of(a, k.table[page_of(a, pos)], 0) >= 0);
        if (there) {
            int const first = min(base + __ffsll((unsigned long long)there) - 1, k.hi - 1);
            return none && limit >= first ? -1.0f : l;
        }
    }
    return l;
}

// What an element of O is multiplied with: 1 / sum, zero for a row that saw nothing.
__device__ inline float weight_of(float sum)
{
    return sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : __builtin_nanf("");
}

// Whether a score is so much above a row's reference that the reference has to follow.
__device__ inline bool rises(float top, float m) { return top > m + 8.0f; }

// Takes the scores of a step into a row's reference m, what exponents are taken relative to
// (`top`: the largest of this lane's).  The reference need not be the maximum: it is raised, and
// what was summed so far scaled down, only where a score passes it by 2^8, which leaves p below
// 2^(8 + LIFT) and f16's relative precision as it is; so the lanes of a column have to agree on their
// maximum only then.  `ref` is m - LIFT, or anything while nothing was seen.
template <int N, int LIFT>
__device__ inline void raise(float top, float& m, float& ref, float& l, float4_t* o)
{
    if (__any(rises(top, m))) {
        float const mn = fmaxf(m, column_max(top));
        float const base = mn == NEG_INF ? 0.0f : mn;
        float const fade = exp2_fast(m - base);
        ref = base - float(LIFT);
        l *= fade;
#pragma unroll
        for (int t = 0; t != N; ++t) o[t] *= fade;
        m = mn;
    }
}

// ------------------------------------------------------------------------------ few rows


template <typename T, int D>
struct few_shared_t {
    static constexpr int DJ = D < 128 ? D : 128;  // elements joined at a time
    deal_t  deal;
    int     limit[FEW];
    int64_t off[WAVES][16];
    float   m[WAVES][FEW], l[WAVES][FEW];
    union {
        float                          o[WAVES][FEW][DJ + 4];
        typename core_t<T, D>::query_t q[core_t<T, D>::QC][64];  // the same for every wavefront
    };
};

// The workgroup's keys against the tile's rows; steps w, w + WAVES, ...
template <typename T, int D, bool PAD>
__device__ void attend_few(attention_dev_t const& a, int64_t* off,
                           typename core_t<T, D>::query_t const (*q)[64], work_t const& wk,
                           row_t const& row, int least, int kvh, float4_t* o, float& m, float& l)
{
    typedef core_t<T, D> core;
    constexpr int        KS = core::KS, KL = core::KL, DV = core::DV;
    int const            lane = int(threadIdx.x) & 63;
    int const            w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    int const            g = lane >> 4, c = lane & 15;
    T const* const       kb = reinterpret_cast<T const*>(a.k) + uint64_t(kvh) * a.head_stride;
    T const* const       vb = reinterpret_cast<T const*>(a.v) + uint64_t(kvh) * a.head_stride;
    core                 x;
    constexpr int        STEP = WAVES * KS;
    int const lo = __builtin_amdgcn_readfirstlane(wk.lo);
    int const hi = __builtin_amdgcn_readfirstlane(wk.hi);
    int const seen_by_all = __builtin_amdgcn_readfirstlane(least);
    // A step ahead: the page of this lane's key.  Positions that are not the workgroup's stand for
    // its first or last.
    int  page = -1, prow = 0;
    auto look_up = [&](int at) {
        int const pos = min(max(at + (lane & (KS - 1)), lo), hi - 1);
        int const pi = page_of(a, pos);
        prow = pos - pi * a.page_size;
        page = wk.table[pi];
    };
    // A weight of zero -- a key that the row may not see, a position without a page, a weight that
    // underflows -- times an infinity or NaN is no zero.  So where some row's result is not finite,
    // the keys are gone through once more with such values made zeros, and in the end they are added
    // to the rows that see them.
    bool bad = false;  // some value was not finite
    for (int careful = 0;; careful = 1) {
        int   base = (lo / KS + w) * KS;
        float ref = 0;
        look_up(base);
        for (; base < hi; base += STEP) {
            // where the keys lie, for all lanes; -1: no such page
            int64_t const at = entry_of(a, page, prow);
            bool const    holes = __any(at < 0);
            __builtin_amdgcn_wave_barrier();
            if (lane < KS) off[lane] = at;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            x.template load_k<PAD>(kb, off, c, g, a.d);
            x.template load_v<PAD>(vb, off, c, g, a.d);
            look_up(base + STEP);
            // all of the step's loads go out before the first is waited for; what hides their
            // latency is the other fifteen wavefronts of the compute unit
            __builtin_amdgcn_sched_barrier(0);
            x.template trim_k<PAD>(g, a.d);
            float s[KL];
            x.scores(s, q, lane);
            x.template trim_v<PAD>(c, a.d);
            bool const edge = holes || base < lo || base + KS > hi || base + KS - 1 > seen_by_all;
            uint32_t   masked = 0;
            if (edge) {
#pragma unroll
                for (int j = 0; j != KL; ++j) {
                    int const key = core::key_of(j, g);
                    masked |= off[key] < 0 || base + key < lo ||
                                      base + key > min(hi - 1, row.limit)
                                  ? 1u << j
                                  : 0;
                }
            }
            if (opaque(careful)) {
#pragma unroll
                for (int j = 0; j != KL; ++j) bad |= x.clean_key(j);
            }
            float top = NEG_INF;
#pragma unroll
            for (int j = 0; j != KL; ++j) {
                s[j] = masked >> j & 1 ? NEG_INF : s[j];
                top = fmaxf(top, s[j]);
            }
            raise<DV, core::LIFT>(top * a.scale, m, ref, l, o);
            float sum = 0;
#pragma unroll
            for (int j = 0; j != KL; ++j) {
                s[j] = exp2_fast(s[j] * a.scale - ref);
                sum += s[j];
            }
            l += sum;
            x.values(s, o);
        }
        if (careful) break;
        bool again = false;
#pragma unroll
        for (int t = 0; t != DV; ++t) {
#pragma unroll
            for (int r = 0; r != 4; ++r) again |= !finite(o[t][r]);
        }
        if (!__any(again && row.token >= 0)) break;
#pragma unroll
        for (int t = 0; t != DV; ++t) o[t] = float4_t{0, 0, 0, 0};
        m = NEG_INF;
        l = 0;
    }
    if (__any(bad)) {
        for (int base = (lo / KS + w) * KS; base < hi; base += STEP) {
            for (int pos = max(base, lo); pos < min(base + KS, hi); ++pos) {
                int const     pi = page_of(a, pos);
                int64_t const at = entry_of(a, wk.table[pi], pos - pi * a.page_size);
                if (at < 0) continue;
#pragma unroll
                for (int t = 0; t != DV; ++t) {
#pragma unroll
                    for (int r = 0; r != 4; ++r) {
                        int const   e = (4 * g + r) * DV + t;
                        float const y = float(vb[at + (!PAD || e < a.d ? e : 0)]);
                        bool const  add = !finite(y) && (!PAD || e < a.d);
                        o[t][r] += add && pos <= row.limit ? y : 0.0f;
                    }
                }
            }
        }
    }
    // the four lanes of a column hold sums over different keys
    l = column_sum(l);
}

// Workgroup `block` of those that have few rows, the first prefix_units units of them the batch's.
template <typename T, int D, bool PAD>
__device__ __forceinline__ void few_rows(attention_dev_t const& a, few_shared_t<T, D>& sh,
                                         int block, int prefix_units)
{
    int const tid = int(threadIdx.x), lane = tid & 63, w = tid >> 6;
    int const c = lane & 15, g = lane >> 4;
    constexpr int KS = core_t<T, D>::KS, DV = core_t<T, D>::DV;
    int           unit, kvh;
    unit_of_block(a, block, unit, kvh);
    work_t wk;
    if (unit < prefix_units) {
        deal_prefix<FEW>(a, unit, kvh, wk);
        prefix_limits<FEW>(a, wk, sh.limit);
    } else if (!piece<FEW, KS>(a, sh.deal, kvh, unit - prefix_units, wk)) {
        return;
    }
    row_t row = row_of(a, wk, kvh, c);
    set_limit(a, wk, sh.limit, row);
    int least = row.limit;
#pragma unroll
    for (int i = 1; i != 16; i <<= 1) least = min(least, __shfl_xor(least, i));

    float4_t o[DV];
#pragma unroll
    for (int t = 0; t != DV; ++t) o[t] = float4_t{0, 0, 0, 0};
    float m = NEG_INF, l = 0;
    // a column without a row computes what nobody stores
    if (w == 0) {
        core_t<T, D>::template load_q<PAD>(sh.q, lane,
                                           reinterpret_cast<T const*>(a.q) +
                                               uint64_t(max(row.token, 0)) * a.q_stride +
                                               uint64_t(row.head) * uint64_t(a.d),
                                           g, a.d, a.q_sign);
    }
    __syncthreads();
    if (wk.lo < wk.hi) attend_few<T, D, PAD>(a, sh.off[w], sh.q, wk, row, least, kvh, o, m, l);
    __syncthreads();  // the queries' place is used again

    // join the wavefronts
    if (g == 0) {
        sh.m[w][c] = m;
        sh.l[w][c] = l;
    }
    __syncthreads();
    float top = NEG_INF;
#pragma unroll
    for (int i = 0; i != WAVES; ++i) top = fmaxf(top, sh.m[i][c]);
    float const   mine = exp2_fast(m - (top == NEG_INF ? 0.0f : top));
    constexpr int DJ = few_shared_t<T, D>::DJ;
    constexpr int TPR = THREADS / FEW;  // threads that store a row
    constexpr int PER = DJ / TPR;
    int const     orow = tid / TPR, oe = tid % TPR * PER;
    // the row that this thread stores, from the lane that knows it
    int const   otoken = __shfl(row.token, orow);
    int const   ohead = __shfl(row.head, orow);
    int const   olimit = __shfl(row.limit, orow);
    float const otop = __shfl(top, orow);
    float       sum = 0;
#pragma unroll
    for (int i = 0; i != WAVES; ++i) {
        float const mi = sh.m[i][orow];
        sum += sh.l[i][orow] * exp2_fast(mi - (otop == NEG_INF ? 0.0f : otop));
    }
    sum = sum_of(a, wk, otoken < 0 ? -1 : olimit, otop, sum);
#pragma unroll
    for (int h = 0; h != D / DJ; ++h) {
        if (h) __syncthreads();
        // O^T: this lane has the elements (4 g + r) * DV + t of its column's row
#pragma unroll
        for (int r = 0; r != 4; ++r) {
            int const e = (4 * g + r) * DV;
            if (D > DJ && e / DJ != h) continue;
#pragma unroll
            for (int t = 0; t != DV; ++t) sh.o[w][c][e - h * DJ + t] = scaled(o[t][r], mine);
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
            if (wk.direct) {
                T* const dst = reinterpret_cast<T*>(a.out) + uint64_t(otoken) * a.out_stride +
                               uint64_t(ohead) * uint64_t(a.d) + h * DJ + oe;
                float const inv = weight_of(sum);
                // PER divides 8, and 8 divides d: all of them or none
                typedef T vec_t __attribute__((ext_vector_type(PER)));
                vec_t     z;
#pragma unroll
                for (int e = 0; e != PER; ++e) z[e] = T(y[e] * inv);
                if (h * DJ + oe < a.d) *reinterpret_cast<vec_t*>(dst) = z;
            } else {
                float* const dst = a.part_o + (wk.part + orow) * D + h * DJ + oe;
#pragma unroll
                for (int e = 0; e != PER; e += 4) {
                    *reinterpret_cast<float4_t*>(dst + e) =
                        float4_t{y[e], y[e + 1], y[e + 2], y[e + 3]};
                }
            }
        }
    }
    if (!wk.direct && otoken >= 0 && oe == 0) {
        a.part_ml[(wk.part + orow) * 2] = otop;
        a.part_ml[(wk.part + orow) * 2 + 1] = sum;
    }
}

// ------------------------------------------------------------------------------ many rows

// What positions without a page, and elements beyond head_dim, are loaded from.
__device__ __align__(16) uint32_t const attention_zeros[128] = {0};

// 64 lanes x 16 bytes from each lane's address to LDS at lds + 16 * lane.
__device__ __forceinline__ void load_to_lds_16(void const* from, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(lds), "v"(from)
                 : "memory");
}

__device__ __forceinline__ void load_to_lds_4(void const* from, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :
                 : "s"(lds), "v"(from)
                 : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads()
{
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

__device__ __forceinline__ uint32_t lds_address(void const* p)
{
    return __builtin_amdgcn_readfirstlane(
        uint32_t(uintptr_t((__attribute__((address_space(3))) char const*)(p))));
}

// f16 only.  Tiles of KT keys lie in LDS as rows of D elements, 16-byte chunks XOR-swizzled with
// the row: K by row % 16 (a fragment read takes one chunk of 16 rows), V by 2 (row % 8) (a
// transposing read takes 32 bytes of four rows); neither read has bank conflicts.  The loads go
// from global memory straight to LDS, NS - 1 tiles ahead, one barrier per tile.  Where a
// position's entry lies is worked out for a window of 256 positions at a time, a position per
// thread; the page numbers of the next window come through LDS as well, several tiles ahead, so
// no wait for them drains the tiles in flight.
//
// The scores of tile i + 1 are computed in the iteration that turns those of tile i into weights:
// the exponentials take the vector unit about as long as the matrix unit needs for the scores,
// and in one stretch of code without dependences the two overlap.
template <int D, int NT>
struct many_t {
    static constexpr int ROWS = WAVES * 16 * NT;
    static constexpr int KT = 32;
    static constexpr int NS = 4;
    static constexpr int CH = D / 8;             // chunks per row
    static constexpr int RPL = 64 / CH;          // rows per load instruction
    static constexpr int LPT = KT / RPL / WAVES; // load instructions per wavefront and tile, of K
    static constexpr int DT = D / 16;
    static constexpr int WINDOW = 256, TPW = WINDOW / KT;
    struct shared_t {
        deal_t      deal;
        int         limit[ROWS];
        char const* kat[2][WINDOW];  // where the entries of a window's positions lie
        char const* vat[2][WINDOW];
        int         page[WINDOW];
        int         holes;  // some position has no page
        int         again;  // some row's result is not finite
        int         bad;    // some value was not finite
        half8_t     k[NS][KT][CH], v[NS][KT][CH];
    };
};

template <int D, int NT, bool PAD>
__device__ __forceinline__ void many_rows(attention_dev_t const& a,
                                          typename many_t<D, NT>::shared_t& sh, int block,
                                          int prefix_units)
{
    typedef many_t<D, NT> M;
    typedef _Float16      T;
    constexpr int         ROWS = M::ROWS, KT = M::KT, CH = M::CH, DT = M::DT, NS = M::NS;
    constexpr int         LPT = M::LPT, ST = KT / 16;
    int const tid = int(threadIdx.x), lane = tid & 63;
    int const w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int const c = lane & 15, g = lane >> 4;
    int       unit, kvh;
    unit_of_block(a, block, unit, kvh);
    bool const prefix = unit < prefix_units;
    work_t     wk;
    if (prefix) {
        deal_prefix<ROWS>(a, unit, kvh, wk);
    } else {
        if (!piece<ROWS, KT>(a, sh.deal, kvh, unit - prefix_units, wk)) return;
    }
    int const lo = __builtin_amdgcn_readfirstlane(wk.lo);
    int const hi = __builtin_amdgcn_readfirstlane(wk.hi);
    int const first = lo / 32 * 32;

    // this thread's position of window n, and its page number
    auto position = [&](int n) { return first + n * M::WINDOW + tid; };
    // (positions that are not the workgroup's stand for its first or last: one place for all of
    // them would be a hot spot in the caches)
    auto inside = [&](int pos) { return min(max(pos, lo), hi - 1); };
    auto page_at = [&](int pos) { return wk.table + page_of(a, inside(pos)); };
    int  page0 = -1;
    if (lo < hi) page0 = *page_at(position(0));

    row_t row[NT];
#pragma unroll
    for (int n = 0; n != NT; ++n) row[n] = row_of(a, wk, kvh, (w * NT + n) * 16 + c);

    half8_t  q[NT][D / 32];
    float4_t o[NT][DT];
    float    m[NT], ref[NT], l[NT];
    auto     start = [&]() {
#pragma unroll
        for (int n = 0; n != NT; ++n) {
#pragma unroll
            for (int t = 0; t != DT; ++t) o[n][t] = float4_t{0, 0, 0, 0};
            m[n] = NEG_INF;
            ref[n] = l[n] = 0;
        }
    };
#pragma unroll
    for (int n = 0; n != NT; ++n) {
        T const* const src = reinterpret_cast<T const*>(a.q) +
                             uint64_t(max(row[n].token, 0)) * a.q_stride +
                             uint64_t(row[n].head) * uint64_t(a.d);
#pragma unroll
        for (int i = 0; i != D / 32; ++i) {
            int const  e = i * 32 + g * 8;
            bool const in = !PAD || e < a.d;
            q[n][i] = *reinterpret_cast<half8_t const*>(src + (in ? e : 0)) * T(a.q_sign);
            if (PAD && !in) q[n][i] = half8_t{};
        }
    }
    start();

    if (lo < hi) {
        char const* const kb = a.k + uint64_t(kvh) * a.head_stride * 2;
        char const* const vb = a.v + uint64_t(kvh) * a.head_stride * 2;
        char const* const zeros = reinterpret_cast<char const*>(attention_zeros);
        int const         tiles = (hi - first + KT - 1) / KT;
        int               least = 0x7fffffff, most = -1;

        auto put_entry = [&](int n, int page) {
            int const     pos = inside(position(n));
            int64_t const at = entry_of(a, page, pos - page_of(a, pos) * a.page_size);
            if (at < 0) sh.holes = 1;
            sh.kat[n & 1][tid] = at < 0 ? zeros : kb + at * 2;
            sh.vat[n & 1][tid] = at < 0 ? zeros : vb + at * 2;
        };
        // this lane's row and chunk in a load instruction; the addresses of a tile are read from
        // the window a tile before its loads go out
        int const   lrow = lane / CH, lpos = lane % CH;
        char const *kp[LPT], *vp[LPT];
        auto        aim = [&](int tile) {
            int const win = tile / M::TPW & 1, at = tile % M::TPW * KT;
#pragma unroll
            for (int i = 0; i != LPT; ++i) {
                int const r = (i * WAVES + w) * M::RPL + lrow;
                int const kc = lpos ^ (r & 15 & (CH - 1));
                int const vc = lpos ^ ((2 * (r & 7)) & (CH - 1));
                kp[i] = sh.kat[win][at + r] + kc * 16;
                vp[i] = sh.vat[win][at + r] + vc * 16;
                if (PAD) {
                    kp[i] = kc * 8 < a.d ? kp[i] : zeros;
                    vp[i] = vc * 8 < a.d ? vp[i] : zeros;
                }
            }
        };
        uint32_t const lds_k = lds_address(&sh.k[0][w * M::RPL][0]);
        uint32_t const lds_v = lds_address(&sh.v[0][w * M::RPL][0]);
        auto           load_tile = [&](int tile) {
            uint32_t const slot = uint32_t(tile % NS) * uint32_t(KT * D * 2);
#pragma unroll
            for (int i = 0; i != LPT; ++i) {
                uint32_t const at = slot + uint32_t(i * WAVES * M::RPL * D * 2);
                load_to_lds_16(kp[i], lds_k + at);
                load_to_lds_16(vp[i], lds_v + at);
            }
        };
        auto scores = [&](int slot, float4_t(&s)[NT][ST]) {
#pragma unroll
            for (int n = 0; n != NT; ++n) {
#pragma unroll
                for (int t = 0; t != ST; ++t) s[n][t] = float4_t{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i != D / 32; ++i) {
#pragma unroll
                for (int t = 0; t != ST; ++t) {
                    half8_t const kf = sh.k[slot][16 * t + c][(4 * i + g) ^ (c & (CH - 1))];
#pragma unroll
                    for (int n = 0; n != NT; ++n) {
                        s[n][t] =
                            __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[n][i], s[n][t], 0, 0, 0);
                    }
                }
            }
        };
        // whether there are positions in a tile that some row may not see
        auto edge = [&](int tile, int holes) {
            int const base = first + tile * KT;
            return holes != 0 || base < lo || base + KT > hi || base + KT - 1 > least;
        };
        auto mask = [&](int tile, float4_t(&s)[NT][ST]) {
            int const base = first + tile * KT;
            char const* const* const at = &sh.kat[tile / M::TPW & 1][tile % M::TPW * KT];
#pragma unroll
            for (int t = 0; t != ST; ++t) {
#pragma unroll
                for (int r = 0; r != 4; ++r) {
                    int const  key = 16 * t + 4 * g + r, pos = base + key;
                    bool const none = pos < lo || pos >= hi || at[key] == zeros;  // no page
#pragma unroll
                    for (int n = 0; n != NT; ++n) {
                        if (none || pos > row[n].limit) s[n][t][r] = NEG_INF;
                    }
                }
            }
        };
        // the largest of this lane's scores of a row
        auto top_of = [&](float4_t const(&s)[ST]) {
            float top = NEG_INF;
#pragma unroll
            for (int t = 0; t != ST; ++t) {
#pragma unroll
                for (int r = 0; r != 4; ++r) top = fmaxf(top, s[t][r]);
            }
            return top * a.scale;
        };
        // (one test for all rows: it is hardly ever true)
        auto raise_all = [&](float4_t const(&s)[NT][ST]) {
            float top[NT];
            bool  more = false;
#pragma unroll
            for (int n = 0; n != NT; ++n) {
                top[n] = top_of(s[n]);
                more |= rises(top[n], m[n]);
            }
            if (!__any(more)) return;
#pragma unroll
            for (int n = 0; n != NT; ++n) {
                raise<DT, WEIGHT_LIFT>(top[n], m[n], ref[n], l[n], o[n]);
            }
        };

        // Values that are not finite become zeros, as in attend_few.  (A second copy of the steps: in
        // one loop for both passes the compiler needed 96 registers more.)
        auto clean = [&](int tile) {
            for (int i = tid; i < KT * CH; i += THREADS) {
                half8_t& x = sh.v[tile % NS][i / CH][i % CH];
                half8_t  y = x;
                bool     any = false;
#pragma unroll
                for (int e = 0; e != 8; ++e) {
                    if (!(y[e] - y[e] == T(0))) {
                        y[e] = T(0);
                        any = true;
                    }
                }
                if (any) {
                    x = y;
                    sh.bad = 1;
                }
            }
        };
        // weights of a tile, scores of the next one, O.  SLOT, the tile's modulo NS, is known to
        // the compiler: places in LDS are then offsets of the instructions.
        auto step = [&](int tile, float4_t(&s)[2][NT][ST], auto slot_, auto careful_) {
            constexpr int  SLOT = decltype(slot_)::value;
            constexpr bool CAREFUL = decltype(careful_)::value;
            float4_t(&now)[NT][ST] = s[SLOT & 1];
            float4_t(&next)[NT][ST] = s[(SLOT + 1) & 1];
            wait_loads<2 * LPT*(NS - 3)>();
            __syncthreads();
            // What is read from LDS is asked for well before its use, in an order that the
            // scheduler may not change: K of the next tile before the addresses of later ones are
            // worked out, V before the last weights.
            constexpr int NEXT = (SLOT + 1) % NS, NI = D / 32, PK = NI < 2 ? NI : 2, PV = 4;
            half8_t       kf[PK][ST];
            auto          read_k = [&](int i) {
#pragma unroll
                for (int t = 0; t != ST; ++t) {
                    kf[i % PK][t] = sh.k[NEXT][16 * t + c][(4 * i + g) ^ (c & (CH - 1))];
                }
            };
#pragma unroll
            for (int i = 0; i != PK; ++i) read_k(i);
            int const holes = sh.holes;
            __builtin_amdgcn_sched_barrier(0);
            // tile + NS - 1 goes where the last one was; windows are prepared on the way
            int const j = tile + NS - 1;
            load_tile(j);
            if (CAREFUL) clean(tile + 1);
            int const n = j / M::TPW, at = j % M::TPW;
            if (at == M::TPW - 3) put_entry(n + 1, sh.page[tid]);
            if (at == M::TPW - 1) {
                load_to_lds_4(page_at(position(n + 2)), lds_address(&sh.page[w * 64]));
            }
            aim(j + 1);
            if (first + tile * KT > most) return;
            // V^T: lane i of sixteen asks for four elements of key i / 4 and gets four keys of its
            // own element
            typedef short tr_t __attribute__((ext_vector_type(4)));
            union {
                tr_t    x[2];
                half8_t h;
            } vf[PV][KT / 32];
            auto read_v = [&](int t) {
#pragma unroll
                for (int ks = 0; ks != KT / 32; ++ks) {
#pragma unroll
                    for (int half = 0; half != 2; ++half) {
                        int const r = 32 * ks + 16 * half + 4 * g + (c >> 2);
                        int const chunk = (2 * t + ((c & 3) >> 1)) ^ ((2 * (r & 7)) & (CH - 1));
                        char*     at = reinterpret_cast<char*>(&sh.v[SLOT][r][chunk]) + (c & 1) * 8;
                        vf[t % PV][ks].x[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) tr_t*)(at));
                    }
                }
            };
#pragma unroll
            for (int n = 0; n != NT; ++n) {
#pragma unroll
                for (int t = 0; t != ST; ++t) next[n][t] = float4_t{0, 0, 0, 0};
            }
            union {
                half2_t pair[4];
                half8_t h;
            } high[NT][KT / 32], low[NT][KT / 32];
            // scores of the next tile and, in between, the weights of this one
#pragma unroll
            for (int i = 0; i != NI; ++i) {
#pragma unroll
                for (int t = 0; t != ST; ++t) {
#pragma unroll
                    for (int n = 0; n != NT; ++n) {
                        next[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i % PK][t], q[n][i],
                                                                           next[n][t], 0, 0, 0);
                    }
                }
                if (i + PK < NI) read_k(i + PK);
                if (i == NI - 1) {
#pragma unroll
                    for (int t = 0; t != PV; ++t) read_v(t);
                }
                constexpr int ALL = NT * ST * 2;
#pragma unroll
                for (int x = ALL * i / NI; x != ALL * (i + 1) / NI; ++x) {
                    int const n = x / (ST * 2), t = x / 2 % ST, r = x % 2;
                    float2_t  p;
                    p.x = exp2_fast(now[n][t][2 * r] * a.scale - ref[n]);
                    p.y = exp2_fast(now[n][t][2 * r + 1] * a.scale - ref[n]);
                    l[n] += p.x + p.y;
                    split_weights(p, high[n][t / 2].pair[2 * (t & 1) + r],
                                  low[n][t / 2].pair[2 * (t & 1) + r]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int t = 0; t != DT; ++t) {
#pragma unroll
                for (int ks = 0; ks != KT / 32; ++ks) {
#pragma unroll
                    for (int n = 0; n != NT; ++n) {
                        o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            vf[t % PV][ks].h, high[n][ks].h, o[n][t], 0, 0, 0);
                    }
#pragma unroll
                    for (int n = 0; n != NT; ++n) {
                        o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            vf[t % PV][ks].h, low[n][ks].h, o[n][t], 0, 0, 0);
                    }
                }
                if (t + PV < DT) read_v(t + PV);
                __builtin_amdgcn_sched_barrier(0);
            }
            // (last: a branch between the scores and the values would keep them from overlapping)
            if (edge(tile + 1, holes)) mask(tile + 1, next);
            raise_all(next);
        };
        // true: some row's result is not finite
        auto pass = [&](auto careful_) {
            constexpr bool CAREFUL = decltype(careful_)::value;
            if (CAREFUL) page0 = *page_at(position(0));
            if (tid == 0) sh.holes = sh.again = sh.bad = 0;
            __syncthreads();
            put_entry(0, page0);
            __syncthreads();
            load_to_lds_4(page_at(position(1)), lds_address(&sh.page[w * 64]));
            // beyond the last tile too: the waits count instructions
#pragma unroll
            for (int i = 0; i != NS - 1; ++i) {
                aim(i);
                load_tile(i);
            }
            aim(NS - 1);
            if (!CAREFUL) {
                // while they are on their way: who sees what
                if (prefix) prefix_limits<ROWS>(a, wk, sh.limit);
#pragma unroll
                for (int n = 0; n != NT; ++n) {
                    set_limit(a, wk, sh.limit, row[n]);
                    least = min(least, row[n].limit);
                    if (row[n].token >= 0) most = max(most, row[n].limit);
                }
#pragma unroll
                for (int i = 1; i != 16; i <<= 1) {
                    least = min(least, __shfl_xor(least, i));
                    most = max(most, __shfl_xor(most, i));
                }
                least = __builtin_amdgcn_readfirstlane(least);
                most = __builtin_amdgcn_readfirstlane(most);
            }
            wait_loads<2 * LPT*(NS - 2)>();
            __syncthreads();
            if (CAREFUL) clean(0);
            float4_t s[2][NT][ST];
            scores(0, s[0]);
            if (edge(0, sh.holes)) mask(0, s[0]);
            raise_all(s[0]);
            for (int tile = 0; tile < tiles; tile += NS) {
                step(tile, s, std::integral_constant<int, 0>(), careful_);
                if (tile + 1 < tiles) step(tile + 1, s, std::integral_constant<int, 1>(), careful_);
                if (tile + 2 < tiles) step(tile + 2, s, std::integral_constant<int, 2>(), careful_);
                if (tile + 3 < tiles) step(tile + 3, s, std::integral_constant<int, 3>(), careful_);
            }
            // nothing may still be on its way to LDS when it is used again, or the workgroup ends
            wait_loads<0>();
            if (!CAREFUL) {
                bool again = false;
#pragma unroll
                for (int n = 0; n != NT; ++n) {
#pragma unroll
                    for (int t = 0; t != DT; ++t) {
#pragma unroll
                        for (int r = 0; r != 4; ++r) {
                            again |= !finite(o[n][t][r]) && row[n].token >= 0;
                        }
                    }
                }
                if (again) sh.again = 1;
            }
            __syncthreads();
            return __builtin_amdgcn_readfirstlane(sh.again) != 0;
        };
        bool bad = false;
        if (pass(std::false_type())) {
            __syncthreads();
            start();
            pass(std::true_type());
            bad = sh.bad != 0;
        }
        if (bad) {
            for (int pos = lo; pos < hi; ++pos) {
                int const     pi = page_of(a, pos);
                int64_t const at = entry_of(a, wk.table[pi], pos - pi * a.page_size);
                if (at < 0) continue;
                T const* const value = reinterpret_cast<T const*>(vb + at * 2);
#pragma unroll
                for (int t = 0; t != DT; ++t) {
#pragma unroll
                    for (int r = 0; r != 4; ++r) {
                        int const   e = 16 * t + 4 * g + r;
                        float const x = float(value[!PAD || e < a.d ? e : 0]);
                        bool const  add = !finite(x) && (!PAD || e < a.d);
#pragma unroll
                        for (int n = 0; n != NT; ++n) {
                            o[n][t][r] += add && pos <= row[n].limit ? x : 0.0f;
                        }
                    }
                }
            }
        }
    } else if (prefix) {
        // the page table does not reach that far
        prefix_limits<ROWS>(a, wk, sh.limit);
#pragma unroll
        for (int n = 0; n != NT; ++n) set_limit(a, wk, sh.limit, row[n]);
    }
#pragma unroll
    for (int n = 0; n != NT; ++n) {
        // the four lanes of a column hold sums over different keys
        l[n] = column_sum(l[n]);
        l[n] = sum_of(a, wk, row[n].token < 0 ? -1 : row[n].limit, m[n], l[n]);
        if (row[n].token < 0) continue;
        // O^T: elements 16 t + 4 g + r of this lane's row
        if (wk.direct) {
            T* const dst = reinterpret_cast<T*>(a.out) + uint64_t(row[n].token) * a.out_stride +
                           uint64_t(row[n].head) * uint64_t(a.d);
            float const inv = weight_of(l[n]);
#pragma unroll
            for (int t = 0; t != DT; ++t) {
                int const e = 16 * t + 4 * g;
                half4_t   y;
#pragma unroll
                for (int r = 0; r != 4; ++r) y[r] = T(o[n][t][r] * inv);
                if (e < a.d) *reinterpret_cast<half4_t*>(dst + e) = y;
            }
        } else {
            int64_t const at = wk.part + (w * NT + n) * 16 + c;
#pragma unroll
            for (int t = 0; t != DT; ++t) {
                *reinterpret_cast<float4_t*>(a.part_o + at * D + 16 * t + 4 * g) = o[n][t];
            }
            if (g == 0) {
                a.part_ml[at * 2] = m[n];
                a.part_ml[at * 2 + 1] = l[n];
            }
        }
    }
}

__device__ inline int prefix_units_of(attention_dev_t const& a)
{
    return a.parts & 1 ? a.prefix_tiles * a.prefix_splits : 0;
}

template <typename T, int D, bool PAD>
__global__ __launch_bounds__(THREADS, D == 256 ? 2 : D == 128 && sizeof(T) == 4 ? 3 : 4) void attention_few_kernel(attention_dev_t a)
{
    __shared__ few_shared_t<T, D> sh;
    few_rows<T, D, PAD>(a, sh, int(blockIdx.x), prefix_units_of(a));
}

template <int D, int NT, bool PAD>
__global__ __launch_bounds__(THREADS, D == 256 ? 1 : 2) void attention_many_kernel(attention_dev_t a)
{
    __shared__ typename many_t<D, NT>::shared_t sh;
    many_rows<D, NT, PAD>(a, sh, int(blockIdx.x), prefix_units_of(a));
}

// The shared positions in tiles of many rows and the own ones in tiles of few, in one launch: the
// former are bound by instructions, the latter by memory, and two workgroups of either kind fit a
// compute unit (64 tokens over a prefix of 8192: 26 + 32 us one after the other, 51 us together; 32
// tokens, 32 heads of keys: 13 + 50 us, 61 us).  The former come first; in turn with the latter
// 64 tokens took 56 us.
template <int D, int NT, bool PAD>
__global__ __launch_bounds__(THREADS, 2) void attention_mixed_kernel(attention_dev_t a)
{
    __shared__ union {
        typename many_t<D, NT>::shared_t many;
        few_shared_t<_Float16, D>        few;
    } sh;
    int const units = a.prefix_tiles * a.prefix_splits, own = int(blockIdx.x) - units * a.h_kv;
    if (own < 0) {
        many_rows<D, NT, PAD>(a, sh.many, int(blockIdx.x), units);
    } else {
        few_rows<_Float16, D, PAD>(a, sh.few, own, 0);
    }
}


// The references and sums of a row's cuts decide their weights, then the cuts' O are added in a
// fixed order: TEAMS teams of sixteen lanes per row take them in turn: four teams where many cuts are
// to be joined (2048 rows of 17: 8.4 us, 10.2 us with one), one where many rows are (26784 rows of
// two: 10.6 us, 23.1 us with four).  Bound by the partial results' bytes, 17 and 41 MB.
template <typename T, int D, int TEAMS>
__global__ __launch_bounds__(THREADS) void attention_join_kernel(attention_dev_t a)
{
    constexpr int LANES = 16, PER = D / LANES;
    int const     lane = int(threadIdx.x) % LANES;
    int const     team = int(threadIdx.x) / LANES % TEAMS;
    int const     heads = a.h_kv * a.group;
    int const     id = int(blockIdx.x) * (THREADS / LANES / TEAMS) +
                   int(threadIdx.x) / (LANES * TEAMS);
    int const     token = id / heads, head = id - token * heads;
    if (token >= a.n_tokens) return;
    int const kvh = head / a.group, hg = head - kvh * a.group;
    int const prow = token * a.group + hg;
    int4 const meta = a.part_meta[prow];
    if (token < a.offsets[0] || token >= a.offsets[a.n_seqs]) return;
    if (meta.y < 0) return;  // stored already
    // both stay inside the workspace whatever the device arrays held
    int const whole = min(meta.y, a.own_slots), srow = min(max(meta.w, 0), a.own_rows - 1);
    int const pslot = a.prefix_splits ? prow / a.prefix_rows : 0;
    int const parts = a.prefix_splits + whole + (meta.z >= 0);
    auto      place = [&](int i) -> int64_t {
        if (i < a.prefix_splits) {
            return (int64_t(pslot + i * a.prefix_tiles) * a.h_kv + kvh) * a.prefix_rows +
                   prow % a.prefix_rows;
        }
        i -= a.prefix_splits;
        int const slot = min(max(i < whole ? meta.x + i : meta.z, 0), a.own_slots - 1);
        return a.own_base + (int64_t(slot) * a.h_kv + kvh) * a.own_rows + srow;
    };
    float top = NEG_INF;
    for (int i = lane; i < parts; i += LANES) top = fmaxf(top, a.part_ml[place(i) * 2]);
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    float4_t y[PER / 4];
    float    sum = 0;
#pragma unroll
    for (int e = 0; e != PER / 4; ++e) y[e] = float4_t{0, 0, 0, 0};
    int const group0 = int(threadIdx.x) & 63 & ~(LANES - 1);
    for (int i0 = 0; i0 < parts; i0 += LANES) {
        // lane i: the place and the weight of cut i0 + i; none without keys for this row, or with
        // scores of -inf only beside a cut of others
        bool const    in = i0 + lane < parts;
        int64_t const at = in ? place(i0 + lane) : 0;
        float const   mi = in ? a.part_ml[at * 2] : NEG_INF;
        float const   li = in ? a.part_ml[at * 2 + 1] : 0.0f;
        float const   f = mi == NEG_INF ? 0.0f : exp2_fast(mi - top);
        sum += mi != NEG_INF ? li * f : li < 0.0f && top != NEG_INF ? 0.0f : li;
        constexpr int U = 4;  // cuts in flight
        int const     n = min(parts - i0, LANES);
        for (int i = team; i < n; i += U * TEAMS) {
            float4_t x[U][PER / 4];
            float    fi[U];
#pragma unroll
            for (int u = 0; u != U; ++u) {
                int const     which = group0 + min(i + u * TEAMS, n - 1);
                int64_t const p = __shfl(at, which);
                float const   fu = __shfl(f, which);
                fi[u] = i + u * TEAMS < n ? fu : 0.0f;
                float4_t const* const src =
                    reinterpret_cast<float4_t const*>(a.part_o + p * D + lane * PER);
#pragma unroll
                for (int e = 0; e != PER / 4; ++e) {
                    x[u][e] = i + u * TEAMS < n ? src[e] : float4_t{0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int u = 0; u != U; ++u) {
#pragma unroll
                for (int e = 0; e != PER / 4; ++e) {
#pragma unroll
                    for (int j = 0; j != 4; ++j) y[e][j] += scaled(x[u][e][j], fi[u]);
                }
            }
        }
    }
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) sum += __shfl_xor(sum, o);
#pragma unroll
    for (int o = LANES; o < LANES * TEAMS; o <<= 1) {
#pragma unroll
        for (int e = 0; e != PER / 4; ++e) {
#pragma unroll
            for (int i = 0; i != 4; ++i) y[e][i] += __shfl_xor(y[e][i], o);
        }
    }
    if (team != 0) return;
    T* const    dst = reinterpret_cast<T*>(a.out) + uint64_t(token) * a.out_stride +
                   uint64_t(head) * uint64_t(a.d) + lane * PER;
    float const inv = weight_of(sum);
    // in vectors of at most 16 bytes; d is a multiple of 8
    constexpr int V = PER < 16 / int(sizeof(T)) ? PER : 16 / int(sizeof(T));
    typedef T     vec_t __attribute__((ext_vector_type(V)));
#pragma unroll
    for (int e = 0; e != PER; e += V) {
        vec_t z;
#pragma unroll
        for (int i = 0; i != V; ++i) {
            z[i] = T(y[(e + i) / 4][(e + i) % 4] * inv);
        }
        if (lane * PER + e < a.d) *reinterpret_cast<vec_t*>(dst + e) = z;
    }
}

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }

template <typename T, int D>
void launch_rows(attention_dev_t a, int parts, int rows, hipStream_t stream)
{
    a.parts = parts;
    uint64_t const units = (parts & 1 ? uint64_t(a.prefix_tiles) * a.prefix_splits : 0) +
                           (parts & 2 ? a.own_slots : 0);
    uint32_t const grid = uint32_t(units * a.h_kv);
    if constexpr (sizeof(T) == 2) {
        if constexpr (D <= 128) {
            if (rows == many_t<D, 2>::ROWS) {
                if (a.d == D) {
                    attention_many_kernel<D, 2, false><<<grid, THREADS, 0, stream>>>(a);
                } else {
                    attention_many_kernel<D, 2, true><<<grid, THREADS, 0, stream>>>(a);
                }
                return;
            }
        }
        if (rows == many_t<D, 1>::ROWS) {
            if (a.d == D) {
                attention_many_kernel<D, 1, false><<<grid, THREADS, 0, stream>>>(a);
            } else {
                attention_many_kernel<D, 1, true><<<grid, THREADS, 0, stream>>>(a);
            }
            return;
        }
    }
    if (a.d == D) {
        attention_few_kernel<T, D, false><<<grid, THREADS, 0, stream>>>(a);
    } else {
        attention_few_kernel<T, D, true><<<grid, THREADS, 0, stream>>>(a);
    }
}

// Whether one launch takes both kinds of tiles.
bool mixed(bool f16, int d, uint64_t prefix_splits, uint64_t prefix_rows, uint64_t own_rows)
{
    return f16 && d <= 128 && prefix_splits > 0 && prefix_rows > FEW && own_rows == FEW;
}

template <typename T, int D>
bool launch_mixed(attention_dev_t const& a, hipStream_t stream)
{
    if constexpr (sizeof(T) == 2 && D <= 128) {
        if (!mixed(true, a.d, uint64_t(a.prefix_splits), uint64_t(a.prefix_rows),
                   uint64_t(a.own_rows))) {
            return false;
        }
        uint32_t const grid = uint32_t((a.prefix_tiles * a.prefix_splits + a.own_slots) * a.h_kv);
        if (a.prefix_rows == many_t<D, 2>::ROWS) {
            if (a.d == D) {
                attention_mixed_kernel<D, 2, false><<<grid, THREADS, 0, stream>>>(a);
            } else {
                attention_mixed_kernel<D, 2, true><<<grid, THREADS, 0, stream>>>(a);
            }
            return true;
        }
        if (a.d == D) {
            attention_mixed_kernel<D, 1, false><<<grid, THREADS, 0, stream>>>(a);
        } else {
            attention_mixed_kernel<D, 1, true><<<grid, THREADS, 0, stream>>>(a);
        }
        return true;
    }
    return false;
}

template <typename T, int D>
void launch_dim(attention_dev_t const& a, hipStream_t stream)
{
    if (a.prefix_splits != 0 && a.prefix_rows == a.own_rows) {
        launch_rows<T, D>(a, 3, a.own_rows, stream);
    } else if (!launch_mixed<T, D>(a, stream)) {
        if (a.prefix_splits != 0) launch_rows<T, D>(a, 1, a.prefix_rows, stream);
        launch_rows<T, D>(a, 2, a.own_rows, stream);
    }
    if (a.prefix_splits != 0 || a.shares != 0) {
        uint64_t const rows = uint64_t(a.n_tokens) * a.h_kv * a.group;
        if (a.prefix_splits >= 8 || rows <= 4096) {
            attention_join_kernel<T, D, 4>
                <<<uint32_t((rows + 3) / 4), THREADS, 0, stream>>>(a);
        } else {
            attention_join_kernel<T, D, 1>
                <<<uint32_t((rows + 15) / 16), THREADS, 0, stream>>>(a);
        }
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

// Rows per tile for `rows` rows that read the same keys.  32 rows of 256 elements per wavefront
// would not fit its registers.
uint32_t tile_rows(es_km_kv_cache_t const& c, uint64_t rows)
{
    if (c.dtype != ES_KM_F16 || rows <= FEW) return FEW;
    return rows <= 64 || c.head_dim > 128 ? 64 : 128;
}

}  // namespace

attention_plan_t plan_attention(es_km_kv_cache_t const& c, int n_seqs, int n_tokens,
                                uint64_t shared)
{
    attention_plan_t p;
    if (n_seqs == 0 || n_tokens == 0) return p;
    uint64_t const kv = uint64_t(c.n_kv_heads), group = uint64_t(c.n_heads / c.n_kv_heads);
    uint64_t const rows = uint64_t(n_tokens) * group;
    // a launch holds less than 2^32 threads; the join takes up to 64 of them for a row
    auto const too_many = []() {
        throw ir_error("prefix_attention: more rows (tokens times heads) than a launch holds");
    };
    if (rows * kv >= (1ull << 32) / 64) too_many();
    uint64_t const seqs = uint64_t(std::min(n_seqs, n_tokens));  // that have tokens, at most
    uint64_t       part_rows = 0;
    p.own_rows = tile_rows(c, rows / seqs);
    // A prefix of its own pays where rows of several sequences fill a tile together.  Sequences
    // that fill tiles by themselves read it through their own tables.
    if (p.own_rows == (c.head_dim > 128 ? 64 : 128)) shared = 0;
    p.shared = uint32_t(shared);
    if (shared > 0) {
        p.prefix_rows = tile_rows(c, rows);
        uint64_t const tiles = (rows + p.prefix_rows - 1) / p.prefix_rows;
        // Workgroups of few rows run four to a compute unit, and those of many are slowed by a
        // second one (64 tokens, with the own positions: 50.5 us with 256, 56.0 with 384, 66.7 and
        // 3 us more to join with 512).  Measured at head_dim 128; at 256 two and one fit.
        uint64_t const slots = p.prefix_rows == FEW ? 1024 : 256;
        uint64_t const want = (slots + tiles * kv - 1) / (tiles * kv);
        // no cuts below 256 positions; below 128 for a single tile of few rows, where the time is a
        // wavefront's steps one after the other (1 token, 512 shared: 7.2 us, 8.6 us in cuts of
        // 256; f32, 15 tiles, 777 shared: no faster, and the join 1 us slower)
        uint64_t const cut = p.prefix_rows == FEW && tiles == 1 ? 128 : 256;
        uint64_t const most = (shared + cut - 1) / cut;
        uint64_t const splits = std::max<uint64_t>(1, std::min(want, most));
        uint64_t const chunk = ((shared + splits - 1) / splits + 63) / 64 * 64;
        p.prefix_tiles = uint32_t(tiles);
        p.prefix_chunk = uint32_t(chunk);
        p.prefix_splits = uint32_t((shared + chunk - 1) / chunk);
        part_rows = tiles * p.prefix_splits * kv * p.prefix_rows;
    }
    p.own_base = part_rows;
    // sum over the sequences with tokens of ceil(tokens * group / own_rows)
    uint64_t tiles = seqs + (rows - seqs) / p.own_rows;
    // where a tile holds at least two groups, a sequence's first token adds no second tile
    if (2 * group <= p.own_rows + 1) {
        tiles = std::min(tiles, seqs + (rows - seqs * group) / (p.own_rows - group + 1));
    }
    // as many as run at once, two or four to a compute unit (64 tokens in one launch with the prefix:
    // 55.7 us with 1024, 50.5 us with 512; head_dim 128, at 256 one or two fit)
    bool const     two = p.own_rows != FEW || mixed(c.dtype == ES_KM_F16, c.head_dim, p.prefix_splits,
                                                p.prefix_rows, p.own_rows);
    uint64_t const aim = two ? 512 : 1024;
    p.shares = tiles * kv >= 4 * aim ? 0 : uint32_t(std::max<uint64_t>(1, aim / kv));
    p.own_slots = uint32_t(tiles + p.shares);
    // room for 1024 pieces of few rows either way: a batch for which both kinds of workgroups share a
    // launch does not need less than a smaller one
    uint64_t const room = p.own_rows == FEW ? std::max<uint64_t>(p.shares, 1024 / kv) : p.shares;
    // nothing is cut: each tile's result goes straight to the output
    bool const joined = p.prefix_splits != 0 || p.shares != 0;
    if (joined) part_rows += (tiles + room) * kv * p.own_rows;
    uint64_t const units = uint64_t(p.prefix_tiles) * p.prefix_splits + p.own_slots;
    if (units * kv >= (1ull << 32) / THREADS) too_many();
    p.part_rows = part_rows;
    p.workspace_bytes = joined ? up256(part_rows * uint64_t(padded_dim(c.head_dim)) * 4) +
                                     up256(part_rows * 8) + up256(rows * 16)
                               : 0;
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
    a.shared = int(p.shared);
    a.scale = g.scale == 0.0f ? 1.0f : __builtin_fabsf(g.scale) * 1.44269504088896340736f;
    a.q_sign = g.scale == 0.0f ? 0.0f : g.scale < 0.0f ? -1.0f : 1.0f;
    int shift = 0;
    while ((1 << shift) < a.page_size) ++shift;
    // (2^(30+s) + e) / page_size with e < page_size <= 2^s: exact for positions below 2^30
    a.page_shift = uint32_t(30 + shift);
    a.page_magic = uint32_t(((1ull << a.page_shift) + uint64_t(a.page_size) - 1) /
                            uint64_t(a.page_size));
    a.prefix_tiles = int(p.prefix_tiles);
    a.prefix_splits = int(p.prefix_splits);
    a.prefix_chunk = int(p.prefix_chunk);
    a.prefix_rows = int(p.prefix_rows);
    a.shares = int(p.shares);
    a.own_slots = int(p.own_slots);
    // the units of the whole batch are counted in 32 bits
    uint64_t const reach = uint64_t(a.max_pages) * uint64_t(a.page_size) / 16 + 2;
    a.grain = 1;
    while (uint64_t(p.own_slots) * (reach / uint64_t(a.grain) + 1) >= (1ull << 30)) a.grain *= 2;
    a.own_rows = int(p.own_rows);
    a.own_base = int64_t(p.own_base);
    a.direct = p.prefix_splits == 0;
    a.parts = 0;
    a.part_o = a.part_ml = nullptr;
    a.part_meta = nullptr;
    if (p.workspace_bytes != 0) {
        char* const    ws = static_cast<char*>(workspace);
        uint64_t const o_bytes = up256(p.part_rows * uint64_t(padded_dim(a.d)) * 4);
        a.part_o = reinterpret_cast<float*>(ws);
        a.part_ml = reinterpret_cast<float*>(ws + o_bytes);
        a.part_meta = reinterpret_cast<int4*>(ws + o_bytes + up256(p.part_rows * 8));
    }
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
