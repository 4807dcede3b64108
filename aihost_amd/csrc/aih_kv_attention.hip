// aih_kv_attention.hip -- grouped-query attention over the paged 8-bit KV cache
// (include/aihost_hip.h), for single tokens, a few tokens and prompts.
//
// Products.  S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16.  The
// codes (integers up to 127, or e4m3 numbers) are exact in fp16; q and the
// probabilities are split into two fp16 values of 22 bits together, so a
// product is two MFMAs and the result is good to fp32: rounding either to one
// fp16 would leave about 1e-4.  The scales stay out of the products: a lane's 16
// scores of a 64-key tile belong to one group of 16 tokens, hence to one block,
// so the key scale is one factor of the lane and the value scale one factor of
// its probabilities.
//
// Layouts (lane l, c = l % 16, g = l / 16): A[i][k] lane i + 16 (k/8) element
// k % 8, B[k][j] lane j + 16 (k/8) element k % 8, D[i][j] lane j + 16 (i/4)
// register i % 4.  A tile is four groups of 16 tokens.
//   S^T product t = 0..3: row i = 4a + b of A is key 16a + 4t + b of the tile,
//     so that D gives lane (c, g) the scores of query c with keys 16g + 4t + b.
//     The 16 bytes that lane (c, g) loads of a key are dimensions 64 C + 16 g ..
//     of it; their halves are the k-slots of two MFMAs, and Q is laid out alike.
//   O^T product (16 dimensions dt, half m): k-slot 8g + j is key 16g + 8m + j,
//     so P is the lane's own registers 8m + j and V the halves of the 16
//     bytes (one dimension, 16 tokens) that lane (c, g) loads from group g.
// The cache's layout is made for these loads: no byte moves between lanes.
//
// Softmax.  In base 2, with the running normalizer, sum and accumulator of each
// query in the registers of the four lanes that hold it.  A weight is the
// probability times the value scale, so the normalizer M is taken over both:
// with t the score and v the exponent of the scale, M is max(t + v) over the keys seen
// so far, rounded up.  A lane's exponentials are p = 2^(t + e - M), the weight
// p vs 2^(15 - e) is at most 2^15, the accumulator holds O 2^15 2^-M and the
// sum 2^-M of the probabilities' (each p 2^-e).  M and e being integers,
// rescaling is exact, and rare.  e is v, but held within 60 of the largest v that
// the query has met and above -100: the sum must not lose the probability of a
// block of zeros (no scale, so v is below all) or of tiny values, whose p would
// underflow.  Into M goes v itself, held above e - 100 and -100: that bounds p
// and the sum by 2^100 a key, and costs nothing where the scales that a query sees
// are above 2^-100 and within 2^160 of each other.  Blocks that a query does not see
// enter neither.  A weight is good to 2^-40 of the largest; a block whose
// visible codes are all 0 counts for its scale there, as 0 was within half a step of it.
//
// Work.  Rows are (token, head of the group) pairs of one KV head, token-major,
// in tiles of R; each tile's keys are split into parts where the tiles alone
// would leave CUs idle or where one request is much longer than the others.
// Every workgroup finds its part from the lengths on the device (find_item, and
// layout_kernel before it for many requests), so a captured launch follows the requests
// as they grow.

#include "aih_kv.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

using aih_kv::f4;
using aih_kv::u4;
using aih_kv::wave_add;
using aih_kv::wave_scan;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kNone = 0xFFFFFFFFu;   // no group of tokens there

struct Args {
    const uint8_t *k, *v;
    const float *ks, *vs;
    const float *Q;
    float *O;
    int64_t ldq, ldo;
    const int32_t *starts, *lens, *tables;
    const float *slopes;
    const int32_t *prefix;
    float *part, *part_ml;      // partial outputs (rows of D floats) and their (maximum, sum)
    int32_t *layout;            // where the requests' items begin (layout_kernel), or null
    int32_t rows, heads, group, n_seqs, width, n_blocks, shift, window;
    int32_t target, least;      // workgroups wanted; the fewest tiles of a part
    int32_t n_part;             // partial tiles that fit the scratch
    float scale, cap, inv_group;
};

// ---------------------------------------------------------------- which part is mine
struct Seq {
    int32_t start, n, len;   // first query row, query rows, cached tokens
};

__device__ __forceinline__ Seq seq_of(const Args &a, int s)
{
    const int32_t b = min(max(a.starts[s], 0), a.rows), e = min(max(a.starts[s + 1], b), a.rows);
    const int64_t most = (int64_t)a.width << a.shift;
    return Seq{b, e - b, (int32_t)min<int64_t>(max(a.lens[s], 0), most)};
}

// Row tiles of R rows of a request, and the key tiles that the longest of them spans.
template <int R>
__device__ __forceinline__ int32_t row_tiles(const Args &a, const Seq &q)
{
    return (int32_t)(((uint32_t)q.n * (uint32_t)a.group + R - 1) / R);
}
__device__ __forceinline__ int32_t key_tiles(const Args &a, const Seq &q)
{
    const int32_t lo = a.window > 0 ? (int32_t)max<int64_t>(0, (int64_t)q.len - q.n + 1 - a.window) : 0;
    return (int32_t)(((int64_t)q.len + 63) / 64) - lo / 64;
}

struct Item {
    int32_t seq, tile, split, n_split, part;   // part: index of the tile's first partial (n_split > 1)
    Seq q;
    bool ok;
};

// A lane's request: its row tiles and the key tiles of the longest of them.
struct Load {
    Seq q;
    int32_t tiles, keys;
};

template <int R>
__device__ __forceinline__ Load load_of(const Args &a, int s)
{
    Load l{{0, 0, 0}, 0, 0};
    if (s < a.n_seqs) {
        l.q = seq_of(a, s);
        l.tiles = row_tiles<R>(a, l.q);
        l.keys = max(key_tiles(a, l.q), 0);
    }
    return l;
}

// Row tiles times key tiles (or parts), rounded by itself: every kernel of a call derives the same lengths from the same sums,
// and a product that the compiler fused into its sum in one of them would not be the same beyond 2^24.
__device__ __forceinline__ float product(int32_t tiles, int32_t n)
{
#pragma clang fp contract(off)
    return (float)tiles * (float)n;
}

// The longest part, in key tiles: the whole work over the wanted workgroups, so
// that all parts are about as long whatever the requests' lengths; longer where
// rounding up would make a few parts more than that number, which would run
// alone after the others.  parts(len): how many there would be.  (The sums are
// floats: the same in every wave, and they only weigh the parts.)
template <typename Parts>
__device__ __forceinline__ int32_t part_length(const Args &a, int32_t heads, float work, float tiles, Parts parts)
{
    float want = (float)a.target / (float)heads;
    // about as many tiles as workgroups wanted, and of different lengths: shorter parts even them out (64 requests of
    // 512 to 7804 tokens, 512 wanted: 94.7 -> 87.3 us)
    if (tiles > 0.75f * want) want *= 2.0f;
    int32_t len = max(a.least, (int32_t)ceilf(work / want));
    if (tiles < want) {
        for (int i = 0; i < 4; ++i) {
            const float n = parts(len);
            if (n <= want) break;
            len = max(len + 1, (int32_t)((float)len * n / want));
        }
    }
    return len;
}
constexpr int32_t kUnsplit = 1 << 30;   // the length where nothing is split
constexpr int kScan = 256;              // requests that every wave looks through for itself

// Item k of a request (its tiles from the last, longest one on, split by split;
// `joined`: its tiles), whose parts begin at `parts`.
__device__ __forceinline__ Item item_of(const Load &l, int32_t seq, int32_t k, int32_t n_split, int32_t parts, bool joined)
{
    Item it;
    it.n_split = n_split;
    it.tile = joined ? k : l.tiles - 1 - k / n_split;
    it.split = joined ? 0 : k % n_split;
    it.seq = seq;
    it.part = parts + it.tile * n_split;
    it.q = l.q;
    it.ok = true;
    return it;
}

// Item `idx` of one KV head: parts are numbered request by request; with
// `joined`, the tiles that are split instead.  Every wave of the launch runs this
// with all lanes.  Up to kScan requests it adds up their lengths itself; more
// have been laid out by layout_kernel, and two rounds of loads find the one.
template <int R>
__device__ __forceinline__ Item find_item(const Args &a, int32_t idx, int32_t heads, bool joined)
{
    const int lane = threadIdx.x & 63;
    Item none{};
    none.ok = false;
    const Load own = load_of<R>(a, lane);   // (before the branch: it is on the way of every small call)
    if (a.layout) {
        const int32_t n = a.n_seqs + 1;
        const int32_t *first = a.layout + 4 + (joined ? 2 * n : 0), *parts = a.layout + 4 + n;
        int32_t base = 0;
#pragma unroll
        for (int step = 64; step; step /= 64) {
            const int32_t s = base + lane * step;
            const bool past = s >= n || first[min(s, n - 1)] > idx;
            base += (63 - __builtin_clzll(~__ballot(past) | 1)) * step;   // the last that is not
        }
        const int32_t seq = base;
        if (seq >= a.n_seqs) return none;
        const Load l = load_of<R>(a, seq);
        const int32_t len = a.layout[0], n_split = max(1, (l.keys + len - 1) / len), k = idx - first[seq];
        if (k < 0 || k >= (joined ? l.tiles : l.tiles * n_split)) return none;
        return item_of(l, seq, k, n_split, parts[seq], joined);
    }
    int32_t len = kUnsplit;
    if (a.n_part) {
        float work = product(own.tiles, own.keys), tiles = (float)own.tiles;
        for (int base = 64; base < a.n_seqs; base += 64) {
            const Load l = load_of<R>(a, base + lane);
            work += product(l.tiles, l.keys);
            tiles += (float)l.tiles;
        }
        len = part_length(a, heads, wave_add(work), wave_add(tiles), [&](int32_t len) {
            float n = product(own.tiles, (own.keys + len - 1) / len);
            for (int base = 64; base < a.n_seqs; base += 64) {
                const Load l = load_of<R>(a, base + lane);
                n += product(l.tiles, (l.keys + len - 1) / len);
            }
            return wave_add(n);
        });
    }
    int32_t before = 0, parts = 0;
    for (int base = 0; base < a.n_seqs; base += 64) {
        const Load l = base ? load_of<R>(a, base + lane) : own;
        const int32_t n_split = max(1, (l.keys + len - 1) / len), part_own = n_split > 1 ? l.tiles * n_split : 0;
        const int32_t items = !joined ? l.tiles * n_split : n_split > 1 ? l.tiles : 0;
        const int32_t upto = wave_scan(items), part_upto = wave_scan(part_own);
        const unsigned long long past = __ballot(before + upto > idx);
        if (past) {
            const int at = __builtin_ctzll(past);
            auto there = [&](int32_t v) { return __builtin_amdgcn_readlane(v, at); };
            const Load mine{{there(l.q.start), there(l.q.n), there(l.q.len)}, there(l.tiles), there(l.keys)};
            return item_of(mine, base + at, idx - (before + there(upto - items)), there(n_split),
                           parts + there(part_upto - part_own), joined);
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        parts += __builtin_amdgcn_readlane(part_upto, 63);
    }
    return none;
}

// The layout of more than kScan requests, by one workgroup, four of them a
// thread: the longest part, and the sums before every request (and over all) of
// items, of parts and of tiles that are split.  Without it every workgroup would go
// over all requests: one token each of 130 requests of 300 28.4 us without it, 33.1
// with it, of 256 50.6 / 55.1 (of 2000 tokens 201 / 203), of 1000 234 / 170, of 4000 1728 / 644.
template <int R>
__global__ void __launch_bounds__(1024)
layout_kernel(Args a, int32_t heads)
{
    static_assert(aih_kv::kMaxSeqs <= 4 * 1024, "");
    __shared__ float fs[16];
    __shared__ int32_t is[3][16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    auto add = [&](float v) {
        v = wave_add(v);
        __syncthreads();
        if (lane == 0) fs[w] = v;
        __syncthreads();
        float all = 0.f;
        for (int i = 0; i < 16; ++i) all += fs[i];
        return all;
    };
    Load l[4];
    float work = 0.f, tiles = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        l[i] = load_of<R>(a, 4 * tid + i);
        work += product(l[i].tiles, l[i].keys);
        tiles += (float)l[i].tiles;
    }
    const int32_t len = !a.n_part ? kUnsplit : part_length(a, heads, add(work), add(tiles), [&](int32_t len) {
        float n = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) n += product(l[i].tiles, (l[i].keys + len - 1) / len);
        return add(n);
    });
    int32_t own[4][3], sum[3] = {0, 0, 0}, before[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int32_t n_split = max(1, (l[i].keys + len - 1) / len);
        own[i][0] = l[i].tiles * n_split;
        own[i][1] = n_split > 1 ? l[i].tiles * n_split : 0;
        own[i][2] = n_split > 1 ? l[i].tiles : 0;
#pragma unroll
        for (int e = 0; e < 3; ++e) sum[e] += own[i][e];
    }
#pragma unroll
    for (int e = 0; e < 3; ++e) {
        const int32_t upto = wave_scan(sum[e]);
        if (lane == 63) is[e][w] = upto;
        before[e] = upto - sum[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 3; ++e)
        for (int i = 0; i < w; ++i) before[e] += is[e][i];
    if (tid == 0) a.layout[0] = len;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int s = 4 * tid + i;
#pragma unroll
        for (int e = 0; e < 3; ++e) {
            if (s < a.n_seqs) a.layout[4 + e * (a.n_seqs + 1) + s] = before[e];
            before[e] += own[i][e];
            if (s + 1 == a.n_seqs) a.layout[4 + e * (a.n_seqs + 1) + s + 1] = before[e];
        }
    }
}

// What a request's queries see: position p the keys max(0, p - window + 1) ..
// min(max(p + 1, prefix), len) - 1.
struct View {
    int32_t prefix, len, window;
    __device__ __forceinline__ int32_t lo(int32_t p) const
    {
        return window > 0 ? (int32_t)max<int64_t>(0, (int64_t)p - window + 1) : 0;
    }
    __device__ __forceinline__ int32_t hi(int32_t p) const { return min(max(p + 1, prefix), len); }
};

__device__ __forceinline__ View view_of(const Args &a, const Item &it)
{
    return View{a.prefix ? a.prefix[it.seq] : 0, it.q.len, a.window};
}

// The key tiles of a row tile, and of its part `split`: an equal share each.
struct Range {
    int32_t lo, hi;
};

template <int R>
__device__ __forceinline__ Range tile_keys(const Args &a, const Item &it, const View &v)
{
    const uint32_t f0 = (uint32_t)it.tile * R;
    const int32_t base = it.q.len - it.q.n;
    const int32_t p0 = base + (int32_t)(f0 / (uint32_t)a.group);
    const int32_t p1 = base + min((int32_t)((f0 + R - 1) / (uint32_t)a.group), it.q.n - 1);
    const int32_t end = v.hi(p1), lo = v.lo(p0);
    return Range{lo / 64, end <= lo ? lo / 64 : (int32_t)(((int64_t)end + 63) / 64)};
}

__device__ __forceinline__ Range part_of(const Range &r, int32_t split, int32_t n_split)
{
    const int32_t per = (r.hi - r.lo + n_split - 1) / n_split;
    const int32_t lo = min(r.lo + split * per, r.hi);
    return Range{lo, min(lo + per, r.hi)};
}

// ---------------------------------------------------------------- codes to fp16
template <int FMT>
__device__ __forceinline__ h8 to_half(uint32_t w0, uint32_t w1);

// A code + 128 below an exponent byte is 1024 + 128 + code; the subtraction is exact.
template <>
__device__ __forceinline__ h8 to_half<AIH_KV_INT8>(uint32_t w0, uint32_t w1)
{
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    constexpr uint32_t e = 0x64646464u;
    const u4 b = {__builtin_amdgcn_perm(w0, e, 0x00050004u), __builtin_amdgcn_perm(w0, e, 0x00070006u),
                  __builtin_amdgcn_perm(w1, e, 0x00050004u), __builtin_amdgcn_perm(w1, e, 0x00070006u)};
    return __builtin_bit_cast(h8, b) - (_Float16)1152.0f;
}

template <>
__device__ __forceinline__ h8 to_half<AIH_KV_E4M3>(uint32_t w0, uint32_t w1)
{
    const u4 b = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true))};
    return __builtin_bit_cast(h8, b);
}

// x0, x1 = hi + lo, two pairs of fp16
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo)
{
    const f2 x = {x0, x1};
    const h2 h = __builtin_convertvector(x, h2);
    const f2 r = {fmaf(-(float)h[0], 1.0f, x0), fmaf(-(float)h[1], 1.0f, x1)};   // one v_fma_mix each
    const h2 l = __builtin_convertvector(r, h2);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Over the four lanes c, c + 16, c + 32, c + 48 of a query.
__device__ __forceinline__ float over4_max(float v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float over4_sum(float v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// tanh to fp32: the continued fraction x / (1 + x^2 / (3 + x^2 / (5 + ...)))
// cut after the fifth level below 0.7 (relative error under 3e-9 there), 1 - 2 / (e^2x + 1) above.
__device__ __forceinline__ float tanh_small(float x)
{
    const float y = x * x;
    const float n = fmaf(fmaf(y, 1.0f, 105.0f), y, 945.0f), d = fmaf(fmaf(y, 15.0f, 420.0f), y, 945.0f);
    return x * n * __builtin_amdgcn_rcpf(d);
}
__device__ __forceinline__ float tanh_any(float x)
{
    const float a = fabsf(x);
    const float e = __builtin_amdgcn_exp2f(2.0f * kLog2e * a);
    const float t = fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
    return a < 0.7f ? tanh_small(x) : copysignf(t, x);
}

// ---------------------------------------------------------------- a query's state
constexpr float kNoExp = -1000.0f;   // no value scale seen yet

// x 2^d for the difference d of two normalizers (-inf, or NaN for two of those: 0)
__device__ __forceinline__ float times2(float x, float d) { return ldexpf(x, (int)fmaxf(d, -1000.0f)); }

// 16 queries of a wave: lane (c, g) holds query c's.
template <int D>
struct State {
    f4 o[D / 16];   // rows 16 dt + 4 g + i of O^T, times 2^(15 - M)
    float m, l;     // M; this lane's part of the sum, times 2^-M
    float e;        // the largest exponent of a value scale seen
    __device__ __forceinline__ void init()
    {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        l = 0.f;
        e = kNoExp;
    }
    __device__ __forceinline__ void times(float f)
    {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i] *= f;
    }
};

// The query of a column: its position (kNobody for a column past the request's
// rows, which is computed and not stored) and the slope of its head, times log2 e.
constexpr int32_t kNobody = -0x40000000;
struct Col {
    int32_t pos;
    float slope;
};

// Row f0 + x of a request (f0 the first of a tile, x < 128): its token and its
// head within the group.  The quotient of the remainder is taken in floats, exact
// below 2^21: it lies half a step or more from an integer.
struct Place {
    int32_t token, head;
};

__device__ __forceinline__ Place place_of(const Args &a, uint32_t f0, uint32_t x)
{
    const uint32_t t0 = f0 / (uint32_t)a.group, r = f0 - t0 * (uint32_t)a.group + x;
    const uint32_t t = (uint32_t)(((float)r + 0.5f) * a.inv_group);
    return Place{(int32_t)(t0 + t), (int32_t)(r - t * (uint32_t)a.group)};
}

// Where the row's values lie: its query row, -1 for none, and its head.
__device__ __forceinline__ Place row_of(const Args &a, const Item &it, int32_t kvh, uint32_t f0, uint32_t x)
{
    const Place p = place_of(a, f0, x);
    return Place{p.token < it.q.n ? it.q.start + p.token : -1, kvh * a.group + p.head};
}

__device__ __forceinline__ Col column(const Args &a, const Item &it, const Place &row)
{
    Col c{kNobody, 0.f};
    if (row.token >= 0) {
        c.pos = it.q.len - it.q.n + (row.token - it.q.start);
        if (a.slopes) c.slope = a.slopes[row.head] * kLog2e;
    }
    return c;
}

// The key tiles of which the queries of 16 columns all see all keys: all_lo .. all_hi - 1.
struct Sight {
    int32_t all_lo, all_hi;
};

__device__ __forceinline__ Sight sight_of(const View &v, const Col &c)
{
    const bool is = c.pos != kNobody;
    int32_t lo = is ? v.lo(c.pos) : 0, hi = is ? v.hi(c.pos) : 0x7FFFFFFF;   // the largest, the smallest
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        lo = max(lo, __shfl_xor(lo, d));
        hi = min(hi, __shfl_xor(hi, d));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    // hi may be 0 or less for a query that sees nothing
    return Sight{(int32_t)(((uint32_t)lo + 63) / 64), hi > 0 ? hi / 64 : 0};
}

// Q of a column: its loads, and its values split; split() returns the factor
// that undoes the split's power of two.
template <int D>
struct QRow {
    f4 x[D / 64][4];
    __device__ __forceinline__ void load(const Args &a, const Place &c, int g)
    {
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[k][i] = f4{0.f, 0.f, 0.f, 0.f};
                if (c.token >= 0)
                    x[k][i] = *reinterpret_cast<const f4 *>(a.Q + (int64_t)c.token * a.ldq + c.head * D + 64 * k + 16 * g + 4 * i);
            }
    }
    __device__ __forceinline__ float split(h8 (*qh)[2], h8 (*ql)[2]) const
    {
        float mx = 0.f;
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) mx = fmaxf(mx, fabsf(x[k][i][u]));
        const int e = 15 - __builtin_amdgcn_frexp_expf(over4_max(mx));   // the largest |q| into [2^14, 2^15)
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                uint32_t h[4], l[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f4 v = x[k][2 * m + i / 2];
                    split2(ldexpf(v[2 * (i % 2)], e), ldexpf(v[2 * (i % 2) + 1], e), h[i], l[i]);
                }
                qh[k][m] = __builtin_bit_cast(h8, u4{h[0], h[1], h[2], h[3]});
                ql[k][m] = __builtin_bit_cast(h8, u4{l[0], l[1], l[2], l[3]});
            }
        return ldexpf(1.0f, -e);
    }
};

// 64 groups of 16 tokens of a request from key tile t0 on (16 tiles), lane l the
// l-th: its place in the cache (in groups; kNone past the request's tokens or
// outside the cache) and its scales.  In two steps, the table's entries and what
// they lead to, so that a loop over tiles can take them ahead of their use.
// What a lane reads in place of a group that is not there: a weight of 0 times a
// byte that is no number would be none.
__device__ const u4 no_group[256] = {};   // 16 tokens of 256 dimensions
__device__ __forceinline__ const uint8_t *group_ptr(const uint8_t *codes, uint32_t at, int bytes)
{
    return at == kNone ? reinterpret_cast<const uint8_t *>(no_group) : codes + (size_t)at * bytes;
}

constexpr float kHidden = -1.0f;   // the value scale of a group that is not there
struct Groups {
    uint32_t at;
    float ks, vs;
};

__device__ __forceinline__ int32_t load_ids(const Args &a, const Item &it, int32_t t0)
{
    const uint32_t group = (uint32_t)t0 * 4 + (threadIdx.x & 63);   // of 16 tokens, of the request
    return group < ((uint32_t)it.q.len + 15) / 16 ? a.tables[(int64_t)it.seq * a.width + (group >> (a.shift - 4))] : -1;
}

__device__ __forceinline__ Groups load_groups(const Args &a, int32_t id, int32_t kvh, int32_t heads, int32_t t0)
{
    const uint32_t group = (uint32_t)t0 * 4 + (threadIdx.x & 63);   // of 16 tokens, of the request
    Groups r{kNone, 0.f, kHidden};
    if (id >= 0 && id < a.n_blocks) {
        const uint32_t block = (uint32_t)id * (uint32_t)heads + (uint32_t)kvh;
        r.at = (block << (a.shift - 4)) + (group & ((1u << (a.shift - 4)) - 1));
        r.ks = a.ks[block];
        r.vs = a.vs[block];
    }
    return r;
}

// The groups of a walk over tiles lo .. hi - 1: advance(t) before tile t's are used.
struct Walk {
    Groups now, then;
    int32_t ids;
    __device__ __forceinline__ void start(const Args &a, const Item &it, int32_t kvh, int32_t heads, int32_t lo, int32_t id)
    {
        now = load_groups(a, id, kvh, heads, lo);
    }
    __device__ __forceinline__ void advance(const Args &a, const Item &it, int32_t kvh, int32_t heads, int32_t lo,
                                            int32_t hi, int32_t t)
    {
        const int32_t in = (t - lo) & 15, next = t - in + 16;
        if (in == 0 && t > lo) now = then;
        if (next < hi) {
            if (in == 2) ids = load_ids(a, it, next);
            if (in == 9) then = load_groups(a, ids, kvh, heads, next);
        }
    }
};

// What a lane needs of its group of a tile: the scales.
struct Lane {
    float ks, vs;
};

// What makes weights of a lane's products of one tile: p = 2^(f s + add), the
// weight p vs, and the sum of the p times 2^-e into the state's.
struct Weights {
    float f, add, vs, e;
};

// The scores of a tile, and the state's normalizer and accumulator brought up to
// them.  s: the lane's 16 products of query c with keys key0 + 0..15 (key0 = 64
// tile + 16 g); f: the factor that makes them scores, times log2 e unless MOD.
// hide (the same in all lanes): some key of the tile is not seen by some query.
template <int D, bool MOD>
__device__ __forceinline__ Weights score_tile(const Args &a, const View &v, const Col &c, const Lane &ln, int32_t key0,
                                              float f, bool hide, f4 *s, State<D> &st)
{
    if constexpr (MOD) {
        float top = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(s[t][i]));
        if (a.cap > 0.f) {
            const float u = f / a.cap, out = a.cap * kLog2e;
            if (__any(!(top * fabsf(u) < 0.7f))) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][i] = out * tanh_any(s[t][i] * u);
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][i] = out * tanh_small(s[t][i] * u);
            }
        } else {
            f *= kLog2e;
#pragma unroll
            for (int t = 0; t < 4; ++t) s[t] *= f;
        }
        const float far = (float)(c.pos - key0);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = fmaf(-c.slope, fabsf(far - (float)(4 * t + i)), s[t][i]);
        f = 1.0f;
    }
    float scale = ln.vs;   // 0 where the query sees no key of this lane's group: that block may have no number for a scale
    if (hide) {
        const int32_t lo = v.lo(c.pos) - key0, hi = ln.vs == kHidden ? -1 : v.hi(c.pos) - key0;
        if (!(lo < 16 && hi > 0)) scale = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int32_t j = 4 * t + i;
                s[t][i] = j >= lo && j < hi ? s[t][i] * f : -INFINITY;
            }
        f = 1.0f;
    }
    const float ve = scale > 0.f && scale < INFINITY ? (float)__builtin_amdgcn_frexp_expf(scale) : kNoExp;
    st.e = fmaxf(st.e, over4_max(ve));
    const float e = fmaxf(fmaxf(ve, st.e - 60.f), -100.f), em = fmaxf(fmaxf(ve, e - 100.f), -100.f);
    const float vs = ldexpf(scale, 15 - (int)e);
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[t][i]);
    // Beyond 2^20, of either sign, the rounding of a score is no longer small beside 1: the normalizer and the exponents below
    // have to come from the same rounded scores (MOD's are rounded already).  Beyond 2^24 the normalizer and the
    // difference to it are rounded too, as coarsely as the scores: `most` keeps p below 2^(e - em) all the same.
    float most = INFINITY;
    if constexpr (MOD) most = (e - em) - mx;
    else {
        const bool large = fabsf(mx * f) > 0x1p20f && mx > -INFINITY;   // -inf: the query sees nothing of the group
        if (__any(large)) {
            const float by = large ? f : 1.0f;   // (a row's result does not depend on the other rows)
#pragma unroll
            for (int t = 0; t < 4; ++t) s[t] *= by;
            mx *= by;
            f = large ? 1.0f : f;
            if (large) most = (e - em) - mx;
        }
    }
    const float m = fmaxf(st.m, ceilf(over4_max(fmaf(mx, f, em))));   // f >= 0; a NaN score is left out here and shows below
    if (__any(m > st.m)) {
        const float back = times2(1.0f, st.m - m);
        st.l *= back;
        st.times(back);
        st.m = m;
    }
    return Weights{f, fminf(e - (m == -INFINITY ? 0.f : m), most), vs, e};
}

// The weights of keys 8 m + 0..7 of the lane's group, split; the sum of their p is added to `sum`.
__device__ __forceinline__ void weigh(const Weights &w, int m, const f4 *s, float &sum, h8 &ph, h8 &pl)
{
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float s0 = s[2 * m + i / 2][2 * (i % 2)], s1 = s[2 * m + i / 2][2 * (i % 2) + 1];
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s0, w.f, w.add)), p1 = __builtin_amdgcn_exp2f(fmaf(s1, w.f, w.add));
        sum += p0;
        sum += p1;
        split2(p0 * w.vs, p1 * w.vs, hi[i], lo[i]);
    }
    ph = __builtin_bit_cast(h8, u4{hi[0], hi[1], hi[2], hi[3]});
    pl = __builtin_bit_cast(h8, u4{lo[0], lo[1], lo[2], lo[3]});
}

// ---------------------------------------------------------------- few rows: 16 at a time
// Workgroup (head fastest): a part of one tile of 16 rows; its four waves take
// a quarter of the part's keys each, straight from memory to the matrix cores,
// and join through LDS.  Bound by memory where the cache is long: one token of
// each of 64 requests of 516 to 7804 tokens (32 heads over 8, D = 128, int8) reads
// 396 MB and takes 83 us, 4.8 TB/s, what a large copy reaches on the card: two such
// workgroups to a CU with half a tile of loads ahead are enough for that.  One request of 513 tokens: 10.1 us, where the
// waves wait for half of their cycles (lengths, table, codes, the join) and issue for 40% of them (three tiles, their
// conversions and softmax); eight waves 0.2 more.
template <int FMT, int D, bool MOD>
__global__ void __launch_bounds__(256)
few_kernel(Args a, int32_t heads)
{
    constexpr int C = D / 64, DT = D / 16;
    __shared__ float os[4][16][D + 4];
    __shared__ float ms[4][16], ls[4][16];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int32_t kvh = blockIdx.x % heads;
    const Item it = find_item<16>(a, blockIdx.x / heads, heads, false);
    if (!it.ok) return;
    const View view = view_of(a, it);
    const Range all = tile_keys<16>(a, it, view), mine = part_of(all, it.split, it.n_split);
    const int32_t nt = mine.hi - mine.lo;
    const int32_t t0 = mine.lo + nt * w / 4, t1 = mine.lo + nt * (w + 1) / 4;

    // the table's entries first, then Q: the codes' addresses wait for the former alone
    const int32_t ids = t0 < t1 ? load_ids(a, it, t0) : -1;
    const Place place = row_of(a, it, kvh, (uint32_t)it.tile * 16, c);
    QRow<D> qrow;
    qrow.load(a, place, g);
    const Col col = column(a, it, place);
    Walk walk;
    walk.start(a, it, kvh, heads, t0, ids);
    // Keys and values of the next tile are loaded as soon as the registers of
    // this one's are free: half a tile ahead each.
    u4 kr[4][C], vr[DT];
    auto load_k = [&](int32_t t) {
        const uint32_t at = __shfl(walk.now.at, 4 * ((t - t0) & 15) + (c >> 2));
        const uint8_t *kp = group_ptr(a.k, at, 16 * D) + ((c & 3) * 4 + g) * 16;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int k = 0; k < C; ++k) kr[q][k] = *reinterpret_cast<const u4 *>(kp + (q * C + k) * 256);
    };
    auto load_v = [&](int32_t t) {
        const int from = 4 * ((t - t0) & 15) + g;
        const uint32_t at = __shfl(walk.now.at, from);
        const uint8_t *vp = group_ptr(a.v, at, 16 * D) + c * 16;
#pragma unroll
        for (int d = 0; d < DT; ++d) vr[d] = *reinterpret_cast<const u4 *>(vp + d * 256);
        return Lane{__shfl(walk.now.ks, from), __shfl(walk.now.vs, from)};
    };
    Lane ln{0.f, kHidden};
    if (t0 < t1) {
        load_k(t0);
        ln = load_v(t0);
    }
    h8 qh[C][2], ql[C][2];
    const float undo = qrow.split(qh, ql) * a.scale * (MOD ? 1.0f : kLog2e);
    const Sight sight = sight_of(view, col);

    State<D> st;
    st.init();
    for (int32_t t = t0; t < t1; ++t) {
        f4 s[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            s[q] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < C; ++k)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const h8 x = to_half<FMT>(kr[q][k][2 * m], kr[q][k][2 * m + 1]);
                    s[q] = mfma(x, qh[k][m], s[q]);
                    s[q] = mfma(x, ql[k][m], s[q]);
                }
        }
        if (t + 1 < t1) {
            walk.advance(a, it, kvh, heads, t0, t1, t + 1);
            load_k(t + 1);
        }
        const bool hide = t < sight.all_lo || t >= sight.all_hi || __any(ln.vs == kHidden);
        const Weights wt = score_tile<D, MOD>(a, view, col, ln, t * 64 + 16 * g, undo * ln.ks, hide, s, st);
        float sum = 0.f;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            h8 ph, pl;
            weigh(wt, m, s, sum, ph, pl);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const h8 x = to_half<FMT>(vr[d][2 * m], vr[d][2 * m + 1]);
                st.o[d] = mfma(x, ph, st.o[d]);
                st.o[d] = mfma(x, pl, st.o[d]);
            }
        }
        st.l += ldexpf(sum, -(int)wt.e);
        if (t + 1 < t1) ln = load_v(t + 1);
    }
    // join the waves
    const float l = over4_sum(st.l);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f4 *>(&os[w][c][16 * d + 4 * g]) = st.o[d];
    if (g == 0) {
        ms[w][c] = st.m;
        ls[w][c] = l;
    }
    __syncthreads();
    const int row = tid >> 4;
    float m = ms[0][row];
#pragma unroll
    for (int i = 1; i < 4; ++i) m = fmaxf(m, ms[i][row]);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += times2(ls[i][row], ms[i][row] - m);
    const bool whole = it.n_split == 1;
    const Place out = row_of(a, it, kvh, (uint32_t)it.tile * 16, row);
    // starts in ascending order never have more parts than the scratch holds
    const int64_t part = ((int64_t)it.part + it.split) * heads + kvh;
    if (!whole && (it.part < 0 || part >= a.n_part)) return;
    const float div = !whole ? 1.0f : sum != 0.f ? 0x1p-15f / sum : 0.f;
    float *to = whole ? a.O + (int64_t)out.token * a.ldo + out.head * D : a.part + (part * 16 + row) * D;
    if (!whole && (tid & 15) == 0) {
        a.part_ml[(part * 16 + row) * 2] = m;
        a.part_ml[(part * 16 + row) * 2 + 1] = sum;
    }
    if (out.token < 0) return;
#pragma unroll
    for (int d = 4 * (tid & 15); d < D; d += 64) {
        f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f4 y = *reinterpret_cast<const f4 *>(&os[i][row][d]);
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] += times2(y[u], ms[i][row] - m);
        }
        *reinterpret_cast<f4 *>(to + d) = x * div;
    }
}

// ---------------------------------------------------------------- many rows: 64 or 128 at a time
// Workgroup (head fastest): a part of one tile of 64 N rows, N columns of 16 to
// a wave.  The codes of a key tile are converted to fp16 once, into LDS, in the
// order in which the lanes read them (unit by unit, so every LDS access is 1 KB in
// a row), and every fragment read feeds the products of N columns and two
// halves.  Two images: while a tile is multiplied, the next one, loaded a tile
// ago, is converted, and the one after it is loaded.  One barrier per tile.
// Bound by the matrix and vector units in turn: four prompts of 363 to 3690
// tokens (32 heads over 8, D = 128, e4m3) take 287 us.  Their attention is 141 GFLOP, 283 on the
// matrix units for the split operands: 985 TFLOP/s, where a large library product in fp16
// reaches 1138 on the card.  The matrix units are busy 45% of the time at 2.1 GHz; the
// rest are exponentials, splits and conversions, which the two workgroups of a CU
// overlap only in part.  200 tokens after 16000: 121 us, 870 TFLOP/s.
template <int FMT, int D, int N, bool MOD>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2)
prompt_kernel(Args a, int32_t heads)
{
    constexpr int C = D / 64, DT = D / 16, FR = 8 * C, R = 64 * N;
    __shared__ h8 image[2][2][4 * C * 2 * 64];   // [buffer][keys, values][(unit row, half)][lane]
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int32_t kvh = blockIdx.x % heads;
    const Item it = find_item<R>(a, blockIdx.x / heads, heads, false);
    if (!it.ok) return;
    const View view = view_of(a, it);
    const Range all = tile_keys<R>(a, it, view), mine = part_of(all, it.split, it.n_split);

    // the table's entries first, then Q: the codes' addresses wait for the former alone
    const int32_t ids = mine.lo < mine.hi ? load_ids(a, it, mine.lo) : -1;
    Col col[N];
    QRow<D> qrow[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const Place place = row_of(a, it, kvh, (uint32_t)it.tile * R, 16 * N * w + 16 * n + c);
        qrow[n].load(a, place, g);
        col[n] = column(a, it, place);
    }
    Walk walk;
    walk.start(a, it, kvh, heads, mine.lo, ids);
    u4 kr[C] = {}, vr[C] = {};
    // loads tile t (this thread's units of it) and returns what its lane needs of it
    auto load = [&](int32_t t) {
        Lane ln{0.f, kHidden};
        if (t >= mine.hi) return ln;
        walk.advance(a, it, kvh, heads, mine.lo, mine.hi, t);
        const int in = (t - mine.lo) & 15;
        const uint32_t at_k = __shfl(walk.now.at, 4 * in + (c >> 2)), at_v = __shfl(walk.now.at, 4 * in + g);
        const uint8_t *kp = group_ptr(a.k, at_k, 16 * D) + ((c & 3) * 4 + g) * 16 + w * 256;
        const uint8_t *vp = group_ptr(a.v, at_v, 16 * D) + c * 16 + w * 256;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            kr[i] = *reinterpret_cast<const u4 *>(kp + i * 1024);
            vr[i] = *reinterpret_cast<const u4 *>(vp + i * 1024);
        }
        ln.ks = __shfl(walk.now.ks, 4 * in + g);
        ln.vs = __shfl(walk.now.vs, 4 * in + g);
        return ln;
    };
    // piece j of 4 C of what this thread converts: eight codes
    auto convert = [&](int b, int j) {
        const int i = j / 4, m = j % 2;
        const u4 x = j / 2 % 2 ? vr[i] : kr[i];
        image[b][j / 2 % 2][((w + 4 * i) * 2 + m) * 64 + lane] = to_half<FMT>(x[2 * m], x[2 * m + 1]);
    };
    Lane ln = load(mine.lo), next{};
    Sight sight[N];
    h8 qh[N][C][2], ql[N][C][2];
    float undo[N];
    State<D> st[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        undo[n] = qrow[n].split(qh[n], ql[n]) * a.scale * (MOD ? 1.0f : kLog2e);
        sight[n] = sight_of(view, col[n]);
        st[n].init();
    }
#pragma unroll
    for (int j = 0; j < 4 * C; ++j) convert(0, j);
    next = load(mine.lo + 1);
    __syncthreads();
    // tile t, in buffer B (a constant: reads of one buffer and writes of the other may then pass each other)
    auto step = [&](auto buffer, int32_t t) {
        constexpr int b = decltype(buffer)::value;
        f4 s[N][4];
        {
            // Fragment i: key rows q = i / (2 C), dimensions (k, m).  Left alone, the compiler reads a fragment, waits
            // for it and multiplies; here the order is fixed: a read three fragments ahead, the products of this one,
            // and at every second a piece of the next tile's conversion (past the last tile: of what was there, for
            // nobody), which the vector units do beside them.
            const h8 *x = &image[b][0][lane];
            h8 f[FR];
#pragma unroll
            for (int i = 0; i < 3; ++i) f[i] = x[i * 64];
#pragma unroll
            for (int i = 0; i < FR; ++i) {
                const int q = i / (2 * C), k = i / 2 % C, m = i % 2;
                if (i + 3 < FR) f[i + 3] = x[(i + 3) * 64];
#pragma unroll
                for (int n = 0; n < N; ++n) s[n][q] = mfma(f[i], qh[n][k][m], i % (2 * C) ? s[n][q] : f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int n = 0; n < N; ++n) s[n][q] = mfma(f[i], ql[n][k][m], s[n][q]);
                if (i % 2) convert(b ^ 1, i / 2);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        const Lane here = ln;
        ln = next;
        next = load(t + 2);
        const bool none = __any(here.vs == kHidden);
        Weights wt[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bool hide = none || t < sight[n].all_lo || t >= sight[n].all_hi;
            wt[n] = score_tile<D, MOD>(a, view, col[n], here, t * 64 + 16 * g, undo[n] * here.ks, hide, s[n], st[n]);
        }
        {
            const h8 *x = &image[b][1][lane];
            float sum[N] = {};
            h8 ph[N], pl[N];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int n = 0; n < N; ++n) weigh(wt[n], m, s[n], sum[n], ph[n], pl[n]);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const h8 f = x[(d * 2 + m) * 64];
#pragma unroll
                    for (int n = 0; n < N; ++n) st[n].o[d] = mfma(f, ph[n], st[n].o[d]);
#pragma unroll
                    for (int n = 0; n < N; ++n) st[n].o[d] = mfma(f, pl[n], st[n].o[d]);
                }
            }
#pragma unroll
            for (int n = 0; n < N; ++n) st[n].l += ldexpf(sum[n], -(int)wt[n].e);
            // the first half's weights, then its products with the second half's weights between them; three fragments ahead,
            // or two where cap and slopes take registers (with three D = 128, N = 2 keeps up to 16 bytes in private memory)
            constexpr int kAhead = MOD ? 2 : 3;
            __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 1);
            __builtin_amdgcn_sched_group_barrier(0x402, 58 * N, 1);
#pragma unroll
            for (int i = 0; i < 2 * DT; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, N, 1);
                if (i < DT) __builtin_amdgcn_sched_group_barrier(0x402, 56 * N / (2 * DT), 1);
                __builtin_amdgcn_sched_group_barrier(0x008, N, 1);
                if (i + kAhead < 2 * DT) __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
                if (i < DT) __builtin_amdgcn_sched_group_barrier(0x402, 56 * N / (2 * DT), 1);
            }
        }
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
    };
    for (int32_t t = mine.lo; t < mine.hi; t += 2) {
        step(std::integral_constant<int, 0>(), t);
        if (t + 1 < mine.hi) step(std::integral_constant<int, 1>(), t + 1);
    }
    const bool whole = it.n_split == 1;
    // starts in ascending order never have more parts than the scratch holds
    const int64_t part = ((int64_t)it.part + it.split) * heads + kvh;
    if (!whole && (it.part < 0 || part >= a.n_part)) return;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const float sum = over4_sum(st[n].l);
        const Place out = row_of(a, it, kvh, (uint32_t)it.tile * R, 16 * N * w + 16 * n + c);
        if (out.token < 0) continue;
        const int64_t row = part * R + 16 * N * w + 16 * n + c;
        float *to = whole ? a.O + (int64_t)out.token * a.ldo + out.head * D : a.part + row * D;
        if (!whole && g == 0) {
            a.part_ml[row * 2] = st[n].m;
            a.part_ml[row * 2 + 1] = sum;
        }
        const float div = !whole ? 1.0f : sum != 0.f ? 0x1p-15f / sum : 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f4 *>(to + 16 * d + 4 * g) = st[n].o[d] * div;
    }
}

// ---------------------------------------------------------------- join the parts
// Workgroup (head fastest): 16 rows of one row tile that was split.  A unit is
// four floats of a row; where the tile has fewer than 256 of them (few rows, as in
// a decode step), the parts are dealt out to slices of the threads, whose sums
// are added through LDS, in the order of the slices.  Bound by the latency of
// finding the tile and of its loads: 4 to 6 us after decode steps, 9.8 for 200
// tokens in parts of 16000.
template <int D, int R>
__global__ void __launch_bounds__(256)
join_kernel(Args a, int32_t heads)
{
    constexpr int Q = D / 4;   // units of a row
    __shared__ f4 xs[256];
    __shared__ float ms[256], ls[256];
    const int tid = threadIdx.x;
    const int32_t kvh = blockIdx.x % heads, sub = blockIdx.x / heads % (R / 16);
    const Item it = find_item<R>(a, blockIdx.x / heads / (R / 16), heads, true);
    if (!it.ok || it.part < 0 || ((int64_t)it.part + it.n_split) * heads > a.n_part) return;
    const int32_t left = it.q.n * a.group - (it.tile * R + 16 * sub);   // rows from the first of these on
    if (left <= 0) return;
    const Range all = tile_keys<R>(a, it, view_of(a, it));
    const int32_t n = all.hi - all.lo, per = (n + it.n_split - 1) / it.n_split;
    const int32_t parts = per ? (n + per - 1) / per : 0;   // the others are empty
    int rows = 1;                                          // a power of two that holds the rows
    while (rows < min(left, 16)) rows *= 2;
    const int units = rows * Q, slices = max(1, 256 / units);
    for (int u0 = 0; u0 < units; u0 += 256) {
        const int u = u0 + tid % min(units, 256), slice = tid / min(units, 256);
        const int row = 16 * sub + u / Q, d = 4 * (u % Q);
        auto index = [&](int32_t p) { return ((int64_t)(it.part + p) * heads + kvh) * R + row; };
        float m = -INFINITY, sum = 0.f;
        f4 x = {0.f, 0.f, 0.f, 0.f};
        for (int32_t p0 = slice; p0 < parts; p0 += 8 * slices) {
            f4 y[8];
            float ym[8], yl[8], top = m;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int32_t p = p0 + i * slices;
                const int64_t at = index(p < parts ? p : p0);
                ym[i] = a.part_ml[at * 2];
                yl[i] = p < parts ? a.part_ml[at * 2 + 1] : 0.f;
                y[i] = *reinterpret_cast<const f4 *>(a.part + at * D + d);
                top = fmaxf(top, ym[i]);
            }
            sum = times2(sum, m - top);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = times2(x[e], m - top);
            m = top;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum += times2(yl[i], ym[i] - m);
                if (p0 + i * slices < parts)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] += times2(y[i][e], ym[i] - m);
            }
        }
        if (slices > 1) {
            xs[tid] = x;
            ms[tid] = m;
            ls[tid] = sum;
            __syncthreads();
            if (slice) return;   // units <= 128: the loop ends here
            for (int i = 1; i < slices; ++i) m = fmaxf(m, ms[u + i * units]);
            x = f4{0.f, 0.f, 0.f, 0.f};
            sum = 0.f;
            for (int i = 0; i < slices; ++i) {
                const int at = u + i * units;
                const float d2 = ms[at] - m;
                const f4 y = xs[at];
                sum += times2(ls[at], d2);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] += times2(y[e], d2);
            }
        }
        const Place out = row_of(a, it, kvh, (uint32_t)it.tile * R, row);
        if (out.token < 0) continue;
        const float div = sum != 0.f ? 0x1p-15f / sum : 0.f;
        *reinterpret_cast<f4 *>(a.O + (int64_t)out.token * a.ldo + out.head * D + d) = x * div;
    }
}

// ---------------------------------------------------------------- how a call is split
// Rows per tile, workgroups wanted, fewest key tiles of a part.
struct Plan {
    int rows, least;
    int64_t target, tiles, items, parts;   // bounds over one KV head (tiles, items) and over all (parts)
    int64_t joins;                         // of one KV head: tiles that are split
};

// Up to this many key tiles are not split: a row tile's own workgroup does them in less time than a second launch takes.
constexpr int64_t kWhole = 16;

Plan plan_of(const aih_ctx *ctx, const aih_kv_cache *kv, int32_t n_heads, int64_t rows, int32_t n_seqs,
             int32_t table_width)
{
    const int64_t cus = ctx->cu_count > 0 ? ctx->cu_count : 256, heads = kv->n_kv_heads, group = n_heads / heads;
    Plan p{};
    const int64_t most_keys = ((int64_t)table_width * kv->block_tokens + 63) / 64;
    auto tiles_of = [&](int r) { return std::min<int64_t>(n_seqs, rows) + rows * group / r; };
    // The tile of a request's rows, by what a call would take with requests of equal rows and full tables (the lengths
    // are on the device): tables much longer than the requests, and prompts beside single tokens, get the tile of another
    // batch, which is right but slower (a prompt of 512 under a table for 8192 tokens 28.9 us in place of 19.8).
    // Tiles of 16: 0.5 us of a CU for a tile and 64 keys, and 5 us for every further round of workgroups; of 64: 1.1 us,
    // or 1.25 us one after the other for the keys of a part, and 12 us for a join.  Measured, 32 heads over 8, D = 128,
    // int8, us of 16 / 64: 64 tokens after 4000 24.1 / 27.3, 100 after 8000 57.4 / 45.8, 300 after 2000 47.2 / 39.7, 16
    // requests of 16 after 1000 20.6 / 28.3, of 8 after 1000 13.3 / 27.0, 4 prompts of 100 14.7 / 9.4, 16 of 40 22.4 /
    // 11.4, one of 150 8.5 / 10.2, of 300 14.3 / 13.1, 8 of 32 after 500 15.1 / 19.4.
    // Tiles of 128 use a converted key twice as often but are fewer and take longer each: us of 64 / 128: prompt of 1024
    // 35.6 / 45.2 (16 tiles of 128 rows and 64 keys a CU), 100 after 8000 45.9 / 48.5 (16), prompt of 2048 90.1 / 90.7
    // (64), of 4096 284 / 260 (256), 200 after 16000 170 / 118 (55).
    const double per_seq = (double)(rows * group) / n_seqs, keys = (double)most_keys, cu = (double)cus;
    auto groups_of = [&](int r) { return n_seqs * std::ceil(per_seq / r) * (double)heads; };
    const bool joined = most_keys > kWhole;
    const double g16 = groups_of(16), g64 = groups_of(64);
    const double us16 = 5.0 * std::max(0.0, g16 / (2 * cu) - 1) + 0.5 * g16 * keys / cu;
    const double part64 = joined ? std::max(4.0, keys * std::min(1.0, g64 / (2 * cu))) : keys;
    const double us64 = std::max(1.25 * part64, 1.1 * g64 * keys / cu) + (joined ? 12.0 : 0.0);
    const bool wide = kv->head_dim < 256 && (double)(tiles_of(128) * heads) * keys >= 48 * cu;
    p.rows = us16 < us64 ? 16 : wide ? 128 : 64;
    p.least = 4;
    // At D = 256 the registers (16 rows) or LDS (64) allow one workgroup to a CU, at D = 128 two; at D = 64 three or four
    // would fit, and two are aimed at as well.  One token each
    // of 16 requests of 1033 to 4884 tokens, D = 256: 48.1 us with one wanted a CU, 50.1 with two, 67 with four; one
    // request of 30000 tokens, D = 128: 22.4 with two, 28.4 with four.
    p.target = (kv->head_dim == 256 ? 1 : 2) * cus;
    p.tiles = tiles_of(p.rows);   // sum of ceil(n_s group / R) over the n_s > 0
    const int64_t most_split = !joined ? 1 : (most_keys + p.least - 1) / p.least;
    // tiles * ceil(keys / length) <= tiles + work / length and work / length <= 2 target / heads, summed in floats
    p.items = std::min(p.tiles * most_split, p.tiles + 2 * p.target / heads + 2);
    // a tile that is split has more keys than one part, so its parts are at most twice its keys over the length
    p.parts = most_split <= 1 ? 0 : std::min(p.items * heads, 4 * p.target + 4 * heads);
    // and there are fewer such tiles than work / length
    p.joins = std::min(p.tiles, 2 * p.target / heads + 2);
    return p;
}

constexpr int64_t kAlign = 4;   // floats: the partial outputs start on 16 bytes

int64_t layout_floats(int32_t n_seqs) { return n_seqs > kScan ? (4 + 3 * ((int64_t)n_seqs + 1) + kAlign - 1) / kAlign * kAlign : 0; }
int64_t ml_floats(const Plan &p) { return (p.parts * p.rows * 2 + kAlign - 1) / kAlign * kAlign; }

template <int FMT, int D, bool MOD>
int launch(aih_ctx *ctx, const Args &a, const Plan &p, int32_t heads)
{
    const dim3 grid((unsigned)(p.items * heads)), join((unsigned)(p.joins * heads * (p.rows / 16))), block(256);
    constexpr int kWide = D == 256 ? 1 : 2;   // at D = 256 a wave's registers hold one column of 16
    if (a.layout) {
        if (p.rows == 16) hipLaunchKernelGGL((layout_kernel<16>), dim3(1), dim3(1024), 0, ctx->stream, a, heads);
        else if (p.rows == 64) hipLaunchKernelGGL((layout_kernel<64>), dim3(1), dim3(1024), 0, ctx->stream, a, heads);
        else hipLaunchKernelGGL((layout_kernel<64 * kWide>), dim3(1), dim3(1024), 0, ctx->stream, a, heads);
        const int rc = aih_launch_status();
        if (rc) return rc;
    }
    if (p.rows == 16) hipLaunchKernelGGL((few_kernel<FMT, D, MOD>), grid, block, 0, ctx->stream, a, heads);
    else if (p.rows == 64) hipLaunchKernelGGL((prompt_kernel<FMT, D, 1, MOD>), grid, block, 0, ctx->stream, a, heads);
    else hipLaunchKernelGGL((prompt_kernel<FMT, D, kWide, MOD>), grid, block, 0, ctx->stream, a, heads);
    if (p.parts) {
        const int rc = aih_launch_status();
        if (rc) return rc;
        if (p.rows == 16) hipLaunchKernelGGL((join_kernel<D, 16>), join, block, 0, ctx->stream, a, heads);
        else if (p.rows == 64) hipLaunchKernelGGL((join_kernel<D, 64>), join, block, 0, ctx->stream, a, heads);
        else hipLaunchKernelGGL((join_kernel<D, 64 * kWide>), join, block, 0, ctx->stream, a, heads);
    }
    return aih_launch_status();
}

template <int FMT, int D>
int launch_mod(aih_ctx *ctx, const Args &a, const Plan &p, int32_t heads)
{
    return a.cap > 0.f || a.slopes ? launch<FMT, D, true>(ctx, a, p, heads) : launch<FMT, D, false>(ctx, a, p, heads);
}

template <int FMT>
int launch_dim(aih_ctx *ctx, int32_t dim, const Args &a, const Plan &p, int32_t heads)
{
    switch (dim) {
    case 64: return launch_mod<FMT, 64>(ctx, a, p, heads);
    case 128: return launch_mod<FMT, 128>(ctx, a, p, heads);
    default: return launch_mod<FMT, 256>(ctx, a, p, heads);
    }
}

int check_batch(const aih_kv_cache *kv, int32_t n_heads, int64_t rows, int32_t n_seqs, int32_t table_width)
{
    if (n_heads <= 0 || rows < 0 || n_seqs <= 0 || table_width <= 0 || n_heads % kv->n_kv_heads) return AIH_E_INVALID;
    if (n_seqs > aih_kv::kMaxSeqs || (int64_t)table_width * kv->block_tokens > 0x7FFFFFFF || rows > 0x7FFFFFFF ||
        rows * (n_heads / kv->n_kv_heads) > 0x7FFFFF00 || n_heads > aih_kv::kMaxHeads)
        return AIH_E_LIMIT;
    return AIH_OK;
}

}  // namespace

extern "C" {

int64_t aih_kv_attention_scratch_floats(aih_ctx *ctx, const aih_kv_cache *kv, int32_t n_heads, int64_t rows,
                                        int32_t n_seqs, int32_t table_width)
{
    if (!ctx) return AIH_E_INVALID;
    int rc = aih_kv::check_shape(kv);
    if (!rc) rc = check_batch(kv, n_heads, rows, n_seqs, table_width);
    if (rc) return rc;
    const Plan p = plan_of(ctx, kv, n_heads, rows, n_seqs, table_width);
    return layout_floats(n_seqs) + ml_floats(p) + p.parts * p.rows * kv->head_dim;
}

int aih_kv_attention_tile_rows(aih_ctx *ctx, const aih_kv_cache *kv, int32_t n_heads, int64_t rows, int32_t n_seqs,
                               int32_t table_width)
{
    if (!ctx) return AIH_E_INVALID;
    int rc = aih_kv::check_shape(kv);
    if (!rc) rc = check_batch(kv, n_heads, rows, n_seqs, table_width);
    return rc ? rc : plan_of(ctx, kv, n_heads, rows, n_seqs, table_width).rows;
}

int aih_kv_attention(aih_ctx *ctx, const aih_kv_cache *kv, const float *Q, int64_t ldq, float *O, int64_t ldo,
                     int64_t rows, int32_t n_heads, int32_t n_seqs, const int32_t *starts, const int32_t *lens,
                     const int32_t *tables, int32_t table_width, float scale, const aih_kv_scores *scores,
                     float *scratch, int64_t scratch_floats)
{
    if (!ctx) return AIH_E_INVALID;
    int rc = aih_kv::check_cache(kv);
    if (!rc) rc = check_batch(kv, n_heads, rows, n_seqs, table_width);
    if (rc) return rc;
    const int64_t wide = (int64_t)n_heads * kv->head_dim;
    if (!Q || !O || !starts || !lens || !tables || ldq < wide || ldo < wide || ldq % 4 || ldo % 4 ||
        !aih_kv::aligned16(Q) || !aih_kv::aligned16(O) || !(scale > 0.0f) || !std::isfinite(scale))
        return AIH_E_INVALID;
    const aih_kv_scores none{};
    if (!scores) scores = &none;
    if (!(scores->cap >= 0.0f) || !std::isfinite(scores->cap) || scores->window < 0) return AIH_E_INVALID;
    const Plan p = plan_of(ctx, kv, n_heads, rows, n_seqs, table_width);
    const int64_t before = layout_floats(n_seqs), need = before + ml_floats(p) + p.parts * p.rows * kv->head_dim;
    if (need && (!scratch || !aih_kv::aligned16(scratch) || scratch_floats < need)) return AIH_E_INVALID;
    if (rows == 0) return AIH_OK;
    if (std::max(p.items, p.joins * (p.rows / 16)) * kv->n_kv_heads > aih_kv::kMaxGroups) return AIH_E_LIMIT;
    Args a{};
    a.k = static_cast<const uint8_t *>(kv->k);
    a.v = static_cast<const uint8_t *>(kv->v);
    a.ks = kv->k_scale;
    a.vs = kv->v_scale;
    a.Q = Q;
    a.O = O;
    a.ldq = ldq;
    a.ldo = ldo;
    a.starts = starts;
    a.lens = lens;
    a.tables = tables;
    a.slopes = scores->slopes;
    a.prefix = scores->prefix;
    a.layout = before ? reinterpret_cast<int32_t *>(scratch) : nullptr;
    a.part_ml = scratch + before;
    a.part = a.part_ml + ml_floats(p);
    a.rows = (int32_t)rows;
    a.heads = n_heads;
    a.group = n_heads / kv->n_kv_heads;
    a.inv_group = 1.0f / (float)a.group;
    a.n_seqs = n_seqs;
    a.width = table_width;
    a.n_blocks = kv->n_blocks;
    a.shift = aih_kv::log2_of(kv->block_tokens);
    a.window = scores->window;
    a.target = (int32_t)p.target;
    a.least = p.least;
    a.n_part = (int32_t)p.parts;
    a.scale = scale;
    // A score divided by the cap must not leave the normal numbers.  2^90 and more cap nothing that 24 bits of a score can
    // tell apart; below 2^-60 all scores are as good as 0.
    a.cap = scores->cap > 0.0f ? std::min(std::max(scores->cap, 0x1p-60f), 0x1p90f) : 0.0f;
    aih_kv::DeviceGuard guard(ctx->device);
    AIH_TRY(guard.status);
    return kv->format == AIH_KV_INT8 ? launch_dim<AIH_KV_INT8>(ctx, kv->head_dim, a, p, kv->n_kv_heads)
                                     : launch_dim<AIH_KV_E4M3>(ctx, kv->head_dim, a, p, kv->n_kv_heads);
}

}  // extern "C"
