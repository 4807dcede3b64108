// aih_kv_cache.hip -- the bookkeeping and the storing side of the paged 8-bit
// KV cache (include/aihost_hip.h): block tables and slot maps from request
// lengths, new rows into the cache with a scale per block and head, and the
// cache's values back as fp32 rows.  The reading side is aih_kv_attention.hip.
//
// This file is compiled without FMA contraction, so that rotated keys round
// like aih_rope's; the one fused multiply-add that the rounding of a quotient
// needs is written out.

#include "aih_kv.h"

#include <algorithm>

namespace {

using aih_kv::f4;
using aih_kv::kMaxSeqs;
using aih_kv::u4;
using aih_kv::wave_max;
using aih_kv::wave_scan;

// ---------------------------------------------------------------- block tables and slot maps
// Sums of counts that stop at kFull, which is above every value that they are
// compared with (aih_kv_plan refuses larger ones).  (Stopped addition of
// non-negative numbers is associative, so it can be scanned.)
constexpr uint32_t kFull = 0x7FFFFFFFu;

__device__ __forceinline__ uint32_t add_full(uint32_t a, uint32_t b) { return min(a + b, kFull); }

// Inclusive scans of v and u over the threads of a workgroup, and their totals.
// red: two words of LDS a wave.
__device__ __forceinline__ void scan_pair(uint32_t &v, uint32_t &u, uint32_t (*red)[16], uint32_t &v_total,
                                          uint32_t &u_total)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
    v = wave_scan(v, add_full);
    u = wave_scan(u, add_full);
    __syncthreads();   // the last use of red
    if (lane == 63) {
        red[0][w] = v;
        red[1][w] = u;
    }
    __syncthreads();
    uint32_t v_before = 0, u_before = 0;
    v_total = u_total = 0;
    for (int i = 0; i < waves; ++i) {
        if (i == w) {
            v_before = v_total;
            u_before = u_total;
        }
        v_total = add_full(v_total, red[0][i]);
        u_total = add_full(u_total, red[1][i]);
    }
    v = add_full(v, v_before);
    u = add_full(u, u_before);
}

// The request of row r (or of block r): the last s with firsts[s] <= r, for
// ascending firsts with firsts[0] <= r.
template <typename T>
__device__ __forceinline__ int request_of(const T *firsts, int n, T r)
{
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (firsts[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

struct PlanArgs {
    const int32_t *lens, *n_new;
    int32_t *tables;
    const int32_t *free_blocks, *n_free;
    int32_t *new_lens, *new_n_free, *starts, *slots, *positions, *refused;
    int32_t n_seqs, width, shift, n_blocks, rows;
};

__device__ __forceinline__ int32_t slot_of(const PlanArgs &a, int32_t id, int32_t pos)
{
    return id >= 0 && id < a.n_blocks ? (id << a.shift) + (pos & ((1 << a.shift) - 1)) : -1;
}

// One workgroup of up to 1024 threads: two rounds of scans over the requests
// (blocks needed and rows asked for; rows and blocks granted), then, with
// `place`, the rows: each finds its request by bisection, takes its block from the
// table or, a new one, off the stack, and the first of a block writes the table's
// entry, so nothing waits for what another thread stores.  Else the blocks alone, and
// place_kernel the rows.  A decode step's plan reads 512 bytes for 64 requests: a launch and four
// memory round trips (lens, stack or table, and the stores): 2.8 us, an empty
// launch being 1.75.  256 prompts of 40088 rows in all: 5.3 us, and 4.2 in
// place_kernel.
__global__ void __launch_bounds__(1024)
plan_kernel(PlanArgs a, int place)
{
    __shared__ int32_t starts[kMaxSeqs + 1];
    __shared__ uint32_t blocks[kMaxSeqs];   // blocks handed out before request s
    __shared__ int32_t old[kMaxSeqs];       // its length before
    __shared__ uint32_t red[2][16];
    __shared__ int32_t n_refused;
    const int tid = threadIdx.x, threads = blockDim.x;
    const int32_t bt = 1 << a.shift;
    const uint32_t n_free = (uint32_t)min(max(*a.n_free, 0), a.n_blocks);
    if (tid == 0) n_refused = 0;
    uint32_t need_before = 0, asked_before = 0, rows_before = 0, taken = 0;
    for (int base = 0; base < a.n_seqs; base += threads) {
        const int s = base + tid;
        int32_t len = 0, n = 0;
        const bool is = s < a.n_seqs;
        if (is) {
            len = a.lens[s];
            n = a.n_new[s];
        }
        const bool valid = len >= 0 && n >= 0 && (int64_t)len + n <= (int64_t)a.width << a.shift;
        uint32_t need = valid ? (uint32_t)((((int64_t)len + n + bt - 1) >> a.shift) - (((int64_t)len + bt - 1) >> a.shift)) : 0u;
        uint32_t need_upto = need, asked = valid ? (uint32_t)n : 0u, need_total, asked_total;
        scan_pair(need_upto, asked, red, need_total, asked_total);
        need_upto = add_full(need_upto, need_before);
        asked = add_full(asked, asked_before);
        need_before = add_full(need_before, need_total);
        asked_before = add_full(asked_before, asked_total);
        const bool ok = valid && (n == 0 || ((need == 0 || need_upto <= n_free) && asked <= (uint32_t)a.rows));
        if (is && !ok) atomicAdd(&n_refused, 1);
        if (!ok || !is) n = need = 0;
        // (granted requests that need blocks come before refused ones that do: these sums are exact)
        uint32_t end = (uint32_t)n, blocks_upto = need, end_total, blocks_total;
        scan_pair(end, blocks_upto, red, end_total, blocks_total);
        if (is) {
            starts[s] = (int32_t)(rows_before + end) - n;
            blocks[s] = taken + blocks_upto - need;
            old[s] = len;
            a.new_lens[s] = len + n;
            a.starts[s] = starts[s];
        }
        rows_before += end_total;
        taken += blocks_total;
    }
    if (tid == 0) starts[a.n_seqs] = a.starts[a.n_seqs] = (int32_t)rows_before;
    __syncthreads();
    if (tid == 0) {
        *a.new_n_free = (int32_t)(n_free - taken);
        *a.refused = n_refused;
    }
    const int32_t top = (int32_t)n_free - 1;
    if (!place) {
        for (uint32_t j = tid; j < taken; j += threads) {
            const int s = request_of(blocks, a.n_seqs, j);
            const int32_t at = (int32_t)(((int64_t)old[s] + bt - 1) >> a.shift) + (int32_t)(j - blocks[s]);
            a.tables[(int64_t)s * a.width + at] = a.free_blocks[top - (int32_t)j];
        }
        return;
    }
    for (int32_t r = tid; r < a.rows; r += threads) {
        int32_t slot = -1, pos = -1;
        if (r < (int32_t)rows_before) {
            const int s = request_of(starts, a.n_seqs, r);
            pos = old[s] + (r - starts[s]);
            const int32_t b = pos >> a.shift, had = (int32_t)(((int64_t)old[s] + bt - 1) >> a.shift);
            int32_t *entry = a.tables + (int64_t)s * a.width + b;
            const int32_t id = *(b < had ? entry : a.free_blocks + (top - (int32_t)blocks[s] - (b - had)));
            if (b >= had && (pos & (bt - 1)) == 0) *entry = id;
            slot = slot_of(a, id, pos);
        }
        a.slots[r] = slot;
        a.positions[r] = pos;
    }
}

// The rows of a plan, where they are too many for its one workgroup: a thread a
// row, which finds its request by bisection of the starts (cached).
__global__ void __launch_bounds__(256)
place_kernel(PlanArgs a)
{
    const int32_t total = a.starts[a.n_seqs];
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * 256) {
        int32_t slot = -1, pos = -1;
        if (r < total) {
            const int s = request_of(a.starts, a.n_seqs, (int32_t)r);
            pos = a.new_lens[s] - (a.starts[s + 1] - (int32_t)r);
            slot = slot_of(a, a.tables[(int64_t)s * a.width + (pos >> a.shift)], pos);
        }
        a.slots[r] = slot;
        a.positions[r] = pos;
    }
}

// One workgroup: a wave counts a request's entries that are blocks, a scan says
// where they go on the stack, and the wave moves them there.  What it takes are
// dependent reads of the tables, twice: 4 requests of up to 31 blocks 3.1 us, all
// of 64 requests with 16500 blocks 21 us (a server releases a few at a time).
__global__ void __launch_bounds__(1024)
release_kernel(int32_t *lens, int32_t n_seqs, int32_t *tables, int32_t width, int32_t shift, int32_t n_blocks,
               const int32_t *done, int32_t *free_blocks, int32_t *n_free)
{
    __shared__ uint32_t first[kMaxSeqs];   // a request's blocks; then where they go on the stack
    __shared__ uint32_t red[2][16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t had = (uint32_t)min(max(*n_free, 0), n_blocks);
    auto blocks_of = [&](int s) {
        if (done && !done[s]) return 0;
        const int64_t b = ((int64_t)max(lens[s], 0) + (1 << shift) - 1) >> shift;
        return (int32_t)min(b, (int64_t)width);
    };
    auto valid = [&](int32_t id) { return id >= 0 && id < n_blocks; };
    for (int s = w; s < n_seqs; s += 16) {   // one wave counts a request's entries
        const int32_t n = blocks_of(s);
        uint32_t c = 0;
        for (int j = 0; j < n; j += 64)
            c += (uint32_t)__popcll(__ballot(j + lane < n && valid(tables[(int64_t)s * width + min(j + lane, n - 1)])));
        if (lane == 0) first[s] = c;
    }
    __syncthreads();
    uint32_t before = 0;
    for (int base = 0; base < n_seqs; base += 1024) {
        const int s = base + tid;
        const uint32_t c = s < n_seqs ? first[s] : 0u;
        uint32_t up = c, none = 0, total, zero;
        scan_pair(up, none, red, total, zero);
        if (s < n_seqs) first[s] = add_full(up, before) - c;
        before = add_full(before, total);
    }
    __syncthreads();
    for (int s = w; s < n_seqs; s += 16) {
        const int32_t n = blocks_of(s);
        uint32_t at = add_full(had, first[s]);
        for (int j = 0; j < n; j += 64) {
            int32_t *entry = tables + (int64_t)s * width + min(j + lane, n - 1);
            const int32_t id = *entry;
            const bool is = j + lane < n && valid(id);
            const unsigned long long all = __ballot(is);
            const uint32_t to = at + (uint32_t)__popcll(all & ((1ull << lane) - 1));
            if (is && to < (uint32_t)n_blocks) free_blocks[to] = id;
            if (j + lane < n) *entry = -1;
            at += (uint32_t)__popcll(all);
        }
        if (lane == 0 && (!done || done[s])) lens[s] = 0;
    }
    __syncthreads();
    if (tid == 0) *n_free = (int32_t)min(add_full(had, before), (uint32_t)n_blocks);
}

// ---------------------------------------------------------------- the formats
template <int FMT>
struct Format;

template <>
struct Format<AIH_KV_INT8> {
    static constexpr float kMost = 127.0f;
    // amax / 127, at least the smallest normal number
    __device__ static __forceinline__ float first_scale(float amax) { return fmaxf(amax / 127.0f, 0x1p-126f); }
    // The code nearest to x / s, ties to even, from c = rint(x * inv), which is right or, beside a tie, off by one: r = x -
    // c s is exact (its bits fit: a multiple of the smaller ulp, at most about s / 2), and 2 r against s says which.
    __device__ static __forceinline__ uint32_t exact(float x, float s, float c)
    {
        const float r2 = 2.0f * __builtin_fmaf(-c, s, x);
        const bool odd = ((int)c & 1) != 0;
        if (r2 > s || (r2 == s && odd)) c += 1.0f;
        else if (r2 < -s || (r2 == -s && odd)) c -= 1.0f;
        return (uint32_t)(int)fminf(fmaxf(c, -127.0f), 127.0f) & 0xFF;
    }
    // Four codes into a word.  t = x * inv is within 2^-16 of the quotient, which is at most 127 (to 2^-17): only where t
    // lies 2^-15 or less from a tie can its rounding be wrong.  Added to 3 2^22 it is rounded to its code in the low byte.
    __device__ static __forceinline__ uint32_t pack(const float *x, float s, float inv)
    {
        constexpr float magic = 12582912.0f;
        float m[4], off = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t = x[i] * inv;
            m[i] = t + magic;
            off = fmaxf(off, fabsf(t - (m[i] - magic)));
        }
        if (off >= 0.5f - 0x1p-15f) {
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) w |= exact(x[i], s, m[i] - magic) << (8 * i);
            return w;
        }
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(m[1]), __float_as_uint(m[0]), 0x0C0C0400u);
        return lo | __builtin_amdgcn_perm(__float_as_uint(m[3]), __float_as_uint(m[2]), 0x04000C0Cu);
    }
    // the codes of a word times f = 2^-d, rounded
    __device__ static __forceinline__ uint32_t shrink(uint32_t w, float f)
    {
        uint32_t o = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o |= (uint32_t)((int)__builtin_rintf((float)(int8_t)(w >> (8 * i)) * f) & 0xFF) << (8 * i);
        return o;
    }
    __device__ static __forceinline__ float value(uint32_t byte) { return (float)(int8_t)byte; }
};

template <>
struct Format<AIH_KV_E4M3> {
    static constexpr float kMost = 448.0f;
    // the smallest power of two s with amax <= 448 s = 0.875 2^9 s
    __device__ static __forceinline__ float first_scale(float amax)
    {
        const float m = __builtin_amdgcn_frexp_mantf(amax);   // [0.5, 1)
        const int e = __builtin_amdgcn_frexp_expf(amax);
        return ldexpf(1.0f, max(e - (m <= 0.875f ? 9 : 8), -126));
    }
    // x / s is exact (s a power of two, 1 / s too) up to what lies far below the smallest code
    __device__ static __forceinline__ uint32_t pack(const float *x, float s, float inv)
    {
        (void)s;
        int w = 0;
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, w, true);
        return (uint32_t)w;
    }
    __device__ static __forceinline__ uint32_t shrink(uint32_t v, float f)
    {
        const float x[4] = {__builtin_amdgcn_cvt_f32_fp8((int)v, 0), __builtin_amdgcn_cvt_f32_fp8((int)v, 1),
                            __builtin_amdgcn_cvt_f32_fp8((int)v, 2), __builtin_amdgcn_cvt_f32_fp8((int)v, 3)};
        return pack(x, 0.0f, f);
    }
    __device__ static __forceinline__ float value(uint32_t byte) { return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0); }
};

// ---------------------------------------------------------------- append
struct AppendArgs {
    uint8_t *k, *v;
    float *ks, *vs;
    const float *K, *V;
    int64_t ldk, ldv;
    const int32_t *slots;
    int64_t rows;
    int32_t heads, n_blocks, shift;   // KV heads; log2 of block_tokens
    // the rotation: table null for none
    float *Q;
    int64_t ldq;
    const int32_t *positions;
    const float *table;
    int32_t table_rows, q_heads;
    int32_t run_groups, q_groups;   // workgroups of the keys and values, and behind them those that rotate Q
};

// Two rotation pairs of a row at position p, dimensions d .. d + 3 (d % 4 == 0) of its head.
template <int D>
__device__ __forceinline__ f4 rotate(const f4 x, const float *__restrict__ table, int32_t p, int d)
{
    const f4 cs = *reinterpret_cast<const f4 *>(table + (int64_t)p * D + d);   // cos, sin of pairs d / 2 and d / 2 + 1
    return f4{x[0] * cs[0] - x[1] * cs[1], x[0] * cs[1] + x[1] * cs[0], x[2] * cs[2] - x[3] * cs[3],
              x[2] * cs[3] + x[3] * cs[2]};
}

// The scale of a block for new values of largest magnitude `top` (bits of
// |x|), and the power of two d that its present codes are divided by.
struct Scale {
    float s, inv;
    int d;
};

template <int FMT>
__device__ __forceinline__ Scale next_scale(uint32_t top, float old, bool fresh)
{
    typedef Format<FMT> F;
    Scale o{fresh ? 0.0f : old, 0.0f, 0};
    const float amax = __uint_as_float(top);
    if (top >= 0x7F800000u || o.s != o.s) {
        o.s = __uint_as_float(0x7FC00000u);
        return o;
    }
    if (top != 0 && o.s == 0.0f) o.s = F::first_scale(amax);
    else if (top != 0) {
        // the smallest d with amax <= most 2^d, from the fractions and exponents of the two (most is exact)
        const double most = (double)F::kMost * (double)o.s;
        const int d = __builtin_amdgcn_frexp_expf(amax) - __builtin_amdgcn_frexp_exp(most) +
                      ((double)__builtin_amdgcn_frexp_mantf(amax) > __builtin_amdgcn_frexp_mant(most) ? 1 : 0);
        o.d = max(d, 0);
        o.s = ldexpf(o.s, o.d);
    }
    if (o.s != 0.0f) o.inv = 1.0f / o.s;
    return o;
}

// One token into a block, keys or values, by one wave: lane l holds dimensions
// 4 l .. 4 l + 3 (x; lanes past the head's nothing).  codes, scale: the block's of
// this head; o: the token's offset.
template <int FMT, int D, bool KEYS>
__device__ __forceinline__ void append_one(uint8_t *codes, float *scale, float old, const f4 x, int o, int bt)
{
    typedef Format<FMT> F;
    constexpr int C = D / 64;
    const int lane = threadIdx.x & 63;
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) top = max(top, __float_as_uint(x[u]) & 0x7FFFFFFFu);
    const Scale s = next_scale<FMT>(wave_max(top), old, o == 0);
    const bool bad = s.s != s.s;
    if (lane == 0) *scale = s.s;
    if (o == 0 || s.d) {   // the rest of the block: started anew, or rescaled
        const float f = ldexpf(1.0f, -s.d);
        for (int u = lane; u < bt * D / 16; u += 64) {
            u4 *to = reinterpret_cast<u4 *>(codes) + u;
            u4 w = {0u, 0u, 0u, 0u};
            if (o) {
                w = *to;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = F::shrink(w[i], f);
            }
            *to = w;
        }
        __threadfence_block();   // these stores before the token's, which go over them
    }
    if (4 * lane < D) {
        const float xs[4] = {x[0], x[1], x[2], x[3]};
        const uint32_t w = bad ? 0u : F::pack(xs, s.s, s.inv);
        uint8_t *group = codes + (o >> 4) * 16 * D;
        if constexpr (KEYS) {
            const int d = 4 * lane, t = (o >> 2) & 3, r = o & 3;
            *reinterpret_cast<uint32_t *>(group + (((t * C + d / 64) * 4 + r) * 4 + d % 64 / 16) * 16 + d % 16) = w;
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) group[(4 * lane + u) * 16 + (o & 15)] = (uint8_t)(w >> (8 * u));
        }
    }
}

// Workgroup (head fastest): one KV head and the runs of rows of one block that
// begin among rpw rows; the last workgroups rotate Q, 1024 units of four values
// each.  A run's values are read twice, for their largest magnitude and
// to be rounded; the second time they come from the caches.  Every 16-byte
// unit of the block belongs to one thread, which reads what it keeps of it
// (rescaled where the scale grew) and writes it once.  A run of one row, as in
// a decode step, is done by two waves without LDS (append_one), two such runs
// at a time.  Bound by memory: 5 waves a SIMD keep two rows each of keys and
// values in flight.  18000 rows of 8 heads, D = 128, blocks of 32, 184 MB: 52 us
// for either format, 3.5 TB/s (a large copy reaches 4.8 on the card); one read with
// the rows held in registers takes 127 of them and 53 us.  With Q of 32
// heads 774 MB and 186 us, 4.2 TB/s, at 4 waves a SIMD: fewer rows of Q in flight suit
// the memory better (at 5 waves 206 us; 1000 single tokens 18.9 against 16.5, smaller
// calls the same).  One token 3.6 us, a launch.
template <int FMT, int D, bool ROPE>
__global__ void __launch_bounds__(256, ROPE ? 3 : 5)
append_kernel(AppendArgs a, int rpw)
{
    typedef Format<FMT> F;
    constexpr int NQ = D / 4, C = D / 64;
    __shared__ int32_t row_of[256];      // the row (from the run's first) whose token is at an offset of the block
    __shared__ uint32_t top[2][4];
    const int tid = threadIdx.x, lane = tid & 63;
    auto placed = [&](int64_t r) {   // the position of row r allows it to be stored
        if constexpr (!ROPE) return true;
        const int32_t p = a.positions[r];
        return p >= 0 && p < a.table_rows;
    };
    if (ROPE && (int)blockIdx.x >= a.run_groups) {
        const uint32_t per = (uint32_t)a.q_heads * NQ;   // units of a row
        const int64_t u0 = (int64_t)((int)blockIdx.x - a.run_groups) * 1024, q0 = u0 / per;
        const uint32_t rest = (uint32_t)(u0 - q0 * per);
        f4 x[4], *at[4];
        int32_t p[4];
        bool is[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // no branches: all loads are in flight at once
            const uint32_t u = rest + 256 * i + tid;
            const int64_t r = min(q0 + u / per, a.rows - 1);
            is[i] = q0 + u / per < a.rows;
            p[i] = a.positions[r];
            at[i] = reinterpret_cast<f4 *>(a.Q + r * a.ldq) + u % per;
            x[i] = *at[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = p[i] >= 0 && p[i] < a.table_rows;
            x[i] = rotate<D>(x[i], a.table, in ? p[i] : 0, 4 * (tid % NQ));
            is[i] = is[i] && in;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (is[i]) *at[i] = x[i];
        return;
    }
    const int head = (int)blockIdx.x % a.heads, bt = 1 << a.shift;
    const int64_t r0 = (int64_t)((int)blockIdx.x / a.heads) * rpw;
    auto block_of = [&](int64_t r) {   // the block of row r, -1 for none
        const int32_t slot = a.slots[min(max(r, (int64_t)0), a.rows - 1)];
        const int32_t b = slot < 0 || r < 0 || r >= a.rows ? -1 : slot >> a.shift;
        return b < a.n_blocks ? b : -1;
    };
    // The blocks of rows r0 - 1 .. r0 + 62, the same in every wave: which of the rows r0 .. begin a run
    // (rpw < 64), and how far the first ones reach.
    const int32_t mine = block_of(r0 - 1 + lane), left = __shfl_up(mine, 1);
    unsigned long long runs = __ballot(lane >= 1 && lane <= rpw && mine >= 0 && mine != left);
    int pair = 0;   // the two waves that do the next run of one row
    while (runs) {
        const int first = __builtin_ctzll(runs);
        runs &= runs - 1;
        const int64_t r = r0 - 1 + first;
        const int32_t block = __builtin_amdgcn_readlane(mine, first);
        // the run: rows r .. r + n - 1
        const unsigned long long others = __ballot(lane > first && mine != block);
        int64_t n = others ? __builtin_ctzll(others) - first : 64 - first;
        while (!others) {
            const unsigned long long more = __ballot(block_of(r + n + lane) != block);
            n += more ? __builtin_ctzll(more) : 64;
            if (more) break;
        }
        const int64_t at = (int64_t)block * a.heads + head;
        const float old_k = a.ks[at], old_v = a.vs[at];
        const float *K = a.K + r * a.ldk + head * D, *V = a.V + r * a.ldv + head * D;
        auto key4 = [&](int64_t j, int d) {
            f4 x = *reinterpret_cast<const f4 *>(K + j * a.ldk + d);
            if constexpr (ROPE) x = rotate<D>(x, a.table, a.positions[r + j], d);
            return x;
        };
        uint8_t *kb = a.k + at * bt * D, *vb = a.v + at * bt * D;
        if (n == 1) {
            const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
            const bool ours = w >> 1 == pair;
            pair ^= 1;
            if (ours && placed(r)) {
                const int o = __builtin_amdgcn_readfirstlane(a.slots[r]) & (bt - 1);
                f4 x = {0.f, 0.f, 0.f, 0.f};
                if (4 * lane < D) x = w & 1 ? *reinterpret_cast<const f4 *>(V + 4 * lane) : key4(0, 4 * lane);
                if (w & 1) append_one<FMT, D, false>(vb, a.vs + at, old_v, x, o, bt);
                else append_one<FMT, D, true>(kb, a.ks + at, old_k, x, o, bt);
            }
            continue;
        }
        __syncthreads();   // the LDS of the run before
        row_of[tid] = -1;
        __syncthreads();
        for (int64_t j = tid; j < n; j += 256)
            if (placed(r + j)) atomicMax(&row_of[a.slots[r + j] & (bt - 1)], (int32_t)min<int64_t>(j, 0x7FFFFFFF));
        // the largest magnitudes, two rows in flight; rows past the last and those that are not placed read another's
        uint32_t tk = 0, tv = 0;
        for (int64_t j0 = tid / NQ; j0 < n; j0 += 2 * (256 / NQ)) {
            const int d = 4 * (tid % NQ);
            f4 x[2], y[2];
            bool is[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t j = min(j0 + i * (256 / NQ), n - 1);
                is[i] = j0 + i * (256 / NQ) < n;
                x[i] = *reinterpret_cast<const f4 *>(K + j * a.ldk + d);
                y[i] = *reinterpret_cast<const f4 *>(V + j * a.ldv + d);
                if constexpr (ROPE) {
                    const int32_t p = a.positions[r + j];
                    const bool in = p >= 0 && p < a.table_rows;
                    is[i] = is[i] && in;
                    x[i] = rotate<D>(x[i], a.table, in ? p : 0, d);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    tk = max(tk, is[i] ? __float_as_uint(x[i][u]) & 0x7FFFFFFFu : 0u);
                    tv = max(tv, is[i] ? __float_as_uint(y[i][u]) & 0x7FFFFFFFu : 0u);
                }
        }
        tk = wave_max(tk);
        tv = wave_max(tv);
        if (lane == 0) {
            top[0][tid >> 6] = tk;
            top[1][tid >> 6] = tv;
        }
        __syncthreads();
        tk = max(max(top[0][0], top[0][1]), max(top[0][2], top[0][3]));
        tv = max(max(top[1][0], top[1][1]), max(top[1][2], top[1][3]));
        const bool fresh = row_of[0] >= 0;
        const Scale sk = next_scale<FMT>(tk, old_k, fresh), sv = next_scale<FMT>(tv, old_v, fresh);
        if (tid == 0) a.ks[at] = sk.s;
        if (tid == 64) a.vs[at] = sv.s;
        const bool bad_k = sk.s != sk.s, bad_v = sv.s != sv.s;
        const float fk = ldexpf(1.0f, -sk.d), fv = ldexpf(1.0f, -sv.d);
        for (int u = tid; u < bt * D / 16; u += 256) {
            // key unit u: 16 dimensions of one token; value unit u: 16 tokens at one dimension.  What both need is
            // loaded before either is rounded.
            const int g = u & 3, rr = (u >> 2) & 3, c = (u >> 4) % C, t = (u >> 4) / C % 4, grp = u / D, d = u % D;
            const int32_t jk = row_of[16 * grp + 4 * t + rr];
            u4 *kt = reinterpret_cast<u4 *>(kb) + u, *vt = reinterpret_cast<u4 *>(vb) + u;
            const bool new_k = jk >= 0 && !bad_k, keep_k = jk < 0 && !fresh;   // round it; leave or rescale it
            uint32_t new_v = 0;                                                // bit i: token i is new
#pragma unroll
            for (int i = 0; i < 16; ++i) new_v |= row_of[16 * grp + i] >= 0 ? 1u << i : 0u;
            const bool keep_v = !fresh && new_v != 0xFFFFu;
            u4 wk = {0u, 0u, 0u, 0u}, wv = {0u, 0u, 0u, 0u};
            if (keep_k && sk.d) {
                wk = *kt;
#pragma unroll
                for (int i = 0; i < 4; ++i) wk[i] = F::shrink(wk[i], fk);
            }
            if (keep_v && (new_v || sv.d)) {
                wv = *vt;
                if (sv.d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) wv[i] = F::shrink(wv[i], fv);
            }
            // a word of either at a time: five loads in flight, few registers (with all twenty 167, and a third of the waves)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f4 x = {0.f, 0.f, 0.f, 0.f};
                float y[4];
                uint32_t keep = 0;
                if (new_k) x = key4(jk, 64 * c + 16 * g + 4 * i);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int32_t j = row_of[16 * grp + 4 * i + b];
                    y[b] = 0.f;
                    if (j < 0) keep |= 0xFFu << (8 * b);
                    else if (!bad_v) y[b] = V[(int64_t)j * a.ldv + d];
                }
                if (new_k) {
                    const float xs[4] = {x[0], x[1], x[2], x[3]};
                    wk[i] = F::pack(xs, sk.s, sk.inv);
                }
                if (keep != 0xFFFFFFFFu) wv[i] = (wv[i] & keep) | (F::pack(y, sv.s, sv.inv) & ~keep);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!keep_k || sk.d) *kt = wk;
            if (new_v || !keep_v || sv.d) *vt = wv;
        }
    }
}

// ---------------------------------------------------------------- read
// Workgroup (x, y): rows 16 x .. 16 x + 15 of KV head y; consecutive lanes
// write consecutive floats.  A token's values lie 16 bytes apart, and the 16
// rows, when they are one group of tokens, find them in the same lines.  Bound by
// memory: 18000 rows of 8 heads, D = 128, 184 MB: 57 us, 3.2 TB/s; with all loads
// of 16 rows ahead 4740 rows take 14.4 instead of 16.1 us, but single rows 5.4
// instead of 4.2.
template <int FMT, int D>
__global__ void __launch_bounds__(256)
read_kernel(const uint8_t *__restrict__ k, const uint8_t *__restrict__ v, const float *__restrict__ ks,
            const float *__restrict__ vs, const int32_t *__restrict__ slots, int64_t rows, int32_t heads,
            int32_t n_blocks, int32_t shift, float *__restrict__ K, int64_t ldk, float *__restrict__ V, int64_t ldv)
{
    typedef Format<FMT> F;
    constexpr int C = D / 64, NQ = D / 4;
    const int head = blockIdx.y;
    for (int i = threadIdx.x; i < 16 * NQ; i += 256) {
        const int64_t r = (int64_t)blockIdx.x * 16 + i / NQ;
        if (r >= rows) continue;
        const int d = 4 * (i % NQ);
        const int32_t slot = slots[r], b = slot >> shift;
        f4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
        if (slot >= 0 && b < n_blocks) {
            const int64_t at = (int64_t)b * heads + head;
            const int o = slot & ((1 << shift) - 1), t = (o >> 2) & 3, rr = o & 3;
            const int64_t base = (at << shift) * D + (int64_t)(o >> 4) * 16 * D;
            const uint32_t w = *reinterpret_cast<const uint32_t *>(
                k + base + (((t * C + d / 64) * 4 + rr) * 4 + d % 64 / 16) * 16 + d % 16);
            const float sk = ks[at], sv = vs[at];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                x[u] = F::value(w >> (8 * u) & 0xFF) * sk;
                y[u] = F::value(v[base + (d + u) * 16 + (o & 15)]) * sv;
            }
        }
        float *kr = K + r * ldk + head * D + d, *vr = V + r * ldv + head * D + d;
        *reinterpret_cast<f4 *>(kr) = x;
        *reinterpret_cast<f4 *>(vr) = y;
    }
}

// Up to this many rows a plan's one workgroup also places them; more are
// placed by a second launch over the whole device.
constexpr int64_t kPlaceRows = 4096;
template <int FMT, int D>
void launch_append(const AppendArgs &a, bool rope, int rpw, hipStream_t stream)
{
    const dim3 grid((unsigned)(a.run_groups + a.q_groups));
    if (rope) hipLaunchKernelGGL((append_kernel<FMT, D, true>), grid, dim3(256), 0, stream, a, rpw);
    else hipLaunchKernelGGL((append_kernel<FMT, D, false>), grid, dim3(256), 0, stream, a, rpw);
}

int append(aih_ctx *ctx, const aih_kv_cache *kv, AppendArgs a, bool rope)
{
    const int64_t wide = (int64_t)kv->n_kv_heads * kv->head_dim;
    if (!a.K || !a.V || !a.slots || a.rows < 0 || a.ldk < wide || a.ldv < wide || a.ldk % 4 || a.ldv % 4 ||
        !aih_kv::aligned16(a.K) || !aih_kv::aligned16(a.V))
        return AIH_E_INVALID;
    if (a.rows == 0) return AIH_OK;
    if (a.rows > 0x7FFFFFFF || a.q_heads > aih_kv::kMaxHeads) return AIH_E_LIMIT;
    a.k = static_cast<uint8_t *>(kv->k);
    a.v = static_cast<uint8_t *>(kv->v);
    a.ks = kv->k_scale;
    a.vs = kv->v_scale;
    a.heads = kv->n_kv_heads;
    a.n_blocks = kv->n_blocks;
    a.shift = aih_kv::log2_of(kv->block_tokens);
    // Rows whose runs one workgroup does.  A prompt's runs are long, and the workgroups of all rows but their first would
    // do nothing; single tokens are a run each, done two at a time.  Append alone, us at 1 / 2 / 4 / 8 / 16 / 32 rows, 8
    // heads, D = 128, int8, blocks of 16: 32 single tokens 3.5 / 3.8 / 5.1 / 7.8 / 12.9 / 23.6, 200 of them 5.5 / 5.3 / 6.2
    // / 8.3 / 13.5 / 24.0, 64 x 4 10.1 / 6.4 / 6.1 / 9.0 / 15.3 / 28.2, 200 x 4 24.9 / 14.8 / 9.9 / 11.2 / 18.2 / 30.4, a
    // prompt of 500 9.4 / 8.1 / 7.4 / 6.8 / 6.4 / 10.1, of 1000 14.4 / 12.7 / 11.6 / 7.7 / 7.1 / 10.4, of 2000 25.8 / 22.3
    // / 19.7 / 13.0 / 9.4 / 12.7; 18000 rows of prompts in blocks of 32 177 / 131 / 115 / 116 / 65 / 53.
    const int rpw = (int)std::min<int64_t>(a.rows / 128 + 1, std::min(kv->block_tokens, 32));
    const int64_t runs = (a.rows + rpw - 1) / rpw * a.heads;
    const int64_t queries = rope ? (a.rows * a.q_heads * (kv->head_dim / 4) + 1023) / 1024 : 0;
    if (runs + queries > aih_kv::kMaxGroups) return AIH_E_LIMIT;
    a.run_groups = (int32_t)runs;
    a.q_groups = (int32_t)queries;
    aih_kv::DeviceGuard guard(ctx->device);
    AIH_TRY(guard.status);
    const bool i8 = kv->format == AIH_KV_INT8;
    switch (kv->head_dim) {
    case 64: i8 ? launch_append<AIH_KV_INT8, 64>(a, rope, rpw, ctx->stream) : launch_append<AIH_KV_E4M3, 64>(a, rope, rpw, ctx->stream); break;
    case 128: i8 ? launch_append<AIH_KV_INT8, 128>(a, rope, rpw, ctx->stream) : launch_append<AIH_KV_E4M3, 128>(a, rope, rpw, ctx->stream); break;
    default: i8 ? launch_append<AIH_KV_INT8, 256>(a, rope, rpw, ctx->stream) : launch_append<AIH_KV_E4M3, 256>(a, rope, rpw, ctx->stream); break;
    }
    return aih_launch_status();
}

template <int FMT, int D>
void launch_read(aih_ctx *ctx, const aih_kv_cache *kv, const int32_t *slots, int64_t rows, float *K, int64_t ldk,
                 float *V, int64_t ldv)
{
    hipLaunchKernelGGL((read_kernel<FMT, D>), dim3((unsigned)((rows + 15) / 16), (unsigned)kv->n_kv_heads), dim3(256),
                       0, ctx->stream, static_cast<const uint8_t *>(kv->k), static_cast<const uint8_t *>(kv->v),
                       kv->k_scale, kv->v_scale, slots, rows, kv->n_kv_heads, kv->n_blocks,
                       aih_kv::log2_of(kv->block_tokens), K, ldk, V, ldv);
}

}  // namespace

extern "C" {

int64_t aih_kv_cache_bytes(const aih_kv_cache *kv)
{
    const int rc = aih_kv::check_shape(kv);
    if (rc) return rc;
    return (int64_t)kv->n_blocks * kv->block_tokens * kv->n_kv_heads * kv->head_dim;
}

int aih_kv_plan(aih_ctx *ctx, const int32_t *lens, const int32_t *n_new, int32_t n_seqs, int32_t *tables,
                int32_t table_width, int32_t block_tokens, int32_t n_blocks, const int32_t *free_blocks,
                const int32_t *n_free, int32_t *new_lens, int32_t *new_n_free, int32_t *starts, int32_t *slots,
                int32_t *positions, int64_t rows, int32_t *refused)
{
    if (!ctx || !lens || !n_new || !tables || !free_blocks || !n_free || !new_lens || !new_n_free || !starts ||
        !slots || !positions || !refused || n_seqs <= 0 || table_width <= 0 || n_blocks <= 0 || rows < 0)
        return AIH_E_INVALID;
    if (block_tokens != 16 && block_tokens != 32 && block_tokens != 64 && block_tokens != 128 && block_tokens != 256)
        return AIH_E_UNSUPPORTED;
    // (a sum of rows that has stopped at kFull has to be above `rows`)
    if (n_seqs > kMaxSeqs || rows >= (int64_t)kFull || (int64_t)n_blocks * block_tokens > 0x7FFFFFFF ||
        (int64_t)table_width * block_tokens > 0x7FFFFFFF)
        return AIH_E_LIMIT;
    aih_kv::DeviceGuard guard(ctx->device);
    AIH_TRY(guard.status);
    PlanArgs a{lens, n_new, tables, free_blocks, n_free, new_lens, new_n_free, starts, slots, positions, refused,
               n_seqs, table_width, aih_kv::log2_of(block_tokens), n_blocks, (int32_t)rows};
    const bool alone = rows <= kPlaceRows;
    // a wave for 64 requests or rows: barriers of few waves are short
    const int64_t threads = std::min<int64_t>(1024, (std::max<int64_t>(n_seqs, alone ? rows : 1024) + 63) / 64 * 64);
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3((unsigned)threads), 0, ctx->stream, a, alone ? 1 : 0);
    if (!alone) {
        const int rc = aih_launch_status();
        if (rc) return rc;
        hipLaunchKernelGGL(place_kernel, dim3((unsigned)std::min<int64_t>((rows + 255) / 256, 8192)), dim3(256), 0,
                           ctx->stream, a);
    }
    return aih_launch_status();
}

int aih_kv_release(aih_ctx *ctx, int32_t *lens, int32_t n_seqs, int32_t *tables, int32_t table_width,
                   int32_t block_tokens, int32_t n_blocks, const int32_t *done, int32_t *free_blocks, int32_t *n_free)
{
    if (!ctx || !lens || !tables || !free_blocks || !n_free || n_seqs <= 0 || table_width <= 0 || n_blocks <= 0)
        return AIH_E_INVALID;
    if (block_tokens != 16 && block_tokens != 32 && block_tokens != 64 && block_tokens != 128 && block_tokens != 256)
        return AIH_E_UNSUPPORTED;
    if (n_seqs > kMaxSeqs || (int64_t)n_blocks * block_tokens > 0x7FFFFFFF ||
        (int64_t)table_width * block_tokens > 0x7FFFFFFF)
        return AIH_E_LIMIT;
    aih_kv::DeviceGuard guard(ctx->device);
    AIH_TRY(guard.status);
    hipLaunchKernelGGL(release_kernel, dim3(1), dim3(1024), 0, ctx->stream, lens, n_seqs, tables, table_width,
                       aih_kv::log2_of(block_tokens), n_blocks, done, free_blocks, n_free);
    return aih_launch_status();
}

int aih_kv_append(aih_ctx *ctx, const aih_kv_cache *kv, const float *K, int64_t ldk, const float *V, int64_t ldv,
                  const int32_t *slots, int64_t rows)
{
    if (!ctx) return AIH_E_INVALID;
    const int rc = aih_kv::check_cache(kv);
    if (rc) return rc;
    AppendArgs a{};
    a.K = K;
    a.V = V;
    a.ldk = ldk;
    a.ldv = ldv;
    a.slots = slots;
    a.rows = rows;
    return append(ctx, kv, a, false);
}

int aih_kv_append_rope(aih_ctx *ctx, const aih_kv_cache *kv, float *Q, int64_t ldq, int32_t n_heads, const float *K,
                       int64_t ldk, const float *V, int64_t ldv, const int32_t *slots, const int32_t *positions,
                       int64_t rows, const float *table, int32_t table_rows)
{
    if (!ctx) return AIH_E_INVALID;
    const int rc = aih_kv::check_cache(kv);
    if (rc) return rc;
    if (!Q || !positions || !table || n_heads <= 0 || table_rows <= 0 || ldq < (int64_t)n_heads * kv->head_dim ||
        ldq % 4 || !aih_kv::aligned16(Q) || !aih_kv::aligned16(table))
        return AIH_E_INVALID;
    AppendArgs a{};
    a.K = K;
    a.V = V;
    a.ldk = ldk;
    a.ldv = ldv;
    a.slots = slots;
    a.rows = rows;
    a.Q = Q;
    a.ldq = ldq;
    a.positions = positions;
    a.table = table;
    a.table_rows = table_rows;
    a.q_heads = n_heads;
    return append(ctx, kv, a, true);
}

int aih_kv_read(aih_ctx *ctx, const aih_kv_cache *kv, const int32_t *slots, int64_t rows, float *K, int64_t ldk,
                float *V, int64_t ldv)
{
    if (!ctx) return AIH_E_INVALID;
    const int rc = aih_kv::check_cache(kv);
    if (rc) return rc;
    const int64_t wide = (int64_t)kv->n_kv_heads * kv->head_dim;
    if (!slots || !K || !V || rows < 0 || ldk < wide || ldv < wide || ldk % 4 || ldv % 4 || !aih_kv::aligned16(K) ||
        !aih_kv::aligned16(V))
        return AIH_E_INVALID;
    if (rows == 0) return AIH_OK;
    if (rows > 16 * aih_kv::kMaxGroups) return AIH_E_LIMIT;
    aih_kv::DeviceGuard guard(ctx->device);
    AIH_TRY(guard.status);
    const bool i8 = kv->format == AIH_KV_INT8;
    switch (kv->head_dim) {
    case 64: i8 ? launch_read<AIH_KV_INT8, 64>(ctx, kv, slots, rows, K, ldk, V, ldv) : launch_read<AIH_KV_E4M3, 64>(ctx, kv, slots, rows, K, ldk, V, ldv); break;
    case 128: i8 ? launch_read<AIH_KV_INT8, 128>(ctx, kv, slots, rows, K, ldk, V, ldv) : launch_read<AIH_KV_E4M3, 128>(ctx, kv, slots, rows, K, ldk, V, ldv); break;
    default: i8 ? launch_read<AIH_KV_INT8, 256>(ctx, kv, slots, rows, K, ldk, V, ldv) : launch_read<AIH_KV_E4M3, 256>(ctx, kv, slots, rows, K, ldk, V, ldv); break;
    }
    return aih_launch_status();
}

}  // extern "C"
