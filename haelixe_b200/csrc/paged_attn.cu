// Attention of one new token per sequence over a paged key/value cache:
// o = sum_j p_j v_j, p = softmax_j(scale q . k_j) over the first len positions
// of the sequence, for G query heads to a key head (G = 1: every head has its own keys).
//
// Every key and value is read once, so the bytes of the cache bound it, and
// the work has to be even over the SMs although lengths differ and are known
// on the device alone. The (sequence, key head, up to HB of its query heads)
// items are cut into tiles of 64 keys, the tiles of all items are numbered in a row,
// each item's after an empty place that stands for the time an item takes
// besides its keys, and every worker (a 4-warp CTA, as many as are resident at
// once) takes an equal run of them. A run that holds all of an item writes its
// result; the others write (max, sum, unnormalised o) to the workspace, at most
// two a worker, and paged_join_kernel joins an item's parts in the order of its
// keys (no atomics: the same call gives the same bits).
//
// Softmax statistics and all sums are f32. A warp keeps a running maximum; in bf16 it
// only moves when a score passes it by 2^8, so that the accumulator is rarely rescaled.
// Positions at or past len are never read: their pages may hold anything.
#include <atomic>
#include <type_traits>

#include "hx_internal.h"
#include "launch.h"
#include "mma_bf16.cuh"
#include "sm100_ptx.cuh"

namespace hx {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kWarpKeys = 16, kTile = kWarps * kWarpKeys;
constexpr int kMaxWorkers = 1024;
// Empty places of an item, where every worker has a tile: 64 sequences of 1 to 8192 keys take 65 us
// without and 50 with 1 or 2; 256 of 1 to 1024 take 62 without, 51 with 1, 55 with 2, 59 with 3. With
// less to do than that none, so that it is spread as far as it goes.
constexpr int kItemPlaces = 1;
constexpr int kLazy = 8;  // log2 growth of the maximum that triggers a rescale
// The weights of the values are 2^shrink_of(len) of the probabilities, so that they add up to less than 1
// and no sum passes the largest value, however large that is; the division by the probabilities' sum takes it
// back. A power of two, so it changes no bit of a result unless values are under 2^-100 or so.
__device__ __forceinline__ int shrink_of(int len) { return __clz(len) - 32 - kLazy; }
// Of normal numbers. (The workers take exp2f, which gives powers of two exactly as well: made of bits, the number is
// no register's own to the compiler, and 64 sequences of 16 heads of 64 take 27.8 us for 26.4.)
__device__ __forceinline__ float power_of_two(int n) { return __int_as_float((127 + n) << 23); }
constexpr float kLn2 = 0.69314718055994530942f;

struct Item {
    int n, h, c;  // sequence, key head, chunk of its query heads
};
// A run's part of an item: tiles [first, first + count) of a sequence of len keys. No tiles: no part.
struct Part {
    Item it;
    int first, count, len, slot;
    bool whole;
};

// Sequences with nothing to read (len <= 0) or longer than their table row (or than 2^31 - 256, so
// that a key past the last tile still is an int) have no tiles and no items; paged_join_kernel
// writes their rows.
__device__ __forceinline__ int tiles_of(const PagedAttn& a, int n) {
    const int64_t len = a.lens[n];
    return len <= 0 || len > (int64_t)a.cache.max_pages * a.cache.page_size || len > 0x7fffff00
               ? 0
               : (int)((len + kTile - 1) / kTile);
}

// Where the work of a call lies: the empty places of an item, the length of a run, the places
// before each sequence. The first worker leaves it in the workspace for the join.
using Plan = PagedPlan;
__device__ __forceinline__ int places_of(int tiles, int empty) { return tiles == 0 ? 0 : tiles + empty; }

__device__ __forceinline__ int64_t div_up(int64_t a, int b) {
    return a >> 31 == 0 ? (int64_t)(((uint32_t)a + (uint32_t)b - 1) / (uint32_t)b) : (a + b - 1) / b;
}

// Sums of two numbers over the block, to every thread.
__device__ __forceinline__ void block_sums(int64_t& x, int64_t& y) {
    __shared__ int64_t sums[2][kWarps];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    if (threadIdx.x % 32 == 0) sums[0][threadIdx.x / 32] = x, sums[1][threadIdx.x / 32] = y;
    __syncthreads();
    x = y = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += sums[0][w], y += sums[1][w];
}

// This worker's run [start, end) and the sequence that holds its first place (each sequence has
// `per` items), with the places before that sequence. False when there is nothing to do.
__device__ __forceinline__ bool find_run(const PagedAttn& a, int per, int64_t& start, int64_t& end, int& n,
                                         int64_t& before, int& empty) {
    __shared__ int64_t warp_sum[kWarps];
    __shared__ int found_n;
    __shared__ int64_t found_before;
    const int mine = (int)threadIdx.x < a.cache.num_seqs ? tiles_of(a, threadIdx.x) : 0;
    int64_t tiles = mine, items = mine > 0;
    for (int i = threadIdx.x + kThreads; i < a.cache.num_seqs; i += kThreads) {
        const int t = tiles_of(a, i);
        tiles += t, items += t > 0;
    }
    block_sums(tiles, items);
    empty = tiles * per >= gridDim.x ? kItemPlaces : 0;
    const int64_t total = (tiles + items * empty) * per, run = div_up(total, gridDim.x);
    const bool first = blockIdx.x == 0;
    if (first && threadIdx.x == 0) *a.plan = Plan{run, empty};
    start = run * blockIdx.x;
    end = min(total, start + run);
    if (start >= end) return false;
    int64_t carry = 0;
    for (int base = 0;; base += kThreads) {
        const int i = base + threadIdx.x;
        const int64_t v = (int64_t)places_of(base == 0 ? mine : i < a.cache.num_seqs ? tiles_of(a, i) : 0, empty) * per;
        int64_t incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
            if ((int)(threadIdx.x % 32) >= o) incl += u;
        }
        if (threadIdx.x % 32 == 31) warp_sum[threadIdx.x / 32] = incl;
        __syncthreads();
        int64_t block = 0, prev = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < (int)(threadIdx.x / 32)) prev += warp_sum[w];
            block += warp_sum[w];
        }
        incl += prev + carry;
        if (incl - v <= start && start < incl) found_n = i, found_before = incl - v;
        if (first && i < a.cache.num_seqs) a.starts[i] = incl - v;
        carry += block;
        __syncthreads();
        if ((start < carry && !first) || base + kThreads >= a.cache.num_seqs) break;
    }
    n = found_n;
    before = found_before;
    return true;
}

// Element offset of key `key` of sequence n in the cache; kNone at or past len, kBad when
// its table entry is no page (such a row comes out as NaN, nothing is read for it).
constexpr int64_t kNone = -1, kBad = -2;
__device__ __forceinline__ int entry_of(const PagedView& c, const int32_t* row, int key, int len) {
    if (key >= len) return 0;
    return row[c.page_shift >= 0 ? key >> c.page_shift : key / c.page_size];
}
__device__ __forceinline__ int64_t offset_of(const PagedView& c, int page, int key, int len) {
    if (key >= len) return kNone;
    if (page < 0 || page >= c.num_pages) return kBad;
    const int slot = c.page_shift >= 0 ? key & (c.page_size - 1) : key % c.page_size;
    return (int64_t)page * c.sp + (int64_t)slot * c.ss;
}

// Not through the read-only path: the kernel may have been launched while the one before it was
// still writing the cache.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 u;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "l"(p));
    return u;
}

// What a warp leaves of its keys of an item, in shared memory: o (unnormalised) in
// [HB][D + pad], (max in log2 units, sum) of each head.
template <int HB, int DP>
struct Parts {
    static constexpr int kRow = DP + 4;
    alignas(16) float o[kWarps][HB * kRow];
    float2 ml[kWarps][HB];
};

__device__ __forceinline__ float safe_max(float m) { return m == -INFINITY ? 0.f : m; }

// A part in the workspace: o of HB heads, then (max, sum) of each, a multiple of 16 bytes.
__host__ __device__ constexpr int part_floats(int HB, int D) { return HB * (D + 4); }

using ptx::ex2;  // to 2^-22, denormals as 0

// Bits whose upper half is the largest bf16 below p > 0; 0 of 0, NaN of NaN.
__device__ __forceinline__ uint32_t below(float p) {
    const uint32_t u = __float_as_uint(p);
    return u - min(u, 1u);
}

// Joins the four warps' parts: the item's output, or the worker's part of it. Four elements a thread.
template <typename T, int HB, int DP>
__device__ __forceinline__ void finish_item(const PagedAttn& a, const Parts<HB, DP>& sp, const Item& it, bool whole,
                                            int len, int slot) {
    const int D = a.cache.D, quads = D / 4;
    const int h0 = it.h * a.G + it.c * HB;
    const int heads = min(HB, a.G - it.c * HB);
    for (int i = threadIdx.x; i < heads * quads; i += kThreads) {
        const int h = i / quads, d = 4 * (i - h * quads);
        float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        float2 ml[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            ml[w] = sp.ml[w][h];
            m = fmaxf(m, ml[w].x);
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(ml[w].x - safe_max(m));
            const float4 u = *reinterpret_cast<const float4*>(&sp.o[w][h * Parts<HB, DP>::kRow + d]);
            l = fmaf(f, ml[w].y, l);
            o[0] = fmaf(f, u.x, o[0]), o[1] = fmaf(f, u.y, o[1]), o[2] = fmaf(f, u.z, o[2]), o[3] = fmaf(f, u.w, o[3]);
        }
        if (whole) {
            T* to = (T*)a.o + (int64_t)it.n * a.o_sn + (int64_t)(h0 + h) * a.o_sh + d;
            struct alignas(4 * sizeof(T)) Four {
                T v[4];
            } four;
#pragma unroll
            for (int e = 0; e < 4; ++e) four.v[e] = T(o[e] / l * power_of_two(-shrink_of(len)));
            if (a.o_vec) {
                *reinterpret_cast<Four*>(to) = four;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) to[e] = four.v[e];
            }
            if (d == 0 && a.lse) a.lse[(int64_t)it.n * a.Hq + h0 + h] = (m + log2f(l)) * kLn2;
        } else {
            float* part = a.part + (int64_t)slot * part_floats(HB, D);
            *reinterpret_cast<float4*>(part + h * D + d) = make_float4(o[0], o[1], o[2], o[3]);
            if (d == 0) reinterpret_cast<float2*>(part + HB * D)[h] = make_float2(m, l);
        }
    }
}

// ---- bf16: the warp's 16 keys as one mma operand --------------------------------
// S^T[16 keys, 8 heads] = K Q^T and O^T[D, 8 heads] += V^T P^T put the keys (or D)
// on the 16-row side and the few query heads on the 8-column side of mma_bf16.
// Both K and V^T fragments come straight from 16-byte global loads, with no
// shared memory: the order of the summed index is free as long as both operands
// use the same one, so lane t's 16 bytes of a key row are its columns of two products,
// and V^T pairs the keys 2t, 2t+1 by two byte permutes. P goes from the first product's
// layout to the second's by an 8x8 transpose, as bf16 hi + lo, so that the
// result carries only its own rounding. hi is the largest bf16 below p, not the nearest, and so lo is
// more than 0: both products with an infinite value then are that infinity (0 times it, or less than 0,
// would make NaN of it; for weights that shrink_of takes under 2^-110 lo is 0 all the same).
// K of the next step is loaded as soon as the scores are taken, V as soon as P V is,
// so one of the two is always in flight. (Loading the worker's next item's while one is joined
// and stored gained nothing: the SM's other workers are in the middle of theirs.)
template <int DC, int NT>
struct AttnBf16 {
    static constexpr int kD = 64 * DC;       // D rounded up; the rest reads as zero
    static constexpr int HB = 8 * NT;
    static constexpr int VC = DC > 2 ? 2 : DC;  // 64-wide chunks of V held at once

    uint4 q[NT][2 * DC], k[2][2 * DC], v[4][VC];
    float acc[NT][DC][4][4];
    float m[NT][2], l[NT][2];
    const PagedAttn& a;
    const __nv_bfloat16 *kh, *vh;
    int g, t;

    __device__ __forceinline__ AttnBf16(const PagedAttn& args) : a(args) {
        g = (threadIdx.x % 32) / 4;
        t = threadIdx.x % 4;
    }

    // WHOLE: the step's keys are all there and of kD elements, so no load asks for anything.
    template <bool WHOLE>
    __device__ __forceinline__ void load_k(int64_t off) {
        const int64_t o0 = __shfl_sync(0xffffffffu, off, g), o1 = __shfl_sync(0xffffffffu, off, g + 8);
        const __nv_bfloat16 *k0 = kh + o0 + 8 * t, *k1 = kh + o1 + 8 * t;
#pragma unroll
        for (int b = 0; b < 2 * DC; ++b) {
            const bool in = WHOLE || 32 * b + 8 * t < a.cache.D;
            k[0][b] = in && (WHOLE || o0 >= 0) ? ld_stream(k0 + 32 * b) : make_uint4(0, 0, 0, 0);
            k[1][b] = in && (WHOLE || o1 >= 0) ? ld_stream(k1 + 32 * b) : make_uint4(0, 0, 0, 0);
        }
    }
    template <bool WHOLE>
    __device__ __forceinline__ void load_v(int64_t off, int c0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t o = __shfl_sync(0xffffffffu, off, 2 * t + (j & 1) + 8 * (j >> 1));
            const __nv_bfloat16* from = vh + o + 64 * c0 + 8 * g;
#pragma unroll
            for (int c = 0; c < VC; ++c)
                v[j][c] = WHOLE || (o >= 0 && 64 * (c0 + c) + 8 * g < a.cache.D) ? ld_stream(from + 64 * c)
                                                                               : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ bool is_whole(int64_t off) const {
        return a.cache.D == kD && __all_sync(0xffffffffu, off >= 0);
    }
    __device__ __forceinline__ void load_k(int64_t off, bool whole) { whole ? load_k<true>(off) : load_k<false>(off); }
    __device__ __forceinline__ void load_v(int64_t off, int c0, bool whole) {
        whole ? load_v<true>(off, c0) : load_v<false>(off, c0);
    }

    __device__ __forceinline__ void run(const Part& part, Parts<HB, kD>& sp) {
        const PagedView& c = a.cache;
        const Item& it = part.it;
        const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, tiles = part.count, len = part.len;
        const int32_t* row = c.table + (int64_t)it.n * c.table_stride;
        kh = (const __nv_bfloat16*)c.k + (int64_t)it.h * c.sh;
        vh = (const __nv_bfloat16*)c.v + (int64_t)it.h * c.sh;
        const int h0 = it.h * a.G + it.c * HB, heads = min(HB, a.G - it.c * HB);
        // Key of this lane (16 of them) at step i: 64 (first + i) + 16 warp + lane % 16.
        int key = part.first * kTile + warp * kWarpKeys + lane % 16;
        int page = entry_of(c, row, key, len);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int b = 0; b < 2 * DC; ++b) {
                const int d = 32 * b + 8 * t;
                q[n][b] = 8 * n + g < heads && d < c.D
                              ? *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + (int64_t)it.n * a.q_sn +
                                                                (int64_t)(h0 + 8 * n + g) * a.q_sh + d)
                              : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int x = 0; x < DC; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[n][x][e][r] = 0.f;
        }
        const float shrink = exp2f((float)shrink_of(len));
        int64_t off = offset_of(c, page, key, len);
        bool whole = is_whole(off);
        load_k(off, whole);
        load_v(off, 0, whole);
        page = entry_of(c, row, key + kTile, len);
        for (int i = 0; i < tiles; ++i) {
            const uint32_t bad = __ballot_sync(0xffffffffu, off == kBad);
            const uint32_t none = __ballot_sync(0xffffffffu, off == kNone);
            // scores, in log2 units: s[n][0..1] key g, heads 2t, 2t+1; s[n][2..3] key g + 8
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[n][r] = 0.f;
#pragma unroll
                for (int b = 0; b < 2 * DC; ++b) {
                    mma_bf16(s[n], k[0][b].x, k[1][b].x, k[0][b].y, k[1][b].y, q[n][b].x, q[n][b].y);
                    mma_bf16(s[n], k[0][b].z, k[1][b].z, k[0][b].w, k[1][b].w, q[n][b].z, q[n][b].w);
                }
            }
            const int64_t off_now = off;
            const bool more = i + 1 < tiles, whole_now = whole;
            if (more) {
                key += kTile;
                off = offset_of(c, page, key, len);
                whole = is_whole(off);
                load_k(off, whole);
                if (i + 2 < tiles) page = entry_of(c, row, key + kTile, len);
            }
            uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[n][r] *= a.scale_log2;
                if (!whole_now) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int kk = g + 8 * (r >> 1);
                        if (bad >> kk & 1) s[n][r] = __int_as_float(0x7fffffff);
                        if (none >> kk & 1) s[n][r] = -INFINITY;
                    }
                }
                float mx[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    mx[r] = fmaxf(s[n][r], s[n][r + 2]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], o));
                }
                if (__any_sync(0xffffffffu, mx[0] > m[n][0] + (float)kLazy || mx[1] > m[n][1] + (float)kLazy)) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float mn = fmaxf(m[n][r], mx[r]);
                        const float f = ex2(m[n][r] - safe_max(mn));
                        m[n][r] = mn;
                        l[n][r] *= f;
#pragma unroll
                        for (int x = 0; x < DC; ++x)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                acc[n][x][e][r] *= f;
                                acc[n][x][e][r + 2] *= f;
                            }
                    }
                }
                const float m0 = safe_max(m[n][0]), m1 = safe_max(m[n][1]);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float p0 = ex2(s[n][2 * r] - m0), p1 = ex2(s[n][2 * r + 1] - m1);
                    l[n][0] += p0;
                    l[n][1] += p1;
                    p0 *= shrink, p1 *= shrink;
                    const uint32_t hi = pair_hi(below(p0), below(p1));
                    const float2 back = unpack_bf16(hi);
                    ph[n][r] = transpose8x8(hi);
                    pl[n][r] = transpose8x8(pack_bf16(p0 - back.x, p1 - back.y));
                }
            }
#pragma unroll
            for (int c0 = 0; c0 < DC; c0 += VC) {
                if (c0 > 0) load_v(off_now, c0, whole_now);
#pragma unroll
                for (int x = 0; x < VC; ++x) {
                    const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&v[0][x]);
                    const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&v[1][x]);
                    const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&v[2][x]);
                    const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&v[3][x]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t a0 = pair_lo(w0[e], w1[e]), a1 = pair_hi(w0[e], w1[e]);
                        const uint32_t a2 = pair_lo(w2[e], w3[e]), a3 = pair_hi(w2[e], w3[e]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma_bf16(acc[n][c0 + x][e], a0, a1, a2, a3, ph[n][0], ph[n][1]);
                            mma_bf16(acc[n][c0 + x][e], a0, a1, a2, a3, pl[n][0], pl[n][1]);
                        }
                    }
                }
            }
            if (more) load_v(off, 0, whole);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], o);
                const int h = 8 * n + 2 * t + r;
                if (g == 0) sp.ml[warp][h] = make_float2(m[n][r], l[n][r]);
#pragma unroll
                for (int x = 0; x < DC; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<float2*>(&sp.o[warp][h * Parts<HB, kD>::kRow + 64 * x + 8 * g + 2 * e]) =
                            make_float2(acc[n][x][e][r], acc[n][x][e][r + 2]);
            }
        }
    }
};

// ---- f32: scores and sums in f32 on the FMA pipes ---------------------------------
// Lane 4 g + t takes keys g and g + 8 and every fourth 16-byte piece of their rows;
// the scores pass through shared memory to a layout with four lanes a head, and the
// probabilities back as one broadcast read a key. Lane l owns DV elements of o.
template <int GH, int DV>
struct AttnF32 {
    static constexpr int kD = 32 * DV;
    static constexpr int HB = GH;

    struct alignas(16) Scratch {
        float q[GH][kD];
        float s[kWarps][GH][kWarpKeys];
        float p[kWarps][kWarpKeys][GH];
        float f[kWarps][GH];
    };

    static constexpr bool kAhead = DV == 2 && GH <= 4;

    // This lane's elements of a value row. WHOLE: there is a row, of kD elements; else what is missing is zero.
    template <bool WHOLE>
    static __device__ __forceinline__ void load_v(float (&v)[DV], const float* row, bool there, int lane, int D) {
        if constexpr (!WHOLE) {
#pragma unroll
            for (int x = 0; x < DV; ++x) v[x] = 0.f;
            if (!there) return;
        }
        if constexpr (DV == 2) {
            if (WHOLE || 2 * lane < D) {
                const float2 u = *reinterpret_cast<const float2*>(row + 2 * lane);
                v[0] = u.x, v[1] = u.y;
            }
        } else {
#pragma unroll
            for (int x = 0; x < DV; x += 4) {
                const int d = 32 * x + 4 * lane;
                if (WHOLE || d < D) {
                    const float4 u = *reinterpret_cast<const float4*>(row + d);
                    v[x] = u.x, v[x + 1] = u.y, v[x + 2] = u.z, v[x + 3] = u.w;
                }
            }
        }
    }

    const PagedAttn& a;
    Scratch& sm;
    __device__ __forceinline__ AttnF32(const PagedAttn& args, Scratch& scratch) : a(args), sm(scratch) {}

    __device__ __forceinline__ void run(const Part& part, Parts<HB, kD>& sp) {
        const PagedView& c = a.cache;
        const Item it = part.it;
        const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
        const int len = part.len, D = c.D, tile = part.first, tiles = part.count;
        const int32_t* row = c.table + (int64_t)it.n * c.table_stride;
        const float* kh = (const float*)c.k + (int64_t)it.h * c.sh;
        const float* vh = (const float*)c.v + (int64_t)it.h * c.sh;
        const int h0 = it.h * a.G + it.c * HB, heads = min(HB, a.G - it.c * HB);
        int key = tile * kTile + warp * kWarpKeys + lane % 16;
        int page = entry_of(c, row, key, len);
        int64_t off = 0;
        // Keys and values a step ahead, as in bf16, where the registers allow it.
        constexpr int kN = kD / 16;
        float4 kx[kN], ky[kN];
        float v[kWarpKeys][DV];
        // Sixteen keys that are all there, of kD elements, ask nothing for each load, and on one page
        // their rows follow each other. (The general way takes three times the instructions.)
        bool whole = false, one_page = false;
        auto locate = [&] {
            whole = D == kD && __all_sync(0xffffffffu, off >= 0);
            const int64_t off0 = __shfl_sync(0xffffffffu, off, 0);
            one_page = __all_sync(0xffffffffu, off == off0 + lane % kWarpKeys * c.ss);
        };
        auto piece = [&](auto fast, int64_t o, int j) {
            const int d = 16 * j + 4 * t;
            if constexpr (decltype(fast)::value) return *reinterpret_cast<const float4*>(kh + o + d);
            return o >= 0 && d < D ? *reinterpret_cast<const float4*>(kh + o + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        auto load_k_as = [&](auto fast) {
            const int64_t o0 = __shfl_sync(0xffffffffu, off, g), o1 = __shfl_sync(0xffffffffu, off, g + 8);
#pragma unroll
            for (int j = 0; j < kN; ++j) kx[j] = piece(fast, o0, j), ky[j] = piece(fast, o1, j);
        };
        auto load_k = [&] { whole ? load_k_as(std::true_type{}) : load_k_as(std::false_type{}); };
        auto load_vs = [&] {
            if (whole && one_page) {
                const float* first = vh + __shfl_sync(0xffffffffu, off, 0);
#pragma unroll
                for (int kk = 0; kk < kWarpKeys; ++kk) load_v<true>(v[kk], first + kk * c.ss, true, lane, D);
            } else if (whole) {
#pragma unroll
                for (int kk = 0; kk < kWarpKeys; ++kk)
                    load_v<true>(v[kk], vh + __shfl_sync(0xffffffffu, off, kk), true, lane, D);
            } else {
#pragma unroll
                for (int kk = 0; kk < kWarpKeys; ++kk) {
                    const int64_t o = __shfl_sync(0xffffffffu, off, kk);
                    load_v<false>(v[kk], vh + o, o >= 0, lane, D);
                }
            }
        };
        if constexpr (kAhead) {
            off = offset_of(c, page, key, len);
            locate();
            load_k();
            load_vs();
            page = entry_of(c, row, key + kTile, len);
        }
        for (int i = threadIdx.x; i < GH * kD; i += kThreads) {
            const int h = i / kD, d = i % kD;
            sm.q[h][d] = h < heads && d < D
                             ? ((const float*)a.q)[(int64_t)it.n * a.q_sn + (int64_t)(h0 + h) * a.q_sh + d]
                             : 0.f;
        }
        __syncthreads();
        // max and sum of head lane / 4 (the same in its four lanes, the sum after the loop)
        const int hs = lane / 4;
        const bool has = hs < GH;
        const float shrink = exp2f((float)shrink_of(len));
        float m = -INFINITY, l = 0.f;
        float acc[GH][DV];
#pragma unroll
        for (int h = 0; h < GH; ++h)
#pragma unroll
            for (int x = 0; x < DV; ++x) acc[h][x] = 0.f;
        for (int i = 0; i < tiles; ++i) {
            if constexpr (!kAhead) {
                off = offset_of(c, page, key, len);
                locate();
                key += kTile;
                if (i + 1 < tiles) page = entry_of(c, row, key, len);
            }
            const uint32_t bad = __ballot_sync(0xffffffffu, off == kBad);
            const uint32_t none = __ballot_sync(0xffffffffu, off == kNone);
            const int64_t o0 = __shfl_sync(0xffffffffu, off, g), o1 = __shfl_sync(0xffffffffu, off, g + 8);
            float s0[GH], s1[GH];
#pragma unroll
            for (int h = 0; h < GH; ++h) s0[h] = s1[h] = 0.f;
            auto dots = [&](auto fast) {
#pragma unroll
                for (int j = 0; j < kN; ++j) {
                    const int d = 16 * j + 4 * t;
                    const float4 x = kAhead ? kx[j] : piece(fast, o0, j), y = kAhead ? ky[j] : piece(fast, o1, j);
#pragma unroll
                    for (int h = 0; h < GH; ++h) {
                        const float4 w = *reinterpret_cast<const float4*>(&sm.q[h][d]);
                        s0[h] = fmaf(x.x, w.x, fmaf(x.y, w.y, fmaf(x.z, w.z, fmaf(x.w, w.w, s0[h]))));
                        s1[h] = fmaf(y.x, w.x, fmaf(y.y, w.y, fmaf(y.z, w.z, fmaf(y.w, w.w, s1[h]))));
                    }
                }
            };
            if (kAhead || !whole)
                dots(std::false_type{});
            else
                dots(std::true_type{});
#pragma unroll
            for (int h = 0; h < GH; ++h) {
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    s0[h] += __shfl_xor_sync(0xffffffffu, s0[h], o);
                    s1[h] += __shfl_xor_sync(0xffffffffu, s1[h], o);
                }
                if (t == 0) sm.s[warp][h][g] = s0[h], sm.s[warp][h][g + 8] = s1[h];
            }
            const bool more = i + 1 < tiles;
            if constexpr (!kAhead) load_vs();
            if (kAhead && more) {
                key += kTile;
                off = offset_of(c, page, key, len);
                locate();
                load_k();
                if (i + 2 < tiles) page = entry_of(c, row, key + kTile, len);
            }
            __syncwarp();
            float f = 1.f;
            if (has) {
                float s[4], mx = -INFINITY;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int kk = 4 * t + r;
                    s[r] = sm.s[warp][hs][kk] * a.scale_log2;
                    if (bad >> kk & 1) s[r] = __int_as_float(0x7fffffff);
                    if (none >> kk & 1) s[r] = -INFINITY;
                    mx = fmaxf(mx, s[r]);
                }
                const uint32_t active = GH == 8 ? 0xffffffffu : (1u << (4 * GH)) - 1u;
                mx = fmaxf(mx, __shfl_xor_sync(active, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(active, mx, 2));
                const float mn = fmaxf(m, mx);
                f = exp2f(m - safe_max(mn));
                m = mn;
                l *= f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = exp2f(s[r] - safe_max(m));
                    l += p;
                    sm.p[warp][4 * t + r][hs] = p * shrink;
                }
                if (t == 0) sm.f[warp][hs] = f;
            }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < GH; ++h) {
                const float fh = sm.f[warp][h];
#pragma unroll
                for (int x = 0; x < DV; ++x) acc[h][x] *= fh;
            }
#pragma unroll
            for (int kk = 0; kk < kWarpKeys; ++kk) {
#pragma unroll
                for (int h = 0; h < GH; ++h) {
                    const float p = sm.p[warp][kk][h];
#pragma unroll
                    for (int x = 0; x < DV; ++x) acc[h][x] = fmaf(p, v[kk][x], acc[h][x]);
                }
            }
            if (kAhead && more) load_vs();
            __syncwarp();
        }
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (has && t == 0) sp.ml[warp][hs] = make_float2(m, l);
#pragma unroll
        for (int h = 0; h < GH; ++h)
#pragma unroll
            for (int x = 0; x < DV; ++x) {
                const int d = DV == 2 ? 2 * lane + x : 32 * (x & ~3) + 4 * lane + (x & 3);
                sp.o[warp][h * Parts<HB, kD>::kRow + d] = acc[h][x];
            }
    }
};

template <typename T, typename W>
__device__ __forceinline__ void paged_worker(const PagedAttn& a, W& w, Parts<W::HB, W::kD>& sp) {
    after_prior_kernels();
    may_start_next();  // the join, which waits for all workers
    const int chunks = (a.G + W::HB - 1) / W::HB;
    const int per = a.cache.H * chunks;
    int64_t start, end, before;
    int n, empty;
    if (!find_run(a, per, start, end, n, before, empty)) return;
    int tiles = tiles_of(a, n), places = places_of(tiles, empty);
    int item = (int)((start - before) / places), place = (int)((start - before) - (int64_t)item * places);
    int64_t at = start;
    auto next_part = [&]() -> Part {
        while (at < end) {
            const int take = (int)min((int64_t)(places - place), end - at);
            const int first = max(place - empty, 0), last = place + take - empty;  // tiles [first, last)
            // The worker's second slot is for the item whose first tile it has.
            const Part p{Item{n, item / chunks, item % chunks}, first, max(last - first, 0), a.lens[n],
                         2 * (int)blockIdx.x + (first == 0 && at - place + empty > start), last - first == tiles};
            at += take;
            place = 0;
            if (++item == per && at < end) {
                item = 0;
                do {
                    if (++n == a.cache.num_seqs) {
                        at = end;
                        break;
                    }
                    tiles = tiles_of(a, n);
                } while (tiles == 0);
                places = places_of(tiles, empty);
            }
            if (p.count) return p;
        }
        return Part{Item{0, 0, 0}, 0, 0, 0, 0, false};
    };
    for (Part part = next_part(); part.count; part = next_part()) {
        w.run(part, sp);
        __syncthreads();
        finish_item<T, W::HB, W::kD>(a, sp, part.it, part.whole, part.len, part.slot);
        __syncthreads();
    }
}

template <int DC, int NT>
__global__ void __launch_bounds__(kThreads, DC == 2 && NT == 1 ? 3 : DC == 1 && NT == 1 ? 4 : 1) paged_attn_bf16_kernel(PagedAttn a) {
    __shared__ Parts<8 * NT, 64 * DC> sp;
    AttnBf16<DC, NT> w(a);
    paged_worker<__nv_bfloat16>(a, w, sp);
}

template <int GH, int DV>
__global__ void __launch_bounds__(kThreads) paged_attn_f32_kernel(PagedAttn a) {
    using W = AttnF32<GH, DV>;
    __shared__ Parts<GH, 32 * DV> sp;
    __shared__ typename W::Scratch scratch;
    W w(a, scratch);
    paged_worker<float>(a, w, sp);
}

// One CTA a query head of a sequence: the join of its item's parts, the zeros of an
// empty sequence, or the NaN of one that is longer than its table row. It is launched with the
// workers and waits for them here.
constexpr int kJoinWarps = 16;  // at most
template <typename T, int HB>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_join_kernel(PagedAttn a, int workers) {
    __shared__ float so[kJoinWarps][256];
    __shared__ float2 sml[kJoinWarps];
    may_start_next();
    const int threads = blockDim.x, warps = threads / 32;
    const int n = blockIdx.x / a.Hq, hq = blockIdx.x % a.Hq, D = a.cache.D;
    const int chunks = (a.G + HB - 1) / HB;
    T* o = (T*)a.o + (int64_t)n * a.o_sn + (int64_t)hq * a.o_sh;
    float* lse = a.lse ? a.lse + (int64_t)n * a.Hq + hq : nullptr;
    after_prior_kernels();
    const int tiles = tiles_of(a, n), in_group = hq % a.G;
    if (tiles == 0) {
        const bool empty = a.lens[n] <= 0;
        const float nan = __int_as_float(0x7fffffff);
        for (int d = threadIdx.x; d < D; d += threads) o[d] = T(empty ? 0.f : nan);
        if (threadIdx.x == 0 && lse) *lse = empty ? -INFINITY : nan;
        return;
    }
    const int64_t run = a.plan->run;
    const int empty = (int)a.plan->empty;
    const int64_t first = a.starts[n] + ((int64_t)(hq / a.G) * chunks + in_group / HB) * places_of(tiles, empty) + empty;
    const int w0 = (int)(first / run), w1 = min((int)((first + tiles - 1) / run), workers - 1);
    if (w0 == w1) return;  // one worker had it all
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, head = in_group % HB;
    float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) acc[x] = 0.f;
    // Warp w takes the parts w0 + w, w0 + w + warps, ..., four at once; lane l the elements l, l + 32, ...
    constexpr int kAtOnce = 4;
    for (int w = w0 + warp; w <= w1; w += kAtOnce * warps) {
        float2 ml[kAtOnce];
        float v[kAtOnce][8];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int wk = w + k * warps;
            ml[k] = make_float2(-INFINITY, 0.f);
            if (wk <= w1) {
                const float* part = a.part + (int64_t)(2 * wk + (first > run * wk)) * part_floats(HB, D);
                ml[k] = reinterpret_cast<const float2*>(part + HB * D)[head];
#pragma unroll
                for (int x = 0; x < 8; ++x) v[k][x] = lane + 32 * x < D ? part[head * D + lane + 32 * x] : 0.f;
            }
        }
        float mn = m;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) mn = fmaxf(mn, ml[k].x);
        const float f = exp2f(m - safe_max(mn));
        m = mn;
        l *= f;
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] *= f;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
            if (w + k * warps <= w1) {
                const float fk = exp2f(ml[k].x - safe_max(mn));
                l += ml[k].y * fk;
#pragma unroll
                for (int x = 0; x < 8; ++x) acc[x] = fmaf(v[k][x], fk, acc[x]);
            }
    }
#pragma unroll
    for (int x = 0; x < 8; ++x)
        if (lane + 32 * x < D) so[warp][lane + 32 * x] = acc[x];
    if (lane == 0) sml[warp] = make_float2(m, l);
    __syncthreads();
    m = -INFINITY;
    for (int w = 0; w < warps; ++w) m = fmaxf(m, sml[w].x);
    l = 0.f;
    float f[kJoinWarps];
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        f[w] = w < warps ? exp2f(sml[w].x - safe_max(m)) : 0.f;
        if (w < warps) l += f[w] * sml[w].y;
    }
    for (int d = threadIdx.x; d < D; d += threads) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w)
            if (w < warps) s += f[w] * so[w][d];
        o[d] = T(s / l * power_of_two(-shrink_of(a.lens[n])));
    }
    if (threadIdx.x == 0 && lse) *lse = (m + log2f(l)) * kLn2;
}

template <typename T, int HB, void (*KERNEL)(PagedAttn)>
cudaError_t launch(cudaStream_t st, int sm_count, const PagedAttn& a) {
    static std::atomic<int> known{0};  // CTAs resident on an SM, a property of the kernel alone
    int resident = known.load(std::memory_order_relaxed);
    cudaError_t e;
    if (resident == 0) {
        if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, KERNEL, kThreads, 0)) != cudaSuccess) return e;
        known.store(resident, std::memory_order_relaxed);
    }
    int workers = sm_count * resident;
    if (workers > kMaxWorkers) workers = kMaxWorkers;
    if ((e = launch_overlapped(st, KERNEL, dim3((unsigned)workers), kThreads, 0, 0, a)) != cudaSuccess) return e;
    // Many rows: smaller CTAs, so that they fit at once. Few: as many warps as an item's parts may need.
    const int rows = a.cache.num_seqs * a.Hq, threads = rows > 8 * sm_count ? 128 : rows > sm_count ? 256 : 512;
    return launch_overlapped(st, paged_join_kernel<T, HB>, dim3((unsigned)rows), threads, 0, 0, a, workers);
}

// Query heads that one worker takes at once: a multiple of the mma's 8 columns in bf16
// (16 where the registers allow it, so that the keys are still read once), up to 8 in f32.
int heads_at_once(hx_dtype dt, int G, int D) {
    if (dt == HX_BF16) return G > 8 && D <= 128 ? 16 : 8;
    return G == 1 ? 1 : G <= 4 ? 4 : 8;
}

}  // namespace

// The plan, then the workers' parts.
static uint64_t plan_bytes(int num_seqs) { return (sizeof(Plan) + (uint64_t)num_seqs * sizeof(int64_t) + 255) / 256 * 256; }

uint64_t paged_attn_workspace_bytes(hx_dtype dt, int Hq, int Hkv, int D, int num_seqs) {
    return plan_bytes(num_seqs) + (uint64_t)2 * kMaxWorkers * part_floats(heads_at_once(dt, Hq / Hkv, D), D) * sizeof(float);
}

cudaError_t paged_attn(cudaStream_t st, int sm_count, hx_dtype dt, PagedAttn a, void* workspace) {
    a.plan = (Plan*)workspace;
    a.starts = (int64_t*)(a.plan + 1);
    a.part = (float*)((char*)workspace + plan_bytes(a.cache.num_seqs));
    const int D = a.cache.D, hb = heads_at_once(dt, a.G, D);
    if (dt == HX_BF16) {
        if (hb == 16)
            return D <= 64 ? launch<__nv_bfloat16, 16, paged_attn_bf16_kernel<1, 2>>(st, sm_count, a)
                           : launch<__nv_bfloat16, 16, paged_attn_bf16_kernel<2, 2>>(st, sm_count, a);
        return D <= 64    ? launch<__nv_bfloat16, 8, paged_attn_bf16_kernel<1, 1>>(st, sm_count, a)
               : D <= 128 ? launch<__nv_bfloat16, 8, paged_attn_bf16_kernel<2, 1>>(st, sm_count, a)
                          : launch<__nv_bfloat16, 8, paged_attn_bf16_kernel<4, 1>>(st, sm_count, a);
    }
    if (hb == 1)
        return D <= 64    ? launch<float, 1, paged_attn_f32_kernel<1, 2>>(st, sm_count, a)
               : D <= 128 ? launch<float, 1, paged_attn_f32_kernel<1, 4>>(st, sm_count, a)
                          : launch<float, 1, paged_attn_f32_kernel<1, 8>>(st, sm_count, a);
    if (hb == 4)
        return D <= 64    ? launch<float, 4, paged_attn_f32_kernel<4, 2>>(st, sm_count, a)
               : D <= 128 ? launch<float, 4, paged_attn_f32_kernel<4, 4>>(st, sm_count, a)
                          : launch<float, 4, paged_attn_f32_kernel<4, 8>>(st, sm_count, a);
    return D <= 64    ? launch<float, 8, paged_attn_f32_kernel<8, 2>>(st, sm_count, a)
           : D <= 128 ? launch<float, 8, paged_attn_f32_kernel<8, 4>>(st, sm_count, a)
                      : launch<float, 8, paged_attn_f32_kernel<8, 8>>(st, sm_count, a);
}

}  // namespace hx
