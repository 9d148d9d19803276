// Log probabilities of given tokens under logits [rows, classes], with the
// entropy and the most likely alternatives of each row, and their gradient:
//   z_i = x_i - m (m the row's maximum), s = sum e^{z_i}, w = sum z_i e^{z_i}
//   logp(t) = z_t - ln s,  H = ln s - w / s
//   dx_i = g_t (1[i = t] - p_i) - g_H p_i (ln p_i + H)
// One read of the logits forward, one read and one write backward: bytes bound
// both, if a logit costs no more than about nine instructions, one of them the
// exponential (7 TB/s of bf16 are 13 logits a clock and SM). So the differences,
// products and sums run two to an instruction (f32x2), and whole 16-byte
// pieces are loaded four at a time, in the forward the next four before these are
// added. It keeps (m, s, w) running, so the row is read once; both terms of H are positive, so nothing cancels. Sums are f32,
// per thread and then joined in a tree, the same for every call. A few rows are
// split over a cluster of CTAs each, which join through distributed shared memory.
//
// The alternatives need no second pass over the row either. Each thread knows the
// best of its own logits; the k best threads' values bound the k-th best logit
// from below, and every logit that reaches the bound belongs to one of those k
// threads, so only their share of the row (k / 256 of it, say) is looked at again.
// Ties go to the lower index.
#include <cooperative_groups.h>

#include <type_traits>

#include "hx_internal.h"
#include "launch.h"
#include "mma_bf16.cuh"
#include "sm100_ptx.cuh"

namespace hx {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -3.402823466e+38f;
constexpr float kFloor = -1.0e4f;  // exp2 of it is 0; keeps 0 * (-inf) out of the sums
constexpr unsigned kAll = 0xffffffffu;
constexpr int kAhead = 4;  // pieces of a thread that are loaded at once

// max that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
using ptx::ex2;
using ptx::f2_add;
using ptx::f2_fma;
using ptx::f2_pack;
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Bits that order as the values do; NaN orders as -inf, -0 as 0. Never 0.
__device__ __forceinline__ uint32_t order_of(float v) {
    if (!(v == v)) v = -INFINITY;
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// A row as 16-byte pieces from the last 16-byte boundary at or before its start: piece j
// holds the elements [E j - lead, E j - lead + E) that are in [0, classes).
template <typename T>
struct RowView {
    static constexpr int E = 16 / sizeof(T);
    const T* x;
    int classes, lead, pieces;
    __device__ __forceinline__ RowView(const T* row, int n)
        : x(row), classes(n), lead((int)(((uintptr_t)row & 15) / sizeof(T))), pieces((int)(((int64_t)lead + n + E - 1) / E)) {}
    __device__ __forceinline__ int first(int j) const { return E * j - lead; }
    __device__ __forceinline__ bool whole(int j) const { return first(j) >= 0 && first(j) + E <= classes; }
    // The whole pieces are [begin(), end()); one before and one after may be partial (or the only one).
    __device__ __forceinline__ int begin() const { return lead > 0; }
    __device__ __forceinline__ int end() const { return (lead + classes) / E; }
    __device__ __forceinline__ uint4 raw(int j) const { return *reinterpret_cast<const uint4*>(x + first(j)); }
    static __device__ __forceinline__ void decode(const uint4& u, float (&v)[E]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack_bf16(w[i]);
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
        }
    }
    // The largest element; NaN does not count unless there is nothing else.
    static __device__ __forceinline__ float top(const uint4& u) {
        if constexpr (sizeof(T) == 2) {
            const float2 f = unpack_bf16(max2(max2(u.x, u.y), max2(u.z, u.w)));
            return fmaxf(f.x, f.y);
        } else {
            return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                         fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
        }
    }
    // Elements outside the row read as `pad`.
    __device__ __forceinline__ void load(int j, float (&v)[E], float pad) const {
        if (whole(j)) {
            decode(raw(j), v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = first(j) + e;
                v[e] = i >= 0 && i < classes ? (float)x[i] : pad;
            }
        }
    }
};

struct Stats {
    float m, s, w;  // maximum, sum of e^z, sum of (z in log2 units) e^z
};
// log2 of the weight that a part with maximum m has under the maximum `to`.
__device__ __forceinline__ float weight_of(float m, float to) { return max_nan((m - to) * kLog2e, kFloor); }
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
    const float m = fmaxf(a.m, b.m), da = weight_of(a.m, m), db = weight_of(b.m, m);
    const float ea = ex2(da), eb = ex2(db);
    return Stats{m, a.s * ea + b.s * eb, ea * (a.w + da * a.s) + eb * (b.w + db * b.s)};
}
// Of the LANES first lanes of a warp, to all of them: the maximum first, so that each part is
// weighted once.
template <int LANES>
__device__ __forceinline__ Stats join_lanes(Stats a) {
    float m = a.m;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
    const float d = weight_of(a.m, m), e = ex2(d);
    a = Stats{m, e * a.s, e * fmaf(d, a.s, a.w)};
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(kAll, a.s, o);
        a.w += __shfl_xor_sync(kAll, a.w, o);
    }
    return a;
}

// A thread's running statistics, the sums in two halves.
struct Running {
    float m = kLowest;
    uint64_t s = 0, w = 0, minus_m = f2_pack(-kLowest, -kLowest);

    // Before logits of at most `top` are added.
    __device__ __forceinline__ void raise(float top) {
        if (top > m) {
            const float d = weight_of(m, top), e = ex2(d);
            const uint64_t e2 = f2_pack(e, e);
            w = f2_mul(e2, f2_fma(f2_pack(d, d), s, w));
            s = f2_mul(e2, s);
            m = top;
            minus_m = f2_pack(-m, -m);
        }
    }
    template <int E>
    __device__ __forceinline__ void add(const float (&v)[E]) {
        const uint64_t l2 = f2_pack(kLog2e, kLog2e);
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            float z0, z1;
            ptx::f2_unpack(f2_mul(f2_add(f2_pack(v[i], v[i + 1]), minus_m), l2), z0, z1);
            z0 = max_nan(z0, kFloor), z1 = max_nan(z1, kFloor);
            const uint64_t e = f2_pack(ex2(z0), ex2(z1));
            s = f2_add(s, e);
            w = f2_fma(f2_pack(z0, z1), e, w);
        }
    }
    __device__ __forceinline__ Stats stats() const {
        float s0, s1, w0, w1;
        ptx::f2_unpack(s, s0, s1);
        ptx::f2_unpack(w, w0, w1);
        return Stats{m, s0 + s1, w0 + w1};
    }
};

// ---- the 32 largest keys of a block -----------------------------------------------
__device__ __forceinline__ uint64_t shfl_key(uint64_t k, int o) { return __shfl_xor_sync(kAll, k, o); }
__device__ __forceinline__ uint64_t pick(uint64_t a, uint64_t b, bool larger) { return (a > b) == larger ? a : b; }

// Sorts a bitonic sequence over the lanes, largest first.
__device__ __forceinline__ uint64_t clean(uint64_t k, int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) k = pick(k, shfl_key(k, o), (lane & o) == 0);
    return k;
}
__device__ __forceinline__ uint64_t sort_keys(uint64_t k, int lane) {
#pragma unroll
    for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
        for (int o = n >> 1; o > 0; o >>= 1) k = pick(k, shfl_key(k, o), ((lane & o) == 0) == ((lane & n) == 0 || n == 32));
    return k;
}
// The 32 largest of two sorted lists, sorted.
__device__ __forceinline__ uint64_t merge_keys(uint64_t a, uint64_t b_reversed, int lane) {
    return clean(a > b_reversed ? a : b_reversed, lane);
}
// Every one of WARPS warps brings a sorted list; warp 0 leaves with the 32 largest of all.
template <int WARPS>
__device__ __forceinline__ uint64_t block_largest(uint64_t k, uint64_t (*lists)[32], int warp, int lane) {
    lists[warp][lane] = k;
#pragma unroll
    for (int s = WARPS / 2; s > 0; s >>= 1) {
        __syncthreads();
        if (warp < s) {
            k = merge_keys(k, lists[warp + s][31 - lane], lane);
            lists[warp][lane] = k;
        }
    }
    return k;
}

struct Fwd {
    const void* logits;
    int64_t stride;
    const uint32_t* targets;
    float *logprob, *entropy, *stats, *top_logprobs;
    int32_t* top_ids;
    int classes, top, splits;  // splits: CTAs of a row, one cluster
};

constexpr int kHits = 128;  // logits that reach the bound, before the slow way

// A CTA of THREADS a row, or of a share of it. grid: rows x splits.
template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(Fwd a) {
    constexpr int E = RowView<T>::E, WARPS = THREADS / 32;
    __shared__ Stats parts[WARPS];
    __shared__ Stats of_cta[8];          // in the cluster's first CTA
    __shared__ uint64_t of_top[TOP ? 8 : 1][32];
    __shared__ uint64_t lists[TOP ? WARPS : 1][32];
    __shared__ uint64_t chosen[32], hits[TOP ? kHits : 1];
    __shared__ int n_hits;
    cg::cluster_group cluster = cg::this_cluster();
    const int splits = a.splits, rank = splits > 1 ? (int)(blockIdx.x % splits) : 0;
    const int64_t r = splits > 1 ? blockIdx.x / splits : blockIdx.x;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const T* x = (const T*)a.logits + r * a.stride;
    const RowView<T> row(x, a.classes);
    if (splits > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");
    if (TOP && tid == 0) n_hits = 0;
    after_prior_kernels();
    may_start_next();

    // Thread tid of CTA rank owns the pieces mine, mine + step, ...
    const int mine = rank * THREADS + tid, step = splits * THREADS;
    Running run;
    float best_v = -INFINITY;
    int best_j = -1;
    auto note = [&](float top, int j) {  // a piece's largest logit; NaN, of a piece of nothing else, ranks as -inf
        if constexpr (TOP) {
            if (top > best_v || best_j < 0) best_j = j, best_v = fmaxf(top, -INFINITY);
        }
    };
    auto add_partial = [&](int j) {
        float v[E];
        row.load(j, v, -INFINITY);
        float top = v[0];
#pragma unroll
        for (int e = 1; e < E; ++e) top = fmaxf(top, v[e]);
        note(top, j);
        run.raise(top);
        run.add(v);
    };
    if (mine == 0 && !row.whole(0)) add_partial(0);
    const int end = row.end();
    int j0 = mine < row.begin() ? mine + step : mine;
    uint4 u[kAhead];
    auto load = [&](int j, auto all) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (decltype(all)::value || j + k * step < end) u[k] = row.raw(j + k * step);
    };
    auto batch = [&](auto all, auto next) {  // kAhead pieces from j0 on; unless all are there, those that are
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (decltype(all)::value || j0 + k * step < end) {
                const float t = RowView<T>::top(u[k]);
                note(t, j0 + k * step);
                top = fmaxf(top, t);
            }
        run.raise(top);
        const uint4 now[kAhead] = {u[0], u[1], u[2], u[3]};
        next();
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (decltype(all)::value || j0 + k * step < end) {
                float v[E];
                RowView<T>::decode(now[k], v);
                run.add(v);
            }
    };
    const int full = kAhead * step, tail = end - (kAhead - 1) * step;
    if (j0 < tail) {
        load(j0, std::true_type{});
        for (; j0 + full < tail; j0 += full) batch(std::true_type{}, [&] { load(j0 + full, std::true_type{}); });
        batch(std::true_type{}, [&] { load(j0 + full, std::false_type{}); });
        j0 += full;
    } else {
        load(j0, std::false_type{});
    }
    if (j0 < end) batch(std::false_type{}, [] {});
    const int last = row.pieces - 1;
    if (last > 0 && last >= end && last % step == mine) add_partial(last);
    Stats st = join_lanes<32>(run.stats());
    if (lane == 0) parts[warp] = st;
    __syncthreads();
    st = join_lanes<WARPS>(parts[lane % WARPS]);

    uint64_t found = 0;
    if constexpr (TOP) {
        const uint64_t key = best_j < 0 ? 0 : (uint64_t)order_of(best_v) << 32 | (uint32_t)~best_j;
        const uint64_t k = block_largest<WARPS>(sort_keys(key, lane), lists, warp, lane);
        if (warp == 0) chosen[lane] = k;
        __syncthreads();
        const uint64_t bound = chosen[a.top - 1];
        // The chosen threads' pieces again, a thread's by so many lanes as it has pieces; a piece's element
        // counts when (its order, ~its piece) reaches the bound.
        const int each = (row.pieces + step - 1) >> (__ffs(step) - 1), lanes_log = each >= 32 ? 5 : 32 - __clz(each - 1);
        auto scan = [&](auto&& take) {
            for (int c0 = warp << (5 - lanes_log); c0 < a.top; c0 += WARPS << (5 - lanes_log)) {
                const int c = c0 + (lane >> lanes_log), j0 = (lane & ((1 << lanes_log) - 1)) * step;
                const uint64_t chose = c < a.top ? chosen[c] : 0;
                const int from = chose != 0 ? (int)(~(uint32_t)chose & (uint32_t)(step - 1)) + j0 : row.pieces;
                for (int n = 0; n < each; n += 1 << lanes_log) {
                    const int j = from + n * step;
                    float v[E];
                    if (j < row.pieces) row.load(j, v, -INFINITY);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int i = row.first(j) + e;
                        uint64_t key = 0;
                        if (j < row.pieces && i >= 0 && i < a.classes) {
                            const uint64_t high = (uint64_t)order_of(v[e]) << 32;
                            if ((high | (uint32_t)~j) >= bound) key = high | (uint32_t)~i;
                        }
                        take(key);
                    }
                }
            }
        };
        scan([&](uint64_t key) {
            if (key != 0) {
                const int at = atomicAdd(&n_hits, 1);
                if (at < kHits) hits[at] = key;
            }
        });
        __syncthreads();
        // There are at least as many hits as alternatives, and rarely many more: one warp puts
        // them in order (their number alone depends on the row, not on the atomics' order).
        const int n = n_hits;
        if (n <= kHits) {
            if (warp == 0)
                for (int i = 0; i < n; i += 32) {
                    const uint64_t sorted = sort_keys(i + lane < n ? hits[i + lane] : 0, lane);
                    found = i == 0 ? sorted : merge_keys(found, __shfl_sync(kAll, sorted, 31 - lane), lane);
                }
        } else {  // a row made of ties, say: every warp keeps the best of what it sees
            scan([&](uint64_t key) {
                if (__any_sync(kAll, key != 0)) {
                    const uint64_t sorted = sort_keys(key, lane);
                    found = merge_keys(found, __shfl_sync(kAll, sorted, 31 - lane), lane);
                }
            });
            found = block_largest<WARPS>(found, lists, warp, lane);
        }
    }
    if (splits > 1) {  // to the first CTA, which joins them in order
        asm volatile("barrier.cluster.wait;" ::: "memory");
        if (tid == 0) *cluster.map_shared_rank(&of_cta[rank], 0) = st;
        if (TOP && warp == 0) *cluster.map_shared_rank(&of_top[TOP ? rank : 0][lane], 0) = found;
        asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
        if (rank != 0) return;
        st = of_cta[0];
        for (int k = 1; k < splits; ++k) st = join(st, of_cta[k]);
        if (TOP && warp == 0) {
            found = of_top[0][lane];
            for (int k = 1; k < splits; ++k) found = merge_keys(found, of_top[TOP ? k : 0][31 - lane], lane);
        }
    }
    const float log_s = logf(st.s);
    if (tid == 0) {
        const uint32_t t = a.targets[r];
        const float h = log_s - kLn2 * st.w / st.s;
        a.logprob[r] = t < (uint32_t)a.classes ? ((float)x[t] - st.m) - log_s : __int_as_float(0x7fffffff);
        a.entropy[r] = h;
        if (a.stats) a.stats[3 * r] = st.m, a.stats[3 * r + 1] = log_s, a.stats[3 * r + 2] = h;
    }
    if (TOP && warp == 0 && lane < a.top) {
        const int i = (int)~(uint32_t)found;
        a.top_ids[r * a.top + lane] = i;
        a.top_logprobs[r * a.top + lane] = ((float)x[i] - st.m) - log_s;
    }
}

// ---- short rows: a warp each -------------------------------------------------------
// As above, with the row's best pieces in a sorted list over the lanes instead of one best
// piece a thread: a group of 32 pieces is sorted and merged into it when one of them beats
// the k-th. Every logit among the k best is in one of the k best pieces.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 3) token_logprobs_warp_kernel(Fwd a, int rows) {
    constexpr int E = RowView<T>::E;
    after_prior_kernels();
    may_start_next();
    const int lane = threadIdx.x % 32;
    const int64_t r = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
    if (r >= rows) return;
    const T* x = (const T*)a.logits + r * a.stride;
    const RowView<T> row(x, a.classes);
    Running run;
    uint64_t best = 0, kth = 0;  // pieces, by (order of the largest logit, ~piece)
    for (int j0 = 0; j0 < row.pieces; j0 += 32 * kAhead) {
        float v[kAhead][E], top = -INFINITY;
        uint64_t key[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int j = j0 + 32 * k + lane;
            key[k] = 0;
            if (j < row.pieces) {
                row.load(j, v[k], -INFINITY);
                float t = v[k][0];
#pragma unroll
                for (int e = 1; e < E; ++e) t = fmaxf(t, v[k][e]);
                if (TOP) key[k] = (uint64_t)order_of(t) << 32 | (uint32_t)~j;
                top = fmaxf(top, t);
            }
        }
        run.raise(top);
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (j0 + 32 * k + lane < row.pieces) run.add(v[k]);
        if constexpr (TOP) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (__any_sync(kAll, key[k] > kth)) {
                    best = merge_keys(best, __shfl_sync(kAll, sort_keys(key[k], lane), 31 - lane), lane);
                    kth = __shfl_sync(kAll, best, a.top - 1);
                }
        }
    }
    const Stats st = join_lanes<32>(run.stats());
    const float log_s = logf(st.s);
    if (lane == 0) {
        const uint32_t t = a.targets[r];
        const float h = log_s - kLn2 * st.w / st.s;
        a.logprob[r] = t < (uint32_t)a.classes ? ((float)x[t] - st.m) - log_s : __int_as_float(0x7fffffff);
        a.entropy[r] = h;
        if (a.stats) a.stats[3 * r] = st.m, a.stats[3 * r + 1] = log_s, a.stats[3 * r + 2] = h;
    }
    if constexpr (TOP) {
        const int j = (int)~(uint32_t)best;
        const bool mine = lane < a.top && best != 0;
        float v[E];
        if (mine) row.load(j, v, -INFINITY);
        uint64_t found = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            uint64_t key = 0;
            if (mine) {
                const int i = row.first(j) + e;
                const uint64_t high = (uint64_t)order_of(v[e]) << 32;
                if (i >= 0 && i < a.classes && (high | (uint32_t)~j) >= kth) key = high | (uint32_t)~i;
            }
            if (__any_sync(kAll, key != 0))
                found = merge_keys(found, __shfl_sync(kAll, sort_keys(key, lane), 31 - lane), lane);
        }
        if (lane < a.top) {
            const int i = (int)~(uint32_t)found;
            a.top_ids[r * a.top + lane] = i;
            a.top_logprobs[r * a.top + lane] = ((float)x[i] - st.m) - log_s;
        }
    }
}

struct Bwd {
    const void* logits;
    void* dlogits;
    int64_t stride, dstride;
    const uint32_t* targets;
    const float *stats, *g_logprob, *g_entropy;
    int classes;
};

template <typename T>
__device__ __forceinline__ void store_piece(T* p, const float (&d)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(d[0], d[1]), pack_bf16(d[2], d[3]), pack_bf16(d[4], d[5]),
                                                  pack_bf16(d[6], d[7]));
    else
        *reinterpret_cast<float4*>(p) = make_float4(d[0], d[1], d[2], d[3]);
}

// grid: (rows, splits of a row).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_bwd_kernel(Bwd a) {
    constexpr int E = RowView<T>::E;
    after_prior_kernels();
    may_start_next();
    const int64_t r = blockIdx.x;
    const RowView<T> row((const T*)a.logits + r * a.stride, a.classes);
    T* out = (T*)a.dlogits + r * a.dstride;
    const bool together = (((uintptr_t)row.x ^ (uintptr_t)out) & 15) == 0;  // pieces line up in both rows
    const float m = a.stats[3 * r], log_s = a.stats[3 * r + 1], h = a.stats[3 * r + 2];
    const uint32_t t = a.targets[r];
    float gt = a.g_logprob ? a.g_logprob[r] : 0.f;
    if (a.g_logprob && t >= (uint32_t)a.classes) gt = __int_as_float(0x7fffffff);  // as its log probability
    const float gh = a.g_entropy ? a.g_entropy[r] : 0.f;
    const float c = gt + gh * h;
    const uint64_t minus_m = f2_pack(-m, -m), minus_ls = f2_pack(-log_s, -log_s), l2 = f2_pack(kLog2e, kLog2e);
    const uint64_t minus_gh = f2_pack(-gh, -gh), minus_c = f2_pack(-c, -c);
    // p (-g_H ln p - (g_t + g_H H)), and g_t more at the target
    auto gradient = [&](float (&v)[E], int i0) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float z0, z1, p0, p1;
            ptx::f2_unpack(f2_add(f2_add(f2_pack(v[e], v[e + 1]), minus_m), minus_ls), z0, z1);
            const uint64_t z = f2_pack(max_nan(z0, kFloor), max_nan(z1, kFloor));
            ptx::f2_unpack(f2_mul(z, l2), p0, p1);
            ptx::f2_unpack(f2_mul(f2_pack(ex2(p0), ex2(p1)), f2_fma(minus_gh, z, minus_c)), v[e], v[e + 1]);
        }
        if ((int)t - i0 >= 0 && (int)t - i0 < E) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (i0 + e == (int)t) v[e] += gt;
        }
    };
    auto one = [&](int j) {
        float v[E];
        row.load(j, v, 0.f);
        gradient(v, row.first(j));
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = row.first(j) + e;
            if (i >= 0 && i < a.classes) out[i] = T(v[e]);
        }
    };
    const int mine = blockIdx.y * kThreads + threadIdx.x, step = gridDim.y * kThreads, end = row.end();
    if (!together) {
        for (int j = mine; j < row.pieces; j += step) one(j);
        return;
    }
    if (mine == 0 && !row.whole(0)) one(0);
    int j0 = mine < row.begin() ? mine + step : mine;
    auto batch = [&](auto all) {
        uint4 u[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (decltype(all)::value || j0 + k * step < end) u[k] = row.raw(j0 + k * step);
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (decltype(all)::value || j0 + k * step < end) {
                float v[E];
                RowView<T>::decode(u[k], v);
                gradient(v, row.first(j0 + k * step));
                store_piece(out + row.first(j0 + k * step), v);
            }
    };
    for (; j0 + (kAhead - 1) * step < end; j0 += kAhead * step) batch(std::true_type{});
    if (j0 < end) batch(std::false_type{});
    const int last = row.pieces - 1;
    if (last > 0 && last >= end && last % step == mine) one(last);
}

template <typename T, bool TOP>
cudaError_t launch_fwd(cudaStream_t st, int sm_count, Fwd a, int rows) {
    const int pieces = (int)(((int64_t)a.classes * (int)sizeof(T) + 15) / 16) + 1;
    const bool many = rows >= 8 * sm_count;  // enough for every place on the SMs
    // A warp a row where a CTA's joins would cost more than its threads gain: 8192 rows of 1200 bf16 (151
    // pieces) take 9.3 us by warps and 13.3 by 128 threads, of 2500 15.4 and 17.9; with 5 alternatives,
    // whose list costs a warp more, of 800 26.8 and 31.5, of 1800 40.8 and 33.0. A few hundred rows
    // are better off with CTAs (300 of 400: 2.4 and 2.2 us, with alternatives 7.8 and 4.6) unless they are
    // very short (of 50: 2.4 and 2.9).
    if (pieces <= (many ? TOP ? 128 : 256 : TOP ? 0 : 32))
        return launch_overlapped(st, token_logprobs_warp_kernel<T, TOP>, dim3(((unsigned)rows + kWarps - 1) / kWarps),
                                 kThreads, 0, 0, a, rows);
    a.splits = 1;
    // Smaller CTAs join for less, as long as they are enough to load what the bandwidth allows: 8192
    // rows of 5000 bf16 take 22 us by 128 threads and 31 by 256, with 20 alternatives 53 and 74; of 32000
    // 89 and 94, 145 and 157; of 65000 with alternatives 291 and 251. 600 rows of 5000 with 5 alternatives take
    // 7.9 and 9.5 us, 600 of 16000 without 8.6 and 6.9.
    if (pieces <= (many ? 4096 : rows >= sm_count ? 1024 : kThreads))
        return launch_overlapped(st, token_logprobs_kernel<T, TOP, kThreads / 2>, dim3((unsigned)rows), kThreads / 2, 0, 0, a);
    // Very long rows with alternatives: larger ones, so that less of the row is looked at again (515
    // rows of 131071 f32 with 20: 57 us against 62).
    if constexpr (TOP) {
        if (rows >= sm_count && pieces > 8192)
            return launch_overlapped(st, token_logprobs_kernel<T, TOP, 2 * kThreads>, dim3((unsigned)rows), 2 * kThreads, 0,
                                     0, a);
    }
    // Rows that do not occupy the SMs are split over a cluster each, as long as every thread keeps
    // a piece. More splits only repeat the joins (515 rows of 131071 f32 with 20
    // alternatives: 62 us whole, 64 in two, 91 in eight).
    while (a.splits < 8 && rows * (int64_t)a.splits < sm_count && pieces > kThreads * a.splits) a.splits *= 2;
    return launch_overlapped(st, token_logprobs_kernel<T, TOP, kThreads>, dim3((unsigned)rows * (unsigned)a.splits),
                             kThreads, 0, a.splits > 1 ? a.splits : 0, a);
}

}  // namespace

cudaError_t token_logprobs_fwd(cudaStream_t st, int sm_count, hx_dtype dt, const void* logits, int64_t stride,
                               const uint32_t* targets, float* logprob, float* entropy, float* stats, int top,
                               int32_t* top_ids, float* top_logprobs, int rows, int classes) {
    const Fwd a{logits, stride, targets, logprob, entropy, stats, top_logprobs, top_ids, classes, top, 1};
    if (dt == HX_F32)
        return top > 0 ? launch_fwd<float, true>(st, sm_count, a, rows) : launch_fwd<float, false>(st, sm_count, a, rows);
    return top > 0 ? launch_fwd<__nv_bfloat16, true>(st, sm_count, a, rows)
                   : launch_fwd<__nv_bfloat16, false>(st, sm_count, a, rows);
}

cudaError_t token_logprobs_bwd(cudaStream_t st, int sm_count, hx_dtype dt, const void* logits, int64_t stride,
                               const uint32_t* targets, const float* stats, const float* g_logprob,
                               const float* g_entropy, void* dlogits, int64_t dstride, int rows, int classes) {
    const Bwd a{logits, dlogits, stride, dstride, targets, stats, g_logprob, g_entropy, classes};
    const int pieces = (int)(((int64_t)classes * (dt == HX_F32 ? 4 : 2) + 15) / 16) + 1;
    int splits = (int)((4ll * sm_count + rows - 1) / rows);  // few rows: several CTAs each
    const int most = (pieces + kThreads - 1) / kThreads;
    if (splits > most) splits = most;
    const dim3 grid((unsigned)rows, (unsigned)splits);
    return launch_overlapped(st, dt == HX_F32 ? token_logprobs_bwd_kernel<float> : token_logprobs_bwd_kernel<__nv_bfloat16>,
                             grid, kThreads, 0, 0, a);
}

}  // namespace hx
