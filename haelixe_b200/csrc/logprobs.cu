// Log probabilities of given tokens under logits [rows, classes], with the
// entropy and the most likely alternatives of each row, and their gradient:
//   z_i = x_i - m (m the row's maximum), s = sum e^{z_i}, w = sum z_i e^{z_i}
//   logp(t) = z_t - ln s,  H = ln s - w / s
//   dx_i = g_t (1[i = t] - p_i) - g_H p_i (ln p_i + H)
// One read of the logits forward, one read and one write backward: bytes bound
// both, and next to them the exponentials (one a logit). The forward keeps
// (m, s, w) running, so the row is read once; both terms of H are
// positive, so nothing cancels. Sums are f32, per thread and then joined in a
// tree, the same for every call.
//
// The alternatives need no second pass over the row either. Each thread knows the
// best of its own logits; the k best threads' values bound the k-th best logit
// from below, and every logit that reaches the bound belongs to one of those k
// threads, so only their share of the row (k / 512 of it) is looked at again.
// Ties go to the lower index.
#include "hx_internal.h"
#include "mma_bf16.cuh"

namespace hx {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -3.402823466e+38f;
constexpr float kFloor = -1.0e4f;  // exp2 of it is 0; keeps 0 * (-inf) out of the sums
constexpr unsigned kAll = 0xffffffffu;

// max that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Bits that order as the values do; NaN orders as -inf, -0 as 0. Never 0.
__device__ __forceinline__ uint32_t order_of(float v) {
    if (!(v == v)) v = -INFINITY;
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
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
    __device__ __forceinline__ void decode(const uint4& u, float (&v)[E]) const {
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
    // Elements outside the row read as `pad`.
    __device__ __forceinline__ void load(int j, float (&v)[E], float pad) const {
        if (whole(j)) {
            decode(*reinterpret_cast<const uint4*>(x + first(j)), v);
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

template <int E>
__device__ __forceinline__ void add_piece(Stats& st, const float (&v)[E], float top) {
    if (top > st.m) {
        const float d = weight_of(st.m, top), e = ex2(d);
        st.w = e * (st.w + d * st.s);
        st.s *= e;
        st.m = top;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float z = max_nan((v[i] - st.m) * kLog2e, kFloor), e = ex2(z);
        st.s += e;
        st.w = fmaf(z, e, st.w);
    }
}

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
// Every warp brings a sorted list; warp 0 leaves with the 32 largest of all.
__device__ __forceinline__ uint64_t block_largest(uint64_t k, uint64_t (*lists)[32], int warp, int lane) {
    lists[warp][lane] = k;
#pragma unroll
    for (int s = kWarps / 2; s > 0; s >>= 1) {
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
    int classes, top;
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(Fwd a) {
    constexpr int E = RowView<T>::E, kAhead = 4;
    __shared__ Stats parts[kWarps];
    __shared__ uint64_t lists[TOP ? kWarps : 1][32];
    __shared__ uint64_t chosen[32];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const T* x = (const T*)a.logits + r * a.stride;
    const RowView<T> row(x, a.classes);

    Stats st{kLowest, 0.f, 0.f};
    uint64_t best = 0;  // (order of the value, ~piece)
    for (int j0 = tid; j0 < row.pieces; j0 += kAhead * kThreads) {
        float v[kAhead][E];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = j0 + u * kThreads;
            if (j < row.pieces) row.load(j, v[u], -INFINITY);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = j0 + u * kThreads;
            if (j >= row.pieces) break;
            float top = v[u][0];
#pragma unroll
            for (int e = 1; e < E; ++e) top = fmaxf(top, v[u][e]);
            if constexpr (TOP) {
                const uint64_t key = (uint64_t)order_of(top) << 32 | (uint32_t)~j;
                best = key > best ? key : best;
            }
            add_piece(st, v[u], top);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        st = join(st, Stats{__shfl_xor_sync(kAll, st.m, o), __shfl_xor_sync(kAll, st.s, o), __shfl_xor_sync(kAll, st.w, o)});
    if (lane == 0) parts[warp] = st;
    __syncthreads();
    st = parts[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) st = join(st, parts[w]);
    const float log_s = logf(st.s);
    if (tid == 0) {
        const uint32_t t = a.targets[r];
        const float h = log_s - kLn2 * st.w / st.s;
        a.logprob[r] = t < (uint32_t)a.classes ? ((float)x[t] - st.m) - log_s : __int_as_float(0x7fffffff);
        a.entropy[r] = h;
        if (a.stats) a.stats[3 * r] = st.m, a.stats[3 * r + 1] = log_s, a.stats[3 * r + 2] = h;
    }
    if constexpr (TOP) {
        const uint64_t k = block_largest(sort_keys(best, lane), lists, warp, lane);
        if (warp == 0) chosen[lane] = k;
        __syncthreads();
        const uint64_t bound = chosen[a.top - 1];
        // The chosen threads' pieces again, each by a warp; a piece's element counts when
        // (its order, ~its piece) reaches the bound.
        uint64_t mine = 0;
        for (int c = warp; c < a.top; c += kWarps) {
            if (chosen[c] == 0) break;
            const int owner = (int)(~(uint32_t)chosen[c] % kThreads);
            for (int j0 = owner; j0 < row.pieces; j0 += 32 * kThreads) {
                const int j = j0 + lane * kThreads;
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
                    if (__any_sync(kAll, key != 0)) {
                        const uint64_t sorted = sort_keys(key, lane);
                        mine = merge_keys(mine, __shfl_sync(kAll, sorted, 31 - lane), lane);
                    }
                }
            }
        }
        const uint64_t found = block_largest(mine, lists, warp, lane);
        if (warp == 0 && lane < a.top) {
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
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(Bwd a) {
    constexpr int E = RowView<T>::E;
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
    for (int j = blockIdx.y * kThreads + threadIdx.x; j < row.pieces; j += gridDim.y * kThreads) {
        float v[E];
        row.load(j, v, 0.f);
        const int i0 = row.first(j);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float z = max_nan((v[e] - m) - log_s, kFloor);
            const float p = ex2(z * kLog2e);
            v[e] = -p * fmaf(gh, z, c) + (i0 + e == (int)t ? gt : 0.f);
        }
        if (together && row.whole(j)) {
            store_piece(out + i0, v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (i0 + e >= 0 && i0 + e < a.classes) out[i0 + e] = T(v[e]);
        }
    }
}

}  // namespace

cudaError_t token_logprobs_fwd(cudaStream_t st, hx_dtype dt, const void* logits, int64_t stride, const uint32_t* targets,
                               float* logprob, float* entropy, float* stats, int top, int32_t* top_ids,
                               float* top_logprobs, int rows, int classes) {
    const Fwd a{logits, stride, targets, logprob, entropy, stats, top_logprobs, top_ids, classes, top};
    if (dt == HX_F32) {
        if (top > 0)
            token_logprobs_kernel<float, true><<<(unsigned)rows, kThreads, 0, st>>>(a);
        else
            token_logprobs_kernel<float, false><<<(unsigned)rows, kThreads, 0, st>>>(a);
    } else if (top > 0) {
        token_logprobs_kernel<__nv_bfloat16, true><<<(unsigned)rows, kThreads, 0, st>>>(a);
    } else {
        token_logprobs_kernel<__nv_bfloat16, false><<<(unsigned)rows, kThreads, 0, st>>>(a);
    }
    note_launch();
    return cudaGetLastError();
}

cudaError_t token_logprobs_bwd(cudaStream_t st, int sm_count, hx_dtype dt, const void* logits, int64_t stride,
                               const uint32_t* targets, const float* stats, const float* g_logprob,
                               const float* g_entropy, void* dlogits, int64_t dstride, int rows, int classes) {
    const Bwd a{logits, dlogits, stride, dstride, targets, stats, g_logprob, g_entropy, classes};
    const int pieces = (int)(((int64_t)classes * (dt == HX_F32 ? 4 : 2) + 15) / 16) + 1;
    int splits = (4 * sm_count + rows - 1) / rows;  // few rows: several CTAs each
    const int most = (pieces + kThreads - 1) / kThreads;
    if (splits > most) splits = most;
    const dim3 grid((unsigned)rows, (unsigned)splits);
    if (dt == HX_F32)
        token_logprobs_bwd_kernel<float><<<grid, kThreads, 0, st>>>(a);
    else
        token_logprobs_bwd_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a);
    note_launch();
    return cudaGetLastError();
}

}  // namespace hx
