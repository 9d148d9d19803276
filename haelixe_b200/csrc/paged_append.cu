// New tokens entering a paged key/value cache: k and q are rotated at the
// tokens' own positions on the way (the pairs of src/kernels/rope.rs:5-44), v is copied.
//
// Bytes bound it for a prompt (every element is read and written once) and
// launch latency for a decode step. The rotation angle is that of the
// position p alone, not of a table row, so it is reduced in f64: p * freq / 2 pi
// loses its whole turns there, and only the remaining fraction of a turn is
// rounded to f32. An f32 product would be off by p * 2^-24 radians, which at
// p = 10^5 is more than a bf16 rounding of the result. One CTA computes the
// D/2 (cos, sin) pairs of its token once, for all of its heads.
#include "hx_internal.h"
#include "launch.h"
#include "mma_bf16.cuh"

namespace hx {
namespace {

constexpr int kThreads = 128;

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    if constexpr (sizeof(T) == 2 && VEC) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = unpack_bf16(w[i]);
            f[2 * i] = v.x, f[2 * i + 1] = v.y;
        }
    } else if constexpr (VEC) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
        f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)p[i];
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    if constexpr (sizeof(T) == 2 && VEC) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]),
                                                  pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    } else if constexpr (VEC) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = T(f[i]);
    }
}

// grid: (tokens, splits of the token's 8-element vectors). The vectors of a
// token: k heads, v heads, then q heads (none when q is NULL).
// VEC: q, q_out, k and v rows start on 16-byte boundaries (the cache's always do).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(PagedAppend a) {
    __shared__ float2 cs[128];  // (cos, sin) of each pair
    after_prior_kernels();
    may_start_next();
    const int t = blockIdx.x;
    const int seq = a.seq_ids[t];
    if (seq < 0) return;  // padding: nothing of this token is touched
    const int pos = a.positions[t];
    const PagedView& c = a.cache;
    int64_t slot = -1;  // element offset of the token's cache slot, -1: no such slot
    if (seq < c.num_seqs && pos >= 0) {
        const int col = c.page_shift >= 0 ? pos >> c.page_shift : pos / c.page_size;
        if (col < c.max_pages) {
            const int page = c.table[(int64_t)seq * c.table_stride + col];
            if (page >= 0 && page < c.num_pages)
                slot = (int64_t)page * c.sp + (int64_t)(pos - col * c.page_size) * c.ss;
        }
    }
    if (a.rotate) {
        for (int i = threadIdx.x; i < c.D / 2; i += kThreads) {
            const double turns = (double)pos * (exp2(a.log2_base * (-2.0 * i / c.D)) * 0.15915494309189533577);
            float s, co;
            sincospif(2.f * (float)(turns - rint(turns)), &s, &co);
            cs[i] = make_float2(co, s);
        }
        __syncthreads();
    }
    const int per_head = c.D / 8;
    const int nk = c.H * per_head, total = 2 * nk + a.Hq * per_head;
    for (int i = blockIdx.y * kThreads + threadIdx.x; i < total; i += gridDim.y * kThreads) {
        const bool is_q = i >= 2 * nk, is_v = !is_q && i >= nk;
        const int j = is_q ? i - 2 * nk : is_v ? i - nk : i;
        const int h = j / per_head, d = 8 * (j - h * per_head);
        if (!is_q && slot < 0) continue;
        const T* src = is_q ? (const T*)a.q + (int64_t)t * a.q_st + (int64_t)h * a.q_sh
                       : is_v ? (const T*)a.v + (int64_t)t * a.v_st + (int64_t)h * a.v_sh
                              : (const T*)a.k + (int64_t)t * a.k_st + (int64_t)h * a.k_sh;
        float x[8];
        load8<T, VEC>(src + d, x);
        if (a.rotate && !is_v) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float2 r = cs[d / 2 + p];
                const float x0 = x[2 * p], x1 = x[2 * p + 1];
                x[2 * p] = x0 * r.x - x1 * r.y;
                x[2 * p + 1] = x0 * r.y + x1 * r.x;
            }
        }
        if (is_q) {
            if (slot < 0) {  // a position without a slot shows in its query
#pragma unroll
                for (int p = 0; p < 8; ++p) x[p] = __int_as_float(0x7fffffff);
            }
            store8<T, VEC>((T*)a.q_out + (int64_t)t * a.qo_st + (int64_t)h * a.qo_sh + d, x);
        } else {
            store8<T, true>((is_v ? (T*)c.v : (T*)c.k) + slot + (int64_t)h * c.sh + d, x);
        }
    }
}

bool rows16(const void* p, int64_t st, int64_t sh, int eb) {
    return (uintptr_t)p % 16 == 0 && (st * eb) % 16 == 0 && (sh * eb) % 16 == 0;
}

template <typename T>
cudaError_t launch(cudaStream_t st, int sm_count, const PagedAppend& a, int tokens) {
    const int eb = (int)sizeof(T);
    const bool vec = rows16(a.k, a.k_st, a.k_sh, eb) && rows16(a.v, a.v_st, a.v_sh, eb) &&
                     (a.q == nullptr || (rows16(a.q, a.q_st, a.q_sh, eb) && rows16(a.q_out, a.qo_st, a.qo_sh, eb)));
    // One CTA a token; a few tokens are spread over more CTAs, so that the
    // heads of one token do not queue behind each other.
    const int total = (2 * a.cache.H + a.Hq) * (a.cache.D / 8);
    int splits = (int)((2ll * sm_count + tokens - 1) / tokens);
    const int most = (total + kThreads - 1) / kThreads;
    if (splits > most) splits = most;
    const dim3 grid((unsigned)tokens, (unsigned)splits);
    return launch_overlapped(st, vec ? paged_append_kernel<T, true> : paged_append_kernel<T, false>, grid, kThreads, 0, 0, a);
}

}  // namespace

cudaError_t paged_append(cudaStream_t st, int sm_count, hx_dtype dt, const PagedAppend& a, int tokens) {
    if (dt == HX_F32) return launch<float>(st, sm_count, a, tokens);
    return launch<__nv_bfloat16>(st, sm_count, a, tokens);
}

}  // namespace hx
