// Linear products with 4-bit weights for a few tokens:
//   y[r, n] = sum_k x[r, k] (q[k, n] - 8) s[k / group, n] (+ bias[n]) (+ residual[r, n])
// q holds 8 consecutive k of a column in a word, the first in the lowest bits.
//
// The weights' bytes bound it (half a byte for each, against 2 rows FLOP), so a
// weight is read once for up to 32 rows and unpacking has to stay cheap: at half
// a byte a weight the memory delivers about 90 weights a clock and SM. Two nibbles
// become two bf16 in three instructions (0x4300 | q is 128 + q, minus 136), and the
// warp's tensor product multiplies them, so that the f32 pipes only see one scale a
// 32-deep step. The order of k inside a product is free as long as both operands
// agree, so the weights go from a 16-byte global load (4 columns of 8 k) to fragments
// with no shared memory. q - 8 and bf16 x are exact operands; f32 x is cut into
// three bf16 that sum to it exactly, three products for one.
//
// A CTA's 8 warps take every 8th step of the same 32 columns; a cluster of up to 8
// CTAs splits k further where there are few columns, and joins its sums through
// distributed shared memory in a fixed order.
#include <cooperative_groups.h>

#include "hx_internal.h"
#include "mma_bf16.cuh"

namespace hx {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kCols = 32, kStep = 32;  // columns of a CTA, k of a warp's step
constexpr int kAhead = 4;              // steps whose loads are in flight together

struct Args {
    const void* x;
    const uint32_t* packed;
    const void *scales, *bias, *residual;
    void* y;
    int rows, in, out, group;
    bool vec_x, vec_w;  // 16-byte loads fit the rows of x; of packed, scales
};

// q - 8 of nibbles p and p + 4 of w, as bf16.
__device__ __forceinline__ uint32_t weights_of(uint32_t w, int p) {
    const uint32_t u = ((w >> (4 * p)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(136.f));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 8 consecutive x as PARTS sets of 4 words, whose sum they are, in the weights' order:
// words (x0, x4), (x1, x5), (x2, x6), (x3, x7).
template <typename T>
struct X8;
template <>
struct X8<__nv_bfloat16> {
    static constexpr int PARTS = 1;
    uint4 raw;
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int valid, bool vec) {
        if (vec && valid >= 8) {
            raw = *reinterpret_cast<const uint4*>(p);
        } else {
            const uint16_t* s = reinterpret_cast<const uint16_t*>(p);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = (2 * i < valid ? s[2 * i] : 0u) | (2 * i + 1 < valid ? (uint32_t)s[2 * i + 1] << 16 : 0u);
            raw = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __device__ __forceinline__ void words(uint32_t (&b)[1][4]) const {
        b[0][0] = pair_lo(raw.x, raw.z);
        b[0][1] = pair_hi(raw.x, raw.z);
        b[0][2] = pair_lo(raw.y, raw.w);
        b[0][3] = pair_hi(raw.y, raw.w);
    }
};
template <>
struct X8<float> {
    static constexpr int PARTS = 3;
    float v[8];
    __device__ __forceinline__ void load(const float* p, int valid, bool vec) {
        if (vec && valid >= 8) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < valid ? p[i] : 0.f;
        }
    }
    // The upper 8 bits of the mantissa, the next 8 and the rest, each exact in bf16.
    // Infinities and NaN stay whole in the first part.
    __device__ __forceinline__ void words(uint32_t (&b)[3][4]) const {
        uint32_t part[3][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t u = __float_as_uint(v[i]);
            const bool finite = (u & 0x7f800000u) != 0x7f800000u;
            const float h = __uint_as_float(u & 0xffff0000u), r = v[i] - h;
            const float m = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
            part[0][i] = finite || (u & 0x007fffffu) == 0 ? u : u | 0x00400000u;
            part[1][i] = finite ? __float_as_uint(r) : 0u;
            part[2][i] = finite ? __float_as_uint(r - m) : 0u;
        }
#pragma unroll
        for (int s = 0; s < 3; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) b[s][i] = pair_hi(part[s][i], part[s][i + 4]);
    }
};

__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 u;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "l"(p));
    return u;
}

template <typename T>
__device__ __forceinline__ float4 load4(const T* p, bool vec, int valid) {
    if (vec && valid >= 4) {
        if constexpr (sizeof(T) == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y);
            return make_float4(a.x, a.y, b.x, b.y);
        } else {
            return *reinterpret_cast<const float4*>(p);
        }
    }
    return make_float4(valid > 0 ? (float)p[0] : 0.f, valid > 1 ? (float)p[1] : 0.f, valid > 2 ? (float)p[2] : 0.f,
                       valid > 3 ? (float)p[3] : 0.f);
}

// NT: sets of 8 rows. grid: (column tiles x cluster, passes of 8 NT rows).
template <typename T, int NT>
__global__ void __launch_bounds__(kThreads) linear_w4_kernel(Args a) {
    constexpr int R = 8 * NT, PARTS = X8<T>::PARTS;
    __shared__ float part[kWarps][R][kCols + 1];
    __shared__ float sums[R][kCols];
    cg::cluster_group cluster = cg::this_cluster();
    const int ks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int n0 = (blockIdx.x / ks) * kCols, r0 = blockIdx.y * R;
    const int n = n0 + 4 * g, cols = a.out - n;  // this lane's 4 columns, those that exist
    const int octets = (a.in + 7) / 8, steps = (a.in + kStep - 1) / kStep;
    const T* x = (const T*)a.x;
    const T* scales = (const T*)a.scales;

    float acc[2][NT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;

    const int stride = kWarps * ks;
    for (int s0 = rank * kWarps + warp; s0 < steps; s0 += kAhead * stride) {
        uint4 w[kAhead];
        float4 sc[kAhead];
        X8<T> xs[kAhead][NT];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int s = s0 + u * stride, o = 4 * s + t;  // this lane's 8 k: 8 o ... 8 o + 7
            w[u] = make_uint4(0, 0, 0, 0);
            sc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (s < steps && cols > 0) {
                if (o < octets) {
                    const uint32_t* p = a.packed + (int64_t)o * a.out + n;
                    if (a.vec_w)
                        w[u] = ld_stream(p);
                    else
                        w[u] = make_uint4(p[0], cols > 1 ? p[1] : 0u, cols > 2 ? p[2] : 0u, cols > 3 ? p[3] : 0u);
                }
                sc[u] = load4<T>(scales + (int64_t)(s * kStep / a.group) * a.out + n, a.vec_w, cols);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int row = r0 + 8 * j + g;
                const bool live = s < steps && row < a.rows;
                xs[u][j].load(x + (live ? (int64_t)row * a.in + 8 * o : 0), live ? a.in - 8 * o : 0, a.vec_x);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            float d[2][NT][4];
            uint32_t b[NT][PARTS][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                xs[u][j].words(b[j]);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[i][j][e] = 0.f;
            }
            const uint32_t col[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int p = 0; p < 4; p += 2) {
                    const uint32_t a0 = weights_of(col[2 * i], p), a1 = weights_of(col[2 * i + 1], p);
                    const uint32_t a2 = weights_of(col[2 * i], p + 1), a3 = weights_of(col[2 * i + 1], p + 1);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int q = PARTS - 1; q >= 0; --q)
                            mma_bf16(d[i][j], a0, a1, a2, a3, b[j][q][p], b[j][q][p + 1]);
                }
            const float s[4] = {sc[u].x, sc[u].y, sc[u].z, sc[u].w};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(s[2 * i + (e >> 1)], d[i][j][e], acc[i][j][e]);
        }
    }
    // acc[i][j][e]: column 4 g + 2 i + e / 2, row 8 j + 2 t + e % 2
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[warp][8 * j + 2 * t + (e & 1)][4 * g + 2 * i + (e >> 1)] = acc[i][j][e];
    __syncthreads();
    const int live = min(R, a.rows - r0);
    for (int i = threadIdx.x; i < live * kCols; i += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) v += part[k][i / kCols][i % kCols];
        sums[i / kCols][i % kCols] = v;
    }
    if (ks > 1) cluster.sync();
    // Each CTA of the cluster finishes its share of the rows.
    for (int i = rank * kThreads + threadIdx.x; i < live * kCols; i += ks * kThreads) {
        const int r = i / kCols, c = i % kCols;
        float v = 0.f;
        if (ks > 1) {
            for (int k = 0; k < ks; ++k) v += cluster.map_shared_rank(&sums[0][0], k)[i];
        } else {
            v = sums[r][c];
        }
        if (n0 + c < a.out) {
            const int64_t at = (int64_t)(r0 + r) * a.out + n0 + c;
            if (a.bias) v += (float)((const T*)a.bias)[n0 + c];
            if (a.residual) v += (float)((const T*)a.residual)[at];
            ((T*)a.y)[at] = T(v);
        }
    }
    if (ks > 1) cluster.sync();  // no CTA leaves while its sums are read
}

// One thread a column of a group: s = max |w| / 7, q = round(w / s) + 8.
template <typename T>
__global__ void __launch_bounds__(256) quantize_w4_kernel(const T* w, uint32_t* packed, T* scales, int in, int out,
                                                          int group) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= out) return;
    for (int gi = blockIdx.y; (int64_t)gi * group < in; gi += gridDim.y) {
        const int k0 = gi * group, k1 = min(in, k0 + group);
        float top = 0.f;
        for (int k = k0; k < k1; ++k) {
            const float v = fabsf((float)w[(int64_t)k * out + n]);
            top = v > top || v != v ? v : top;
        }
        const T st = T(top / 7.f);
        const float s = (float)st;
        scales[(int64_t)gi * out + n] = st;
        for (int o = k0 / 8; 8 * o < k1; ++o) {
            uint32_t word = 0;
            for (int i = 0; i < 8; ++i) {
                const int k = 8 * o + i;
                const float v = k < k1 && s > 0.f ? (float)w[(int64_t)k * out + n] / s : 0.f;
                word |= (uint32_t)(int)fminf(fmaxf(rintf(v) + 8.f, 0.f), 15.f) << (4 * i);
            }
            packed[(int64_t)o * out + n] = word;
        }
    }
}

template <typename T, int NT>
cudaError_t launch(cudaStream_t st, int sm_count, const Args& a) {
    const int tiles = (a.out + kCols - 1) / kCols, steps = (a.in + kStep - 1) / kStep;
    int ks = 1;
    while (ks < 8 && tiles * ks < 3 * sm_count && steps >= 2 * kWarps * kAhead * ks) ks *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(tiles * ks), (unsigned)((a.rows + 8 * NT - 1) / (8 * NT)));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)ks;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_w4_kernel<T, NT>, a);
    if (e == cudaSuccess) note_launch();
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T>
cudaError_t by_rows(cudaStream_t st, int sm_count, const Args& a) {
    if (a.rows <= 8) return launch<T, 1>(st, sm_count, a);
    if (a.rows <= 16) return launch<T, 2>(st, sm_count, a);
    return launch<T, 4>(st, sm_count, a);
}

}  // namespace

cudaError_t linear_w4(cudaStream_t st, int sm_count, hx_dtype dt, const void* x, const uint32_t* packed,
                      const void* scales, const void* bias, const void* residual, void* y, int rows, int in, int out,
                      int group) {
    const int eb = dt == HX_F32 ? 4 : 2;
    Args a{x, packed, scales, bias, residual, y, rows, in, out, group, false, false};
    a.vec_x = (uintptr_t)x % 16 == 0 && ((int64_t)in * eb) % 16 == 0;
    a.vec_w = (uintptr_t)packed % 16 == 0 && (uintptr_t)scales % 16 == 0 && out % 4 == 0;
    return dt == HX_F32 ? by_rows<float>(st, sm_count, a) : by_rows<__nv_bfloat16>(st, sm_count, a);
}

cudaError_t quantize_w4(cudaStream_t st, hx_dtype dt, const void* w, uint32_t* packed, void* scales, int in, int out,
                        int group) {
    const int groups = (in + group - 1) / group;
    const dim3 grid((unsigned)((out + 255) / 256), (unsigned)(groups < 65535 ? groups : 65535));
    if (dt == HX_F32)
        quantize_w4_kernel<float><<<grid, 256, 0, st>>>((const float*)w, packed, (float*)scales, in, out, group);
    else
        quantize_w4_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>((const __nv_bfloat16*)w, packed, (__nv_bfloat16*)scales,
                                                                in, out, group);
    note_launch();
    return cudaGetLastError();
}

}  // namespace hx
