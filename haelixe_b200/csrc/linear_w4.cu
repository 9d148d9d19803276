// Linear products with 4-bit weights for a few tokens:
//   y[r, n] = sum_k x[r, k] (q[k, n] - 8) s[k / group, n] (+ bias[n]) (+ residual[r, n])
// q holds 8 consecutive k of a column in a word, the first in the lowest bits.
//
// The weights' bytes bound it (half a byte for each, against 2 rows FLOP), so a
// weight is read once for up to 32 rows and unpacking has to stay cheap: at half
// a byte a weight the memory delivers about 90 weights a clock and SM. Two nibbles
// become two bf16 in two instructions and a half (see Unpack), and the
// warp's tensor product multiplies them, so that the f32 pipes only see one scale a
// group. 16 rows of 8192 x 8192 in groups of 64 take 15.0 us, of which reading is 5.6. No pipe is full then
// (issue slots 44 %, ALU 34 %, tensor 28 %): the 3.5 warps of a scheduler issue once in 8 cycles each, so the
// latency of unpacking and multiplying bounds it, and filling and joining within so short a call.
// The order of k inside a product is free as long as both operands agree, so one 16-byte read of a stage
// (4 columns of 8 k) is the weights' fragments of four products, with nothing exchanged between lanes.
// q - 8 and bf16 x are exact operands; f32 x is cut into three bf16 that sum to it
// exactly (from 2^-109 up; below, to bf16's smallest step of 2^-133), three products for one.
//
// A CTA's 8 warps form k groups of wn warps: a group takes every so many units of 128 k of
// 64 wn columns (32 wn for over 16 rows), each warp its own columns. A unit's weights and x come
// by TMA into one of the group's two stages while the other is computed on, so the bytes in
// flight cost neither registers nor issue slots (16-byte loads and row-wise bulk copies took longer
// to issue than the products) and x is read once a group. The groups' sums are
// joined in shared memory; a cluster of up to 8 CTAs splits k further where there
// are few columns, and joins its sums through distributed shared memory. Every
// join has a fixed order.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "hx_internal.h"
#include "launch.h"
#include "mma_bf16.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.h"

namespace hx {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kStep = 32;  // k of a warp's tensor products: a lane's one 16-byte read of weights for 32 columns

struct Args {
    CUtensorMap w_map, x_map;
    const void* x;
    const uint32_t* packed;
    const void *scales, *bias, *residual;
    void* y;
    DeviceStatus* status;
    int rows, in, out, group, scale_rows;
    int skip_rows, skip_rest;  // what the other groups of warps take between two units of one, in rows of scales and k
    bool vec_y;          // y on a boundary of 4 elements
    int wn_log, ks_log;  // log2 of the warps that share a unit, side by side, and of the cluster's size
};

// (q - 8) / 64 of nibbles p and p + 4 of w, as bf16. A nibble in the lowest 8 bits of a half, read
// as a (denormal) bf16, is itself times 2^-133, or 2^-129 in the upper 4 bits: one logic operation
// and one fused multiply-add, exact, and one shift for two of the four pairs. (Making 128 + q by a
// shift and a logic operation and taking 136 from it is three for each.)
constexpr float kWeightUnit = 64.f;
struct Unpack {
    uint32_t low, high, minus_8;
    __device__ __forceinline__ Unpack() {
        // Opaque to the compiler, so that they stay in registers.
        asm volatile("mov.b32 %0, 0x7f007f00;" : "=r"(low));      // 2^127
        asm volatile("mov.b32 %0, 0x7d007d00;" : "=r"(high));     // 2^123
        asm volatile("mov.b32 %0, 0xbe00be00;" : "=r"(minus_8));  // -8 / 64
    }
    __device__ __forceinline__ uint32_t scaled(uint32_t bits, uint32_t by) const {
        uint32_t u;
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(u) : "r"(bits), "r"(by), "r"(minus_8));
        return u;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t w, int p) const {
        const uint32_t v = p < 2 ? w : w >> 8;
        return p % 2 == 0 ? scaled(v & 0x000f000fu, low) : scaled(v & 0x00f000f0u, high);
    }
};

// 8 consecutive x as PARTS sets of 4 words, whose sum they are, in the weights' order:
// words (x0, x4), (x1, x5), (x2, x6), (x3, x7).
template <typename T>
struct X8;
template <>
struct X8<__nv_bfloat16> {
    static constexpr int PARTS = 1;
    uint4 raw;
    // The 8 from 16-byte chunk `chunk` of a swizzled row whose number ends in g.
    __device__ __forceinline__ void load(const unsigned char* row, int chunk, int g) {
        raw = *reinterpret_cast<const uint4*>(row + 16 * (chunk ^ g));
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
    __device__ __forceinline__ void load(const unsigned char* row, int chunk, int g) {
        const float4 a = *reinterpret_cast<const float4*>(row + 16 * (chunk ^ g));
        const float4 b = *reinterpret_cast<const float4*>(row + 16 * ((chunk + 1) ^ g));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
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

// 4 bytes, or 4 zero bytes.
__device__ __forceinline__ void copy4_async(void* smem, const void* global, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)),
                 "l"(global), "r"(valid ? 4 : 0)
                 : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// Scales of 4 columns.
template <typename T>
struct alignas(4 * sizeof(T)) S4 {
    T s[4];
};

constexpr int kUnit = 4;                    // steps whose weights and x are copied together
constexpr int kUnitK = kUnit * kStep;       // 128
constexpr int kUnitRows = kUnitK / 8;       // rows of packed words
constexpr int kStages = 2;

// Shared memory of a CTA. A stage holds the group's words as boxes of kUnitRows rows of 32
// (a warp's CH boxes after another's), then x as boxes of R rows of 128 bytes, each 128-byte
// row with its 16-byte chunks exchanged by the row number (the TMA's swizzle). With
// column_of a quarter warp's 16-byte reads of the words fall on all banks. The stages become the
// groups' sums, [8 / wn][R][C + 4].
constexpr int kBox = kUnitRows * 128;
struct Layout {
    int w_bytes, stage, recv, bars, total;  // bytes, then byte offsets
    __host__ __device__ Layout(int R, int CH, int wn, int eb) {
        const int C = 32 * CH * wn, groups = kWarps / wn;
        w_bytes = CH * wn * kBox;
        stage = w_bytes + R * kUnitK * eb;
        const int sums = groups * R * (C + 4) * 4;
        recv = groups * kStages * stage;
        if (recv < sums) recv = (sums + 15) / 16 * 16;
        bars = recv + ((R * C + kThreads - 1) / kThreads + 7) * kThreads * 4;
        total = bars + 2 * groups * kStages * 8 + 16;
    }
};

// First of the 4 columns of lane group g within a set of 32.
__device__ __forceinline__ int column_of(int g) { return 4 * ((g >> 1) | ((g & 1) << 2)); }

// NT: sets of 8 rows; CH: sets of 32 columns of a warp; L: consecutive steps of a unit that
// lie in one group of scales, so that their products are scaled once. grid: (column
// tiles x cluster, passes of 8 NT rows).
// VEC: the rows of x and of packed are multiples of 16 bytes and x, packed and scales are
// aligned, as TMA needs. Otherwise wn is 1 and each warp fills its stages with 4-byte asynchronous
// copies of its own (bf16 x of an odd width with plain loads).
template <typename T, int NT, int CH, int L, bool VEC>
__global__ void __launch_bounds__(kThreads, sizeof(T) * NT * CH <= 8 ? 2 : 1) linear_w4_kernel(const __grid_constant__ Args a) {
    constexpr int R = 8 * NT, PARTS = X8<T>::PARTS, kBoxK = 128 / sizeof(T);  // k of a box of x
    extern __shared__ __align__(1024) unsigned char smem[];
    // Everything that is shared out is a power of two, so that no index costs a division.
    const int wn_log = VEC ? a.wn_log : 0, wn = 1 << wn_log, c_log = (CH == 2 ? 6 : 5) + wn_log, C = 1 << c_log;
    const int groups = kWarps >> wn_log, ks_log = a.ks_log, ks = 1 << ks_log, rank = blockIdx.x & (ks - 1);
    const Layout lay(R, CH, wn, sizeof(T));
    cg::cluster_group cluster = cg::this_cluster();
    if (ks > 1) cluster_arrive();  // waited for before the first write to another CTA: all have started
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int group = warp >> wn_log, sub = warp & (wn - 1);
    const int n0 = (blockIdx.x >> ks_log) << c_log, r0 = blockIdx.y * R;
    const int rows = min(R, a.rows - r0);
    const int octets = (a.in + 7) / 8, units = (a.in + kUnitK - 1) / kUnitK, stride = groups * ks;
    const int first = rank * groups + group;

    unsigned char* stages = smem + group * kStages * lay.stage;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + lay.bars) + 2 * kStages * group;
    volatile int* abort_flag = reinterpret_cast<int*>(smem + lay.bars + 2 * groups * kStages * 8);
    const uint32_t bar = ptx::smem_addr(bars);
    auto full = [&](int i) { return bar + 8 * i; };
    auto empty = [&](int i) { return bar + 8 * (kStages + i); };
    if constexpr (VEC) {
        if (threadIdx.x == 0) *abort_flag = 0;
        if (sub == 0 && lane == 0) {
#pragma unroll
            for (int i = 0; i < kStages; ++i) {
                ptx::mbar_init(full(i), wn);
                ptx::mbar_init(empty(i), wn);
            }
            ptx::fence_mbar_init();
        }
        __syncthreads();
    }
    after_prior_kernels();
    may_start_next();

    // Unit u into stage i: each warp its own words, the group's first warp x as well. What is
    // past the last row, column or k reads as zero.
    auto copy_unit = [&](int u, int i) {
        unsigned char* st = stages + i * lay.stage;
        if constexpr (VEC) {
            if (lane == 0) {
                ptx::mbar_arrive_expect_tx(full(i), CH * kBox + (sub == 0 ? R * kUnitK * (int)sizeof(T) : 0));
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    ptx::tma_load_2d(ptx::smem_addr(st + (CH * sub + c) * kBox), &a.w_map, full(i),
                                     n0 + 32 * (CH * sub + c), kUnitRows * u);
                if (sub == 0)
#pragma unroll
                    for (int c = 0; c < kUnitK / kBoxK; ++c)
                        ptx::tma_load_2d(ptx::smem_addr(st + lay.w_bytes + c * R * 128), &a.x_map, full(i),
                                         kUnitK * u + c * kBoxK, r0);
            }
        } else {
#pragma unroll 4
            for (int k = 0; k < kUnitRows; ++k) {
                const int o = kUnitRows * u + k;
                const uint32_t* from = a.packed + (int64_t)min(o, octets - 1) * a.out;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int n = n0 + 32 * c + lane;
                    copy4_async(st + c * kBox + k * 128 + 4 * (lane ^ (4 * (k & 7))), from + min(n, a.out - 1),
                                n < a.out && o < octets);
                }
            }
            // x: pairs of bf16 where the rows allow it, else single elements
            constexpr int kPer = 4 / sizeof(T);
            const bool words = sizeof(T) == 4 || (a.in % 2 == 0 && ((uintptr_t)a.x & 3) == 0);
            for (int r = 0; r < rows; ++r) {
                const T* from = (const T*)a.x + (int64_t)(r0 + r) * a.in;
                auto place = [&](int k) {  // of element k of the unit, which its pair follows
                    return st + lay.w_bytes + (k / kBoxK) * R * 128 + r * 128 +
                           16 * ((k % kBoxK) * (int)sizeof(T) / 16 ^ (r & 7)) + (k * (int)sizeof(T)) % 16;
                };
                if (words) {
#pragma unroll
                    for (int k = kPer * lane; k < kUnitK; k += 32 * kPer) {
                        const int at = kUnitK * u + k;
                        copy4_async(place(k), from + (at < a.in ? at : 0), at < a.in);
                    }
                } else {
#pragma unroll
                    for (int k = lane; k < kUnitK; k += 32) {
                        const int at = kUnitK * u + k;
                        *reinterpret_cast<T*>(place(k)) = at < a.in ? from[at] : T(0.f);
                    }
                }
            }
        }
    };
    auto copies_commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };

    int col[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        col[c] = n0 + 32 * (CH * sub + c) + column_of(g);
        if (VEC) col[c] = min(col[c], a.out - 4);
    }
    // Steps of a pass of the inner loop, and its scales. It stays a loop: unrolled over a unit, the
    // compiler moves so much of it ahead that registers spill (16 rows of 8192 x 8192 in groups of 64:
    // 21.2 us).
    constexpr int kPass = L == 1 ? 2 : L;
    S4<T> sc[kPass / L][CH];
    // Row of the next scales to load, and k from its first; between two units of this group of warps lie
    // a.skip_rows rows and a.skip_rest k.
    int scale_row = kUnitK * first / a.group, scale_rest = kUnitK * first - scale_row * a.group;
    auto load_scales = [&](int l, bool last_of_unit) {
        const T* p = (const T*)a.scales + (int64_t)min(scale_row, a.scale_rows - 1) * a.out;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if constexpr (VEC) {
                sc[l][c] = *reinterpret_cast<const S4<T>*>(p + col[c]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[l][c].s[i] = col[c] + i < a.out ? p[col[c] + i] : T(0.f);
            }
        }
        scale_rest += L * kStep + (last_of_unit ? a.skip_rest : 0);
        scale_row += last_of_unit ? a.skip_rows : 0;
        if (scale_rest >= a.group) scale_rest -= a.group, ++scale_row;
    };

    float acc[CH][2][NT][4];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[c][m][j][e] = 0.f;

    const Unpack weight;
    uint32_t issued = 0, done = 0;  // units of this group
    for (int u = first; issued < kStages; u += stride) {
        if (u < units) copy_unit(u, issued);
        if (VEC && u >= units) break;
        if constexpr (!VEC) copies_commit();
        ++issued;
    }
    if (first < units) {
#pragma unroll
        for (int l = 0; l < kPass / L; ++l) load_scales(l, (l + 1) * L == kUnit);
    }
    for (int u = first; u < units; u += stride) {
        const int i = done % kStages;
        if constexpr (VEC) {
            if (!ptx::mbar_wait(full(i), done / kStages & 1, abort_flag, a.status, 50)) break;
        } else {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
            __syncwarp();
        }
        ++done;
        const unsigned char* ws = stages + i * lay.stage + CH * sub * kBox + t * 128;
        const unsigned char* xs = stages + i * lay.stage + lay.w_bytes + g * 128;
        float d[CH][2][NT][4];
#pragma unroll 1
        for (int pass = 0; pass < kUnit / kPass; ++pass, ws += kPass * 4 * 128, xs += kPass * kStep / kBoxK * R * 128)
#pragma unroll
            for (int l = 0; l < kPass; ++l) {
                if (l % L == 0) {
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e) d[c][m][j][e] = 0.f;
                }
                uint32_t b[NT][PARTS][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    X8<T> x;
                    x.load(xs + 8 * j * 128 + (l * kStep / kBoxK) * R * 128,
                           (l * kStep % kBoxK + 8 * t) * sizeof(T) / 16, g);
                    x.words(b[j]);
                }
                uint32_t q[CH][4];
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const uint4 w = *reinterpret_cast<const uint4*>(
                        ws + c * kBox + 4 * l * 128 + 16 * (column_of(g) / 4 ^ (4 * (l & 1) + t)));
                    q[c][0] = w.x, q[c][1] = w.y, q[c][2] = w.z, q[c][3] = w.w;
                }
                // All tiles' products of two nibble pairs before the next two: they do not wait for each other.
#pragma unroll
                for (int p = 0; p < 4; p += 2)
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const uint32_t a0 = weight(q[c][2 * m], p), a1 = weight(q[c][2 * m + 1], p);
                            const uint32_t a2 = weight(q[c][2 * m], p + 1), a3 = weight(q[c][2 * m + 1], p + 1);
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int k = PARTS - 1; k >= 0; --k)
                                    mma_bf16(d[c][m][j], a0, a1, a2, a3, b[j][k][p], b[j][k][p + 1]);
                        }
                if (l % L == L - 1) {
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        const S4<T> s = sc[l / L][c];
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    acc[c][m][j][e] = fmaf((float)s.s[2 * m + (e >> 1)], d[c][m][j][e], acc[c][m][j][e]);
                    }
                    // Those of the next pass; past the last unit they are of no use. The unit's last ones are
                    // loaded in its last pass but one.
                    load_scales(l / L, l == kPass - 1 && pass == (kUnit / kPass == 1 ? 0 : kUnit / kPass - 2));
                }
            }
        __syncwarp();  // all lanes have read the stage
        if constexpr (VEC) {
            if (lane == 0) ptx::mbar_arrive(empty(i));
            const int next = u + kStages * stride;
            if (next < units) {
                // A warp's words are its own; x goes over what the group's other warps have to have read.
                if (sub == 0 && !ptx::mbar_wait(empty(i), (issued / kStages - 1) & 1, abort_flag, a.status, 51)) break;
                copy_unit(next, i);
                ++issued;
            }
        } else {
            if (u + kStages * stride < units) copy_unit(u + kStages * stride, i);
            copies_commit();
        }
    }
    if constexpr (VEC)  // after an expired wait alone: no copy outlives the stages
        for (; done < issued; ++done) ptx::mbar_wait_drain(full(done % kStages), done / kStages & 1);
    __syncthreads();  // the stages are free: the groups' sums take their place
    float* sums = reinterpret_cast<float*>(smem);
    const int pitch = C + 4;
    // acc[c][m][j][e]: column 32 c + column_of(g) + 2 m + e / 2 of the warp's, row 8 j + 2 t + e % 2
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                *reinterpret_cast<float4*>(
                    &sums[(group * R + 8 * j + 2 * t + e) * pitch + 32 * (CH * sub + c) + column_of(g)]) =
                    make_float4(acc[c][0][j][e], acc[c][0][j][e + 2], acc[c][1][j][e], acc[c][1][j][e + 2]);
    if (ks > 1) cluster_wait();
    __syncthreads();
    // Four results at a time: quad q of the tile, row by row, is in block q / 64, which CTA block % ks
    // finishes: it receives its blocks from all CTAs of the cluster.
    float4* recv = reinterpret_cast<float4*>(smem + lay.recv);
    const int quads = (rows << c_log) / 4, mine = (((quads + 63) / 64 + ks - 1) >> ks_log) * 64;  // that a CTA finishes
    for (int q = threadIdx.x; q < quads; q += kThreads) {
        const int r = (4 * q) >> c_log, n = (4 * q) & (C - 1), block = q / 64;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < groups; ++k) {
            const float4 u = *reinterpret_cast<const float4*>(&sums[(k * R + r) * pitch + n]);
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        float4* to = &recv[rank * mine + (block >> ks_log) * 64 + q % 64];
        if (ks > 1)
            *cluster.map_shared_rank(to, block & (ks - 1)) = v;
        else
            *to = v;
    }
    if (ks > 1) {
        cluster_arrive();
        cluster_wait();
    }
    for (int i = threadIdx.x; i < mine; i += kThreads) {  // without a cluster: what this thread wrote
        const int q = (((i / 64) << ks_log) + rank) * 64 + i % 64, r = (4 * q) >> c_log, n = n0 + ((4 * q) & (C - 1));
        if (q >= quads || n >= a.out) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < ks; ++k) {
            const float4 u = recv[k * mine + i];
            v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
        }
        const int64_t to = (int64_t)(r0 + r) * a.out + n;
        S4<T> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!VEC && n + e >= a.out) break;
            v[e] *= kWeightUnit;
            if (a.bias) v[e] += (float)((const T*)a.bias)[n + e];
            if (a.residual) v[e] += (float)((const T*)a.residual)[to + e];
            y.s[e] = T(v[e]);
            if (!VEC || !a.vec_y) ((T*)a.y)[to + e] = y.s[e];
        }
        if (VEC && a.vec_y) *reinterpret_cast<S4<T>*>((T*)a.y + to) = y;
    }
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

// Row-major [rows][cols], boxes of box_rows rows of box_cols (128 bytes), 128-byte swizzle; outside reads as 0.
bool row_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int rows, int cols, int eb, int box_cols,
             int box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols * eb};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int NT, int CH, int L, bool VEC>
cudaError_t launch(cudaStream_t st, int sm_count, Args a) {
    const int units = (a.in + kUnitK - 1) / kUnitK, R = 8 * NT;
    auto tiles = [&] { return (a.out + (32 * CH << a.wn_log) - 1) / (32 * CH << a.wn_log); };
    // Two warps share a unit, or none where the columns are too few to occupy the SMs (8192 x
    // 2048 in f32, 5 rows: 7.6 us against 11.0 with two).
    a.wn_log = VEC ? 1 : 0;
    if (VEC && 4 * tiles() < sm_count) a.wn_log = 0;
    const int groups = kWarps >> a.wn_log, bytes = Layout(R, CH, 1 << a.wn_log, sizeof(T)).total;
    auto kernel = linear_w4_kernel<T, NT, CH, L, VEC>;
    // The kernel may have what its larger form needs, whichever comes first: then it does not matter in which
    // order threads get here.
    const int most = std::max(Layout(R, CH, 1, sizeof(T)).total, Layout(R, CH, 2, sizeof(T)).total);
    static std::atomic<bool> allowed[64];  // by device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !allowed[dev].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) != cudaSuccess) return e;
        if (dev < 64) allowed[dev].store(true, std::memory_order_release);
    }
    // CTAs resident on an SM: one or two, as the form's shared memory allows.
    static std::atomic<int> known[2];
    int resident = known[a.wn_log].load(std::memory_order_relaxed);
    if (resident == 0) {
        if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kThreads, bytes)) != cudaSuccess) return e;
        known[a.wn_log].store(resident, std::memory_order_relaxed);
    }
    // k is split as long as all CTAs are resident at once and every group keeps two units (8192 x 8192, 16
    // rows, two an SM: 16.8 us at 128 CTAs, 15.5 at 256, 19.5 at 512; 16384 x 2048, 16 rows, one an SM: 9.8 us at
    // 128, 18.6 at 256; 32 rows of 8192 x 2048 8.5 and 11.4; 8192 x 8192 in f32, 16 rows: 29.6 and 33.1).
    while (a.ks_log < 3 && (int64_t)tiles() << (a.ks_log + 1) <= (int64_t)sm_count * resident && units >= 4 * groups << a.ks_log)
        ++a.ks_log;
    const int skip = ((groups << a.ks_log) - 1) * kUnitK;
    a.skip_rows = skip / a.group, a.skip_rest = skip % a.group;
    if (VEC && (!row_map(&a.w_map, CU_TENSOR_MAP_DATA_TYPE_UINT32, a.packed, (a.in + 7) / 8, a.out, 4, 32, kUnitRows) ||
                !row_map(&a.x_map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.x,
                         a.rows, a.in, sizeof(T), 128 / (int)sizeof(T), R)))
        return cudaErrorInvalidValue;
    return launch_overlapped(st, kernel, dim3((unsigned)(tiles() << a.ks_log), (unsigned)((a.rows + R - 1) / R)), kThreads,
                             (size_t)bytes, 1 << a.ks_log, a);
}

// Unaligned operands and odd widths take one form of the kernel each, the rest one by the
// steps of a unit that share a group.
template <typename T, int NT, int CH>
cudaError_t by_group(cudaStream_t st, int sm_count, const Args& a, bool vec) {
    if (!vec) return launch<T, NT, CH, 1, false>(st, sm_count, a);
    if (a.group % 128 == 0) return launch<T, NT, CH, 4, true>(st, sm_count, a);
    if (a.group % 64 == 0) return launch<T, NT, CH, 2, true>(st, sm_count, a);
    return launch<T, NT, CH, 1, true>(st, sm_count, a);
}

// Up to 16 rows a warp takes 64 columns, which halves the reads of x; 32 rows
// fit the registers with 32 columns, and only in bf16.
template <typename T>
cudaError_t by_rows(cudaStream_t st, int sm_count, const Args& a, bool vec) {
    if (a.rows <= 8) return by_group<T, 1, 2>(st, sm_count, a, vec);
    if constexpr (sizeof(T) == 4) {
        return by_group<T, 2, 2>(st, sm_count, a, vec);
    } else {
        if (a.rows <= 16) return by_group<T, 2, 2>(st, sm_count, a, vec);
        return by_group<T, 4, 1>(st, sm_count, a, vec);
    }
}

}  // namespace

cudaError_t linear_w4(cudaStream_t st, int sm_count, DeviceStatus* status, hx_dtype dt, const void* x, const uint32_t* packed,
                      const void* scales, const void* bias, const void* residual, void* y, int rows, int in, int out,
                      int group) {
    Args a{CUtensorMap{}, CUtensorMap{}, x, packed, scales, bias, residual, y, status, rows, in, out, group,
                 (in + group - 1) / group, 0, 0,
           (uintptr_t)y % (dt == HX_F32 ? 16 : 8) == 0, 0, 0};
    const bool vec = (uintptr_t)x % 16 == 0 && (int64_t)in * (dt == HX_F32 ? 4 : 2) % 16 == 0 && (uintptr_t)packed % 16 == 0 && (uintptr_t)scales % 16 == 0 && out % 4 == 0;
    return dt == HX_F32 ? by_rows<float>(st, sm_count, a, vec) : by_rows<__nv_bfloat16>(st, sm_count, a, vec);
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
