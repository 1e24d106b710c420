// Forward products of few rows (tokens of one decode step): bound by reading the weight once
// and by latency, not by arithmetic.
//
// 16-bit: the weight is the 16-row operand of mma.sync.m16n8k16 and the tokens its 8 columns,
// so up to 64 tokens ride on one pass over the weight.  A CTA owns 16 output features (16
// pairs of the gated block); its 8 warps take the contraction in blocks of 32, interleaved,
// and their partial tiles are added in warp order in shared memory.  The contraction index
// may be permuted as long as both operands agree: lane (g, c) takes the 8 contiguous
// elements 8 c .. 8 c + 7 of a block, one 16-byte load per row, and feeds them as the pairs
// (2c, 2c+1), (2c+8, 2c+9) of two products, so fragments come straight from global memory.
//
// float32: a warp owns two features (or a pair) of up to 8 tokens, lanes along the
// contraction, four elements per lane and step.
//
// Both read any strides (element by element where rows are not 16-byte aligned).
//
// On the device, bf16: one token through 640 -> 2 x 1248 3.3 us, through 1248 -> 640 3.6 us (3.2 MB
// and 1.6 MB of weights: a quarter of the time is their bytes, the rest one chain of loads, the
// exchange and the launch); 48 tokens through 640 -> 1544 5.4 us, where a tile of the tensor-core
// kernel (128 rows, its set-up and its pipeline's fill) takes 7.
#include "dense.cuh"
#include "mma_util.cuh"

#include <type_traits>

namespace maba {
namespace dense {
namespace {

constexpr int NWARP = 8, NTHR = 32 * NWARP, ROWS = 16;

// The epilogue of one element; z1 is the up projection of the gated block.
template <typename T> __device__ __forceinline__ void finish(const Epilogue& e, int64_t m, int64_t n, float z, float z1) {
    if (e.kind == E_GLU) {
        z = act_f(z, e.act) * z1;
    } else {
        if (e.bias.p) z += side_at<T>(e.bias, 0, n);
        z = act_f(z, e.act);
        if (e.scale.p) z *= side_at<T>(e.scale, 0, n);
        if (e.res.p) z += side_at<T>(e.res, m, n);
    }
    if (e.out_f32) static_cast<float*>(e.out)[m * e.ldo + n] = z;
    else static_cast<T*>(e.out)[m * e.ldo + n] = Cvt<T>::from_f(z);
}

// 8 consecutive contraction elements of one row, zeros outside
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load8(const Matrix& a, int64_t r, int64_t rows, int64_t k, int64_t K) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r >= rows || k >= K) return v;
    const uint16_t* p = static_cast<const uint16_t*>(a.p) + r * a.sr + k * a.sk;
    if (VEC) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < K) w[e >> 1] |= (uint32_t)p[e * a.sk] << (16 * (e & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int NT, bool DUAL, bool VEC>
__global__ void __launch_bounds__(NTHR) skinny_kernel(const Product p) {
    constexpr int NB = DUAL ? 2 : 1, LD = 8 * NT + 1, U = NT * NB <= 4 ? 4 : 2;
    extern __shared__ float red[];  // [NB][8 warps][16 features][tokens]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int64_t n0 = (int64_t)blockIdx.x * ROWS;
    const int64_t nblk = (p.K + 31) / 32;
    float acc[NB][NT][4] = {};
    for (int64_t b0 = warp; b0 < nblk; b0 += NWARP * U) {
        uint4 wl[U][NB], wh[U][NB], xv[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = (b0 + u * NWARP) * 32 + c * 8;
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                wl[u][q] = load8<T, VEC>(p.b[q], n0 + g, p.N, k, p.K);
                wh[u][q] = load8<T, VEC>(p.b[q], n0 + g + 8, p.N, k, p.K);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) xv[u][t] = load8<T, VEC>(p.a[0], t * 8 + g, p.M, k, p.K);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const uint32_t a0[4] = {wl[u][q].x, wh[u][q].x, wl[u][q].y, wh[u][q].y};
                const uint32_t a1[4] = {wl[u][q].z, wh[u][q].z, wl[u][q].w, wh[u][q].w};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    Mma16<T>::mma(acc[q][t], a0, xv[u][t].x, xv[u][t].y);
                    Mma16<T>::mma(acc[q][t], a1, xv[u][t].z, xv[u][t].w);
                }
            }
    }
#pragma unroll
    for (int q = 0; q < NB; ++q)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                red[((q * NWARP + warp) * ROWS + g + (i >> 1) * 8) * LD + t * 8 + 2 * c + (i & 1)] = acc[q][t][i];
    __syncthreads();
    for (int o = tid; o < ROWS * 8 * NT; o += NTHR) {
        const int r = o & (ROWS - 1), m = o / ROWS;
        if (m >= p.M || n0 + r >= p.N) continue;
        float z[2] = {0.f, 0.f};
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int w = 0; w < NWARP; ++w) z[q] += red[((q * NWARP + w) * ROWS + r) * LD + m];
        finish<T>(p.e, m, n0 + r, z[0], z[1]);
    }
}

// four contraction elements of a float32 row, zeros outside
template <bool VEC> __device__ __forceinline__ float4 load4(const Matrix& a, int64_t r, int64_t rows, int64_t k, int64_t K) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < rows && k < K) {
        const float* p = static_cast<const float*>(a.p) + r * a.sr + k * a.sk;
        if (VEC) return *reinterpret_cast<const float4*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + e < K) v[e] = p[e * a.sk];
    }
    return make_float4(v[0], v[1], v[2], v[3]);
}

template <int MT, bool DUAL, bool VEC> __global__ void __launch_bounds__(NTHR) skinny32_kernel(const Product p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n = ((int64_t)blockIdx.x * NWARP + warp) * (DUAL ? 1 : 2);
    if (n >= p.N) return;
    constexpr int U = MT <= 2 ? 4 : 2;
    float acc[2][MT] = {};
    for (int64_t k0 = lane * 4; k0 < p.K; k0 += 128 * U) {
        float4 w[U][2], x[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = k0 + u * 128;
            w[u][0] = load4<VEC>(p.b[0], n, p.N, k, p.K);
            w[u][1] = DUAL ? load4<VEC>(p.b[1], n, p.N, k, p.K) : load4<VEC>(p.b[0], n + 1, p.N, k, p.K);
#pragma unroll
            for (int m = 0; m < MT; ++m) x[u][m] = load4<VEC>(p.a[0], m, p.M, k, p.K);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    acc[q][m] = fmaf(w[u][q].x, x[u][m].x, acc[q][m]);
                    acc[q][m] = fmaf(w[u][q].y, x[u][m].y, acc[q][m]);
                    acc[q][m] = fmaf(w[u][q].z, x[u][m].z, acc[q][m]);
                    acc[q][m] = fmaf(w[u][q].w, x[u][m].w, acc[q][m]);
                }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc[q][m] += __shfl_xor_sync(0xffffffffu, acc[q][m], o);
    // every lane holds every sum; lane m (and 8 + m for the second feature) finishes its own
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (m >= p.M) break;
        if (lane == m) finish<float>(p.e, m, n, acc[0][m], acc[1][m]);
        if (!DUAL && lane == 8 + m && n + 1 < p.N) finish<float>(p.e, m, n + 1, acc[1][m], 0.f);
    }
}

// every row of the operand starts on a 16-byte boundary and holds whole 16-byte pieces
bool pieces(const Matrix& a, int64_t rows, int64_t K, int el) {
    const int per = 16 / el;
    return a.sk == 1 && K % per == 0 && (rows == 1 || a.sr % per == 0) && (reinterpret_cast<uintptr_t>(a.p) & 15u) == 0;
}

template <typename T, int NT, bool DUAL> int launch16(const Product& p, bool vec, cudaStream_t s) {
    const size_t smem = (size_t)(DUAL ? 2 : 1) * NWARP * ROWS * (8 * NT + 1) * sizeof(float);
    const auto kern = vec ? skinny_kernel<T, NT, DUAL, true> : skinny_kernel<T, NT, DUAL, false>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return set_error(MABA_ERR_CUDA, "dense(few rows): %s", cudaGetErrorString(e));
    }
    kern<<<(unsigned)ceil_div(p.N, ROWS), NTHR, smem, s>>>(p);
    return check_launch("dense(few rows)");
}
template <typename T, bool DUAL> int by_rows16(const Product& p, bool vec, cudaStream_t s) {
    if (p.M <= 8) return launch16<T, 1, DUAL>(p, vec, s);
    if (p.M <= 16) return launch16<T, 2, DUAL>(p, vec, s);
    if (p.M <= 32) return launch16<T, 4, DUAL>(p, vec, s);
    return launch16<T, 8, DUAL>(p, vec, s);
}
template <int MT, bool DUAL> int launch32(const Product& p, bool vec, cudaStream_t s) {
    const unsigned grid = (unsigned)ceil_div(p.N, NWARP * (DUAL ? 1 : 2));
    if (vec) skinny32_kernel<MT, DUAL, true><<<grid, NTHR, 0, s>>>(p);
    else skinny32_kernel<MT, DUAL, false><<<grid, NTHR, 0, s>>>(p);
    return check_launch("dense(few rows)");
}
template <bool DUAL> int by_rows32(const Product& p, bool vec, cudaStream_t s) {
    if (p.M == 1) return launch32<1, DUAL>(p, vec, s);
    if (p.M == 2) return launch32<2, DUAL>(p, vec, s);
    if (p.M <= 4) return launch32<4, DUAL>(p, vec, s);
    return launch32<8, DUAL>(p, vec, s);
}

}  // namespace

bool skinny_takes(const Product& p, int dt) {
    return (p.e.kind == E_LINEAR || p.e.kind == E_GLU) && p.M <= (dt == MABA_F32 ? 8 : 64);
}

template <typename T> int skinny_product(const Product& p, cudaStream_t s) {
    const bool dual = p.form == F_DUAL;
    bool vec = pieces(p.a[0], p.M, p.K, sizeof(T)) && pieces(p.b[0], p.N, p.K, sizeof(T));
    if (dual) vec = vec && pieces(p.b[1], p.N, p.K, sizeof(T));
    if constexpr (sizeof(T) == 4) return dual ? by_rows32<true>(p, vec, s) : by_rows32<false>(p, vec, s);
    else return dual ? by_rows16<T, true>(p, vec, s) : by_rows16<T, false>(p, vec, s);
}
template int skinny_product<float>(const Product&, cudaStream_t);
template int skinny_product<__half>(const Product&, cudaStream_t);
template int skinny_product<__nv_bfloat16>(const Product&, cudaStream_t);

}  // namespace dense
}  // namespace maba
