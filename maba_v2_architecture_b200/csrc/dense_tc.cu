// Products of 16-bit operands on the 5th-generation tensor cores (tcgen05, TMEM, TMA).
//
// Persistent, one CTA per SM.  A work unit is a tile of C (128 rows of A by bn rows of B;
// with CG = 2 a cluster's two CTAs share a tile of 256 rows: each loads its own 128 rows of
// A and one half of B, so a k-block costs an SM 32 KB for 128 x 256 x 64 products instead
// of 48 KB, below what L2 delivers per SM) over one split of the contraction.  Ten warps:
//  * 0..7   epilogue: warp w reads TMEM lanes 32 (w & 3).. and every second 32-column
//           chunk, applies the epilogue and stores whole rows' segments, staged through
//           shared memory so that global accesses run along the rows;
//  * 8      TMA producer: 64 contraction indices per stage, 128-byte swizzle, operands
//           K-major or (for the transposed products of the backward pass) MN-major;
//  * 9      allocates TMEM and issues the products.
// The float32 accumulator is double-buffered in TMEM (2 x 256 columns): a unit's epilogue
// runs under the next unit's products.  The gated block's tile holds bn/2 rows of w_gate and
// bn/2 of w_up, so a thread sees both projections of an element in its own row.
//
// Every mbarrier wait is bounded; a wait that runs out raises the CTA's abort flag, all
// roles leave their loops, copies and products in flight are drained (bounded), TMEM is
// freed and the error word behind maba_device_error() is set.
#include "activations.cuh"
#include "dense.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

#include <type_traits>

namespace maba {
namespace dense {

__device__ int g_dense_error = 0;

namespace {
using namespace tc;

constexpr int NTHR = 320, EPI_WARPS = 8, W_TMA = 8, W_MMA = 9;
constexpr int BK = 64;
constexpr uint32_t A_BYTES = 128 * BK * 2;
constexpr int MAX_STAGES = 8;
constexpr uint32_t STAGING = 32 * 128;  // one warp's 32 x 32 float32 chunk
constexpr uint32_t TAIL = EPI_WARPS * STAGING + EPI_WARPS * 2 * 32 * 4 + 256;
constexpr uint32_t SMEM_MAX = 227 * 1024;
constexpr int TMEM_COLS = 512, ACC_COLS = 256;

enum { B_FULL = 0, B_EMPTY = MAX_STAGES, B_TFULL = 2 * MAX_STAGES, B_TEMPTY = B_TFULL + 2, B_DRAIN = B_TEMPTY + 2, N_BARS };
static_assert(N_BARS * 8 + 8 <= 256, "barrier area");

struct TcArgs {
    int64_t M, N;
    int kblocks, kseg;  // contraction blocks over all segments, and of one
    int tiles_n, splits, pairs, units, dual;
    int bn, b_rows;  // columns of the MMA, rows of B per CTA
    int stages;
    uint32_t stage_bytes, load_bytes;  // load_bytes: what one stage's barrier receives
    uint32_t idesc;
    int side_vec, out_vec;
    Epilogue e;
    float* partial;
    int64_t ldp;
};

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// phi and phi' on the SFU's exponential and reciprocal: a few float32 ulp, and the results
// are rounded to 16 bits or come from sums of 16-bit products.
template <int ACT> __device__ __forceinline__ float act16(float z) {
    if (ACT == ACT_SILU) return silu_f(z);
    return act_f(z, ACT);
}
template <int ACT> __device__ __forceinline__ void act_grad16(float z, float& y, float& d) {
    if (ACT == ACT_SILU) {
        const float s = sigmoid_f(z);
        y = z * s;
        d = s * (1.f + z * (1.f - s));
    } else {
        act_grad_f(z, ACT, y, d);
    }
}
template <typename F> __device__ __forceinline__ void with_act(int act, F f) {
    if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>());
    else if (act == ACT_GELU) f(std::integral_constant<int, ACT_GELU>());
    else if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>());
    else f(std::integral_constant<int, ACT_NONE>());
}

// --------------------------------------------------------------------------
// 32 x 32 chunks between global memory (a warp's lanes along the rows) and registers (lane
// = row), through the warp's staging area; 16-byte pieces are swizzled so that both
// directions are free of bank conflicts.
// --------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void fetch_chunk(uint4* v, const Side& s, bool vec, int64_t row0, int64_t col0, int64_t M,
                                            int64_t N, int lane) {
    if (s.f32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = row0 + i * 4 + (lane >> 3), c = col0 + (lane & 7) * 4;
            float t[4] = {0.f, 0.f, 0.f, 0.f};
            const float* p = static_cast<const float*>(s.p) + r * s.sr + c * s.sc;
            if (r < M) {
                if (vec && c + 4 <= N) *reinterpret_cast<float4*>(t) = *reinterpret_cast<const float4*>(p);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < N) t[e] = p[e * s.sc];
            }
            v[i] = *reinterpret_cast<uint4*>(t);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = row0 + i * 8 + (lane >> 2), c = col0 + (lane & 3) * 8;
            uint32_t t[4] = {0u, 0u, 0u, 0u};
            const uint16_t* p = static_cast<const uint16_t*>(s.p) + r * s.sr + c * s.sc;
            if (r < M) {
                if (vec && c + 8 <= N) *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c + e < N) t[e >> 1] |= (uint32_t)p[e * s.sc] << (16 * (e & 1));
            }
            v[i] = *reinterpret_cast<uint4*>(t);
        }
    }
}
__device__ __forceinline__ uint4* at32(unsigned char* st, int row, int piece) {
    return reinterpret_cast<uint4*>(st + row * 128 + ((piece ^ (row & 7)) << 4));
}
__device__ __forceinline__ uint4* at16(unsigned char* st, int row, int piece) {
    return reinterpret_cast<uint4*>(st + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}
template <typename T>
__device__ __forceinline__ void chunk_to_rows(float* x, const uint4* v, bool f32, unsigned char* st, int lane) {
    __syncwarp();
    if (f32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) *at32(st, i * 4 + (lane >> 3), lane & 7) = v[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(x + 4 * i) = *at32(st, lane, i);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) *at16(st, i * 8 + (lane >> 2), lane & 3) = v[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 q = *at16(st, lane, i);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<T>(w[e]);
                x[8 * i + 2 * e] = f.x, x[8 * i + 2 * e + 1] = f.y;
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void store_rows(const float* x, void* out, bool f32, int64_t ld, bool vec, int64_t row0,
                                           int64_t col0, int64_t M, int64_t N, unsigned char* st, int lane) {
    __syncwarp();
    if (f32) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4*>(at32(st, lane, i)) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = row0 + i * 4 + (lane >> 3), c = col0 + (lane & 7) * 4;
            const uint4 q = *at32(st, i * 4 + (lane >> 3), lane & 7);
            if (r >= M) continue;
            float* p = static_cast<float*>(out) + r * ld + c;
            if (vec && c + 4 <= N) *reinterpret_cast<uint4*>(p) = q;
            else {
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < N) p[e] = __uint_as_float(w[e]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *at16(st, lane, i) = make_uint4(pack2<T>(x[8 * i], x[8 * i + 1]), pack2<T>(x[8 * i + 2], x[8 * i + 3]),
                                            pack2<T>(x[8 * i + 4], x[8 * i + 5]), pack2<T>(x[8 * i + 6], x[8 * i + 7]));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = row0 + i * 8 + (lane >> 2), c = col0 + (lane & 3) * 8;
            const uint4 q = *at16(st, i * 8 + (lane >> 2), lane & 3);
            if (r >= M) continue;
            uint16_t* p = static_cast<uint16_t*>(out) + r * ld + c;
            if (vec && c + 8 <= N) *reinterpret_cast<uint4*>(p) = q;
            else {
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < N) p[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            }
        }
    }
}
// Sums of 32 columns over the warp's 32 rows, in a fixed tree; lane l returns column l's.
__device__ __forceinline__ float column_sum(float* v, int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const bool hi = (lane & o) != 0;
#pragma unroll
        for (int j = 0; j < o; ++j) {
            const float keep = hi ? v[j + o] : v[j], give = hi ? v[j] : v[j + o];
            v[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    return v[0];
}

template <typename T, int CG, bool A_MN, bool B_MN, int KIND>
__global__ void __launch_bounds__(NTHR, 1)
    tc_kernel(const TcArgs a, const __grid_constant__ CUtensorMap ta0, const __grid_constant__ CUtensorMap ta1,
              const __grid_constant__ CUtensorMap tb0, const __grid_constant__ CUtensorMap tb1) {
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    unsigned char* tail = base + a.stages * a.stage_bytes;
    float* vecs = reinterpret_cast<float*>(tail + EPI_WARPS * STAGING);  // [8 warps][scale, bias][32]
    uint64_t* bars = reinterpret_cast<uint64_t*>(tail + EPI_WARPS * STAGING + EPI_WARPS * 2 * 32 * 4);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + N_BARS);
    volatile int* abort_f = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
    const int worker = blockIdx.x / CG, workers = gridDim.x / CG;

    if (tid == 0) {
        for (int i = 0; i < N_BARS; ++i) mbar_init(&bars[i], i == B_TEMPTY || i == B_TEMPTY + 1 ? EPI_WARPS * CG : 1);
        *abort_f = 0;
        fence_barrier_init();
    }
    if (warp == W_TMA && lane == 0) {
        prefetch_tmap(&ta0);
        prefetch_tmap(&tb0);
    }
    if (warp == W_MMA) {
        if (CG == 2) tmem_alloc_pair<TMEM_COLS>(tmem_slot);
        else tmem_alloc<TMEM_COLS>(tmem_slot);
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // a unit: splits innermost, then the pair index, then columns, then rows of tiles
    struct Unit {
        int split, pair, kb0, kb1;
        int64_t m0, n0;
    };
    auto unit_of = [&](int u) {
        Unit t;
        t.split = u % a.splits;
        u /= a.splits;
        t.pair = u % a.pairs;
        u /= a.pairs;
        t.n0 = (int64_t)(u % a.tiles_n) * (a.dual ? a.bn / 2 : a.bn);
        t.m0 = (int64_t)(u / a.tiles_n) * (128 * CG) + rank * 128;
        t.kb0 = (int)((int64_t)a.kblocks * t.split / a.splits);
        t.kb1 = (int)((int64_t)a.kblocks * (t.split + 1) / a.splits);
        return t;
    };

    if (warp == W_TMA) {
        // ============================ TMA producer ============================
        int it = 0;
        bool ok = true;
        for (int u = worker; u < a.units && ok; u += workers) {
            const Unit t = unit_of(u);
            for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                const int st = it % a.stages, round = it / a.stages;
                if (round > 0) ok = mbar_wait_warp(&bars[B_EMPTY + st], (round - 1) & 1, abort_f);
                if (!ok) break;
                const int seg = kb >= a.kseg ? 1 : 0, k0 = (kb - seg * a.kseg) * BK;
                const CUtensorMap* ma = (a.pairs == 2 ? t.pair : seg) ? &ta1 : &ta0;
                unsigned char* sa = base + st * a.stage_bytes;
                unsigned char* sb = sa + A_BYTES;
                if (elect_one()) {
                    uint64_t* full = &bars[B_FULL + st];
                    const uint32_t full0 = CG == 2 ? cluster_addr(full, 0) : 0u;
                    auto load = [&](unsigned char* dst, const CUtensorMap* m, int x, int y) {
                        if (CG == 2) tma_load_2d_pair(dst, m, full0, x, y);
                        else tma_load_2d(dst, m, full, x, y);
                    };
                    if (rank == 0) mbar_arrive_expect_tx(full, a.load_bytes);
                    if (A_MN) {
                        load(sa, ma, (int)t.m0, k0);
                        load(sa + A_BYTES / 2, ma, (int)t.m0 + 64, k0);
                    } else {
                        load(sa, ma, k0, (int)t.m0);
                    }
                    if (KIND == E_GLU || KIND == E_GLU_BWD) {
                        if (CG == 2) {
                            load(sb, rank ? &tb1 : &tb0, k0, (int)t.n0);
                        } else {
                            load(sb, &tb0, k0, (int)t.n0);
                            load(sb + a.bn / 2 * 128, &tb1, k0, (int)t.n0);
                        }
                    } else {
                        const CUtensorMap* mb = seg ? &tb1 : &tb0;
                        const int y = (int)t.n0 + (int)rank * a.b_rows;
                        if (B_MN) {
                            for (int i = 0; i < a.b_rows; i += 64) load(sb + i * 128, mb, y + i, k0);
                        } else {
                            load(sb, mb, k0, y);
                        }
                    }
                }
                __syncwarp();
            }
        }
        // every copy has landed before a CTA may exit (rank 0's barriers count the pair's)
        if (rank == 0)
            for (int s = 0; s < a.stages && s < it; ++s)
                mbar_wait_warp(&bars[B_FULL + s], (((it - 1 - s) / a.stages)) & 1, nullptr);
    } else if (warp == W_MMA) {
        // ============================ MMA issuer ==============================
        if (rank == 0) {
            const uint64_t ad0 = sdesc_sw128(smem_addr(base), A_MN ? A_BYTES / 2 : 16, 1024);
            const uint64_t bd0 = sdesc_sw128(smem_addr(base + A_BYTES), B_MN ? 8192 : 16, 1024);
            constexpr uint32_t ak = A_MN ? 2048 >> 4 : 32 >> 4, bk = B_MN ? 2048 >> 4 : 32 >> 4;
            int it = 0, i = 0;
            bool ok = true;
            for (int u = worker; u < a.units && ok; u += workers, ++i) {
                const Unit t = unit_of(u);
                const int buf = i & 1;
                if (i >= 2) ok = mbar_wait_warp(&bars[B_TEMPTY + buf], ((i >> 1) - 1) & 1, abort_f);
                if (!ok) break;
                tc_fence_after();
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                    const int st = it % a.stages;
                    ok = mbar_wait_warp(&bars[B_FULL + st], (it / a.stages) & 1, abort_f);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t so = (uint64_t)(st * (a.stage_bytes >> 4));
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k) {
                        const uint32_t acc = kb > t.kb0 || k > 0 ? 1u : 0u;
                        if (CG == 2)
                            umma_f16_ss_pair_elect(tmem + buf * ACC_COLS, ad0 + so + k * ak, bd0 + so + k * bk, a.idesc, acc);
                        else
                            umma_f16_ss_elect(tmem + buf * ACC_COLS, ad0 + so + k * ak, bd0 + so + k * bk, a.idesc, acc);
                    }
                    if (CG == 2) umma_commit_pair_elect(&bars[B_EMPTY + st]);
                    else umma_commit_elect(&bars[B_EMPTY + st]);
                }
                if (!ok) break;
                if (CG == 2) umma_commit_pair_elect(&bars[B_TFULL + buf]);
                else umma_commit_elect(&bars[B_TFULL + buf]);
            }
            // every product has completed before TMEM is freed
            if (CG == 2) umma_commit_pair_elect(&bars[B_DRAIN]);
            else umma_commit_elect(&bars[B_DRAIN]);
            mbar_wait_warp(&bars[B_DRAIN], 0, nullptr);
        }
    } else {
        // ============================== epilogue ==============================
        constexpr bool DUAL = KIND == E_GLU || KIND == E_GLU_BWD;
        const int q = warp & 3, h = warp >> 2;
        unsigned char* st = tail + warp * STAGING;
        float* vscale = vecs + warp * 64;
        float* vbias = vscale + 32;
        const Epilogue& e = a.e;
        const int width = DUAL ? a.bn / 2 : a.bn;
        const bool has_side = KIND != E_STORE && KIND != E_GLU && e.res.p != nullptr;
        int i = 0;
        for (int u = worker; u < a.units; u += workers, ++i) {
            const Unit t = unit_of(u);
            const int buf = i & 1;
            const int64_t row0 = t.m0 + q * 32;
            const bool live = row0 < a.M;
            uint4 side[8];
            float ps = 0.f, pb = 0.f;  // this lane's column of scale and bias
            auto fetch = [&](int c) {
                const int64_t col0 = t.n0 + c * 32;
                if (has_side) fetch_chunk<T>(side, e.res, a.side_vec, row0, col0, a.M, a.N, lane);
                if (KIND == E_LINEAR || KIND == E_LINEAR_BWD) {
                    const bool in = col0 + lane < a.N;
                    ps = in && e.scale.p ? side_at<T>(e.scale, 0, col0 + lane) : 1.f;
                    pb = in && e.bias.p ? side_at<T>(e.bias, 0, col0 + lane) : 0.f;
                }
            };
            if (live && h * 32 < width) fetch(h);
            if (!mbar_wait_warp(&bars[B_TFULL + buf], (i >> 1) & 1, abort_f)) break;
            tc_fence_after();
            const uint32_t acc = tmem + buf * ACC_COLS + ((uint32_t)(q * 32) << 16);
            for (int c = h; c * 32 < width; c += 2) {
                const int64_t col0 = t.n0 + c * 32;
                float z[32], w[DUAL ? 32 : 1];
                tmem_ld32(acc + c * 32, reinterpret_cast<uint32_t*>(z));
                if (DUAL) tmem_ld32(acc + width + c * 32, reinterpret_cast<uint32_t*>(w));
                tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(z));
                if (DUAL) tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(w));
                if (!live || col0 >= a.N) continue;
                float g[32];
                if (has_side) chunk_to_rows<T>(g, side, e.res.f32, st, lane);
                if (KIND == E_LINEAR || KIND == E_LINEAR_BWD) {
                    __syncwarp();
                    vscale[lane] = ps;
                    vbias[lane] = pb;
                    __syncwarp();
                }
                if ((c + 2) * 32 < width) fetch(c + 2);
                if (KIND == E_STORE) {
                    const int64_t rows = a.pairs * a.M;
                    if (a.splits > 1)
                        store_rows<T>(z, a.partial + ((int64_t)t.split * rows + t.pair * a.M) * a.ldp, true, a.ldp, true, row0,
                                      col0, a.M, a.N, st, lane);
                    else
                        store_rows<T>(z, t.pair ? e.out2 : e.out, false, e.ldo, a.out_vec, row0, col0, a.M, a.N, st, lane);
                } else if (KIND == E_LINEAR) {
                    with_act(e.act, [&](auto A) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            z[j] = act16<A.value>(z[j] + vbias[j]) * vscale[j];
                            if (has_side) z[j] += g[j];
                        }
                    });
                    store_rows<T>(z, e.out, e.out_f32, e.ldo, a.out_vec, row0, col0, a.M, a.N, st, lane);
                } else if (KIND == E_LINEAR_BWD) {
                    float y[32];
                    const bool in = row0 + lane < a.M;  // rows past the last: no part in the sums
                    with_act(e.act, [&](auto A) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            float f, d;
                            act_grad16<A.value>(z[j] + vbias[j], f, d);
                            z[j] = in ? g[j] * vscale[j] * d : 0.f;
                            y[j] = in ? g[j] * f : 0.f;
                        }
                    });
                    store_rows<T>(z, e.out, false, e.ldo, a.out_vec, row0, col0, a.M, a.N, st, lane);
                    const int64_t at = (row0 >> 5) * a.N + col0 + lane;
                    if (e.part_bias) {
                        const float s = column_sum(z, lane);
                        if (col0 + lane < a.N) e.part_bias[at] = s;
                    }
                    if (e.part_scale) {
                        const float s = column_sum(y, lane);
                        if (col0 + lane < a.N) e.part_scale[at] = s;
                    }
                } else if (KIND == E_GLU) {
                    with_act(e.act, [&](auto A) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) z[j] = act16<A.value>(z[j]) * w[j];
                    });
                    store_rows<T>(z, e.out, false, e.ldo, a.out_vec, row0, col0, a.M, a.N, st, lane);
                } else {
                    with_act(e.act, [&](auto A) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            float f, d;
                            act_grad16<A.value>(z[j], f, d);
                            z[j] = g[j] * w[j] * d;
                            w[j] = g[j] * f;
                        }
                    });
                    store_rows<T>(z, e.out, false, e.ldo, a.out_vec, row0, col0, a.M, a.N, st, lane);
                    store_rows<T>(w, e.out2, false, e.ldo, a.out_vec, row0, col0, a.M, a.N, st, lane);
                }
            }
            // this warp has read its part of the accumulator
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) mbar_arrive_cluster(cluster_addr(&bars[B_TEMPTY + buf], 0));
                else mbar_arrive(&bars[B_TEMPTY + buf]);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) {
        // the last arrival that rank 0's products make on this CTA's barriers
        if (rank == 1 && warp == W_MMA) mbar_wait_warp(&bars[B_DRAIN], 0, nullptr);
        cluster_sync();
    }
    if (warp == W_MMA) {
        tc_fence_after();
        if (CG == 2) tmem_dealloc_pair<TMEM_COLS>(tmem);
        else tmem_dealloc<TMEM_COLS>(tmem);
    }
    if (tid == 0 && *abort_f) atomicExch(&g_dense_error, 1);
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------
struct Plan {
    int cg = 1, bn = 32, splits = 1;
};

inline int b_rows_of(int cg, int bn) { return bn / cg; }
inline uint32_t b_bytes_of(int cg, int bn, bool mn) {
    const int r = b_rows_of(cg, bn);
    return (uint32_t)(mn ? (r + 63) / 64 * 64 : r) * 128u;
}

// The tile and the splits with the least estimated time.  Per k-block and SM: the larger of
// the products (128 x bn x 64 at 4,096 per cycle) and the loads (60 bytes per cycle from L2);
// a unit that is not hidden under another adds its fill and epilogue.
Plan plan_of(const Product& p) {
    const bool dual = p.form == F_DUAL, store = p.e.kind == E_STORE;
    const bool b_mn = store;
    const int64_t kblocks = ceil_div(p.K, BK) * (p.form == F_SUM ? 2 : 1);
    const int64_t pairs = p.form == F_PAIR ? 2 : 1;
    Plan best;
    double least = 1e300;
    for (int cg = 1; cg <= 2; ++cg) {
        for (int bn = dual ? 64 : 32; bn <= (cg == 2 ? 256 : 192); bn += dual ? 64 : 32) {
            const int64_t tiles = ceil_div(p.M, 128 * cg) * ceil_div(p.N, dual ? bn / 2 : bn) * pairs;
            const int64_t slots = sm_count() / cg;
            const double mma = 2.0 * bn, load = (A_BYTES + b_bytes_of(cg, bn, b_mn)) / 60.0;
            const double kcost = mma > load ? mma : load;
            for (int splits = 1; splits <= (store ? 16 : 1) && splits <= kblocks; ++splits) {
                const int64_t units = tiles * splits;
                const double waves = (double)ceil_div(units, slots);
                const double kb = (double)ceil_div(kblocks, splits);
                double t = waves * kb * kcost + 2000.0 + 12.0 * bn;
                // the partial sums, written and read: bytes at ~3,500 per cycle over the GPU, and a launch
                if (splits > 1) t += 2000.0 + 8.0 * (double)splits * pairs * p.M * p.N / 3500.0;
                if (t < least) least = t, best = Plan{cg, bn, splits};
            }
        }
    }
    return best;
}

// One operand's map: rows x contraction, read K-major (contraction contiguous) or MN-major.
bool operand_map(CUtensorMap* m, int dt, const Matrix& x, int64_t rows, int64_t k, bool mn, int box_rows) {
    const int64_t dims[2] = {mn ? rows : k, mn ? k : rows};
    const int64_t outer = mn ? x.sk : x.sr;
    const int64_t stride[1] = {dims[1] > 1 ? outer : (dims[0] + 7) / 8 * 8};
    const uint32_t box[2] = {(uint32_t)BK, (uint32_t)(mn ? BK : box_rows)};
    return make_map(m, dt, x.p, 2, dims, stride, box);
}

bool aligned16(const void* p, int64_t ld, int el) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * el) % 16 == 0;
}

using Kernel = void (*)(const TcArgs, const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap);

template <typename T, int CG> Kernel kernel_of(const Product& p) {
    switch (p.e.kind) {
        case E_LINEAR: return tc_kernel<T, CG, false, false, E_LINEAR>;
        case E_LINEAR_BWD: return tc_kernel<T, CG, false, false, E_LINEAR_BWD>;
        case E_GLU: return tc_kernel<T, CG, false, false, E_GLU>;
        case E_GLU_BWD: return tc_kernel<T, CG, false, false, E_GLU_BWD>;
        default: return p.a_mn ? tc_kernel<T, CG, true, true, E_STORE> : tc_kernel<T, CG, false, true, E_STORE>;
    }
}

}  // namespace

bool tc_readable(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t col_stride) {
    if (col_stride != 1 && cols > 1) return false;
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return false;
    return rows == 1 || (ld % 8 == 0 && ld >= cols);
}

int tc_splits(const Product& p) { return plan_of(p).splits; }

template <typename T> int tc_product(const Product& p, float* partial, int64_t ldp, cudaStream_t s) {
    if (encode_fn() == nullptr) return set_error(MABA_ERR_CUDA, "dense: cuTensorMapEncodeTiled not found");
    constexpr int dt = std::is_same<T, __nv_bfloat16>::value ? MABA_BF16 : MABA_F16;
    const Plan pl = plan_of(p);
    const bool dual = p.form == F_DUAL, store = p.e.kind == E_STORE, a_mn = p.a_mn, b_mn = store;
    TcArgs a{};
    a.M = p.M, a.N = p.N;
    a.kseg = (int)ceil_div(p.K, BK);
    a.kblocks = a.kseg * (p.form == F_SUM ? 2 : 1);
    a.pairs = p.form == F_PAIR ? 2 : 1;
    a.dual = dual;
    a.splits = pl.splits;
    a.bn = pl.bn;
    a.b_rows = b_rows_of(pl.cg, pl.bn);
    a.tiles_n = (int)ceil_div(p.N, dual ? pl.bn / 2 : pl.bn);
    const int64_t units = ceil_div(p.M, 128 * pl.cg) * a.tiles_n * a.pairs * a.splits;
    if (units > 0x7fffffff) return set_error(MABA_ERR_UNSUPPORTED, "dense: %lld tiles", (long long)units);
    a.units = (int)units;
    const uint32_t bb = b_bytes_of(pl.cg, pl.bn, b_mn);
    a.stage_bytes = A_BYTES + (bb + 1023) / 1024 * 1024;
    a.load_bytes = (A_BYTES + bb) * pl.cg;
    const uint32_t room = SMEM_MAX - 1024 - TAIL;
    a.stages = (int)(room / a.stage_bytes);
    if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
    const size_t smem = 1024 + (size_t)a.stages * a.stage_bytes + TAIL;
    a.idesc = idesc_f16(128 * pl.cg, pl.bn, dt == MABA_BF16, a_mn, b_mn);
    a.e = p.e;
    const int sl = p.e.res.f32 ? 4 : 2;
    a.side_vec = p.e.res.p && p.e.res.sc == 1 && aligned16(p.e.res.p, p.e.res.sr, sl);
    a.out_vec = aligned16(p.e.out, p.e.ldo, p.e.out_f32 ? 4 : 2) && (!p.e.out2 || aligned16(p.e.out2, p.e.ldo, 2));
    a.partial = partial;
    a.ldp = ldp;
    // (before the maps: this call binds the device's context to the thread, which encoding a
    // map needs and autograd's threads may not have)
    const Kernel kern = pl.cg == 2 ? kernel_of<T, 2>(p) : kernel_of<T, 1>(p);
    cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) return set_error(MABA_ERR_CUDA, "dense(tcgen05): %s", cudaGetErrorString(err));
    CUtensorMap m[4];
    const int na = p.form == F_SUM || p.form == F_PAIR ? 2 : 1, nb = p.form == F_SUM || dual ? 2 : 1;
    const int box = dual ? pl.bn / 2 : a.b_rows;
    bool ok = true;
    for (int i = 0; i < 2; ++i) {
        ok = ok && operand_map(&m[i], dt, p.a[i < na ? i : 0], p.M, p.K, a_mn, 128);
        ok = ok && operand_map(&m[2 + i], dt, p.b[i < nb ? i : 0], p.N, p.K, b_mn, box);
    }
    if (!ok) return set_error(MABA_ERR_CUDA, "dense: tensor map refused");
    const int slots = sm_count() / pl.cg;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.units < slots ? a.units : slots) * pl.cg));
    cfg.blockDim = dim3(NTHR);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)pl.cg;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pl.cg == 2 ? 1 : 0;
    err = cudaLaunchKernelEx(&cfg, kern, a, m[0], m[1], m[2], m[3]);
    if (err != cudaSuccess) return set_error(MABA_ERR_CUDA, "dense(tcgen05): %s", cudaGetErrorString(err));
    return check_launch("dense(tcgen05)");
}
template int tc_product<__half>(const Product&, float*, int64_t, cudaStream_t);
template int tc_product<__nv_bfloat16>(const Product&, float*, int64_t, cudaStream_t);

int device_error_take(cudaStream_t s, int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_dense_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return set_error(MABA_ERR_CUDA, "device_error: %s", cudaGetErrorString(e));
    const int zero = 0;
    if (v != 0) cudaMemcpyToSymbolAsync(g_dense_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
    *out = v;
    return MABA_OK;
}

}  // namespace dense
}  // namespace maba
