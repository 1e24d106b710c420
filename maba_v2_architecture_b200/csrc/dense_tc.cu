// Products on the 5th-generation tensor cores (tcgen05, TMEM, TMA).
//
// 16-bit operands are multiplied as they are.  A float32 operand is three bf16 planes,
// x = x1 + x2 + x3 exactly, |x2| <= 2^-8 |x|, |x3| <= 2^-16 |x|; of the nine products the
// six down to 2^-16 are taken, x1 w1 into one accumulator, x1 w2 + x2 w1 + x2 w2 + x1 w3 +
// x3 w1 into a second, and what is left out is below 2^-23 of |x w|: float32's own rounding,
// at six tensor products instead of the CUDA cores' one (where main is an infinity or NaN the
// second sum, which may hold inf * 0, is not added).
//
// The tensor cores truncate when they add to their float32 accumulator, once per 16
// contraction indices: a sum over K loses about K 5.6e-10 of itself toward zero (measured
// 6e-7 relative at K = 640, 4.4e-6 at 4,096).  That is far below a 16-bit result's rounding,
// but not below a float32 result's, so sums that end in float32 (MODE 1 and 2) leave TMEM
// every 512 (256) indices and are added, rounded to nearest, in the epilogue's registers.
//
// Persistent, one CTA per SM.  A work unit is a tile of C (128 rows of A by bn rows of B;
// with CG = 2 a cluster's two CTAs share a tile of 256 rows: each loads its own 128 rows of
// A and one half of B, so a k-block costs an SM 32 KB for 128 x 256 x 64 products instead
// of 48 KB, below what L2 delivers per SM) over one split of the contraction.  Twelve warps:
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

// Three warpgroups: 0..7 epilogue, 8 TMA, 9 MMA, 10 and 11 idle (they complete the warpgroup
// that lends its registers): 256 x REG_EPI + 128 x REG_OTHER is what 384 threads are launched
// with, and the epilogue's sums and pieces in flight do not spill.
constexpr int NTHR = 384, EPI_WARPS = 8, W_TMA = 8, W_MMA = 9;
constexpr int REG_LAUNCH = 168, REG_EPI = 224, REG_OTHER = 56;
static_assert(256 * REG_EPI + 128 * REG_OTHER <= NTHR * REG_LAUNCH, "register split exceeds the launch");
constexpr int BK = 64;
constexpr uint32_t A_BYTES = 128 * BK * 2;
constexpr int MAX_STAGES = 8;
constexpr uint32_t STAGING = 32 * 128;  // one warp's 32 x 32 float32 chunk
constexpr uint32_t ROW_TAIL = EPI_WARPS * STAGING + EPI_WARPS * 2 * 32 * 4;  // (not in fragment order)
constexpr uint32_t BAR_BYTES = 256;
constexpr uint32_t SMEM_MAX = 227 * 1024;
constexpr int TMEM_COLS = 512, ACC_COLS = 256, MINOR = 128;  // MINOR: the second accumulator of float32 products

enum { B_FULL = 0, B_EMPTY = MAX_STAGES, B_TFULL = 2 * MAX_STAGES, B_TEMPTY = B_TFULL + 2, B_DRAIN = B_TEMPTY + 2, N_BARS };
static_assert(N_BARS * 8 + 8 <= 256, "barrier area");

struct TcArgs {
    int64_t M, N;
    int kblocks, kseg, kb_split;  // contraction blocks over all segments, of one segment, of one split
    int tiles_n, splits, pairs, units, dual;
    int bn, b_rows;  // columns of the MMA, rows of B per CTA
    int flush;       // contraction blocks between two readings of the accumulator
    int stages;
    uint32_t stage_bytes, b_at, b_bytes, load_bytes;  // B's place in a stage, one plane of it, bytes per stage
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

// phi and phi' of 16-bit operands on the SFU's exponential and reciprocal (a few float32
// ulp); of float32 ones (EXACT) as dense.cuh has them.
template <int ACT, bool EXACT> __device__ __forceinline__ float act16(float z) {
    if (ACT == ACT_SILU && !EXACT) return silu_f(z);
    return act_f(z, ACT);
}
template <int ACT, bool EXACT> __device__ __forceinline__ void act_grad16(float z, float& y, float& d) {
    if (ACT == ACT_SILU && !EXACT) {
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
// directions are free of bank conflicts.  A chunk that lies inside the matrix and on 16-byte
// boundaries moves in 16-byte pieces with one address and constant steps (the epilogue is
// bound by its instruction count); the others go element by element, out of line.
// --------------------------------------------------------------------------
__device__ __forceinline__ uint4* at32(unsigned char* st, int row, int piece) {
    return reinterpret_cast<uint4*>(st + row * 128 + ((piece ^ (row & 7)) << 4));
}
__device__ __forceinline__ uint4* at16(unsigned char* st, int row, int piece) {
    return reinterpret_cast<uint4*>(st + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}
struct Chunk {
    int64_t row0, col0;
    int rows, cols;  // of 32, inside the matrix
};

template <typename E> __device__ __forceinline__ E* element(unsigned char* st, int r, int c) {
    return sizeof(E) == 4 ? reinterpret_cast<E*>(at32(st, r, c >> 2)) + (c & 3)
                          : reinterpret_cast<E*>(at16(st, r, c >> 3)) + (c & 7);
}
// (src, dst: the chunk's first element)
template <typename E>
__device__ __noinline__ void stage_in(unsigned char* st, const E* src, int64_t sr, int64_t sc, int rows, int cols, int lane) {
    for (int r = 0; r < 32; ++r) *element<E>(st, r, lane) = r < rows && lane < cols ? src[r * sr + lane * sc] : E(0);
}
template <typename E>
__device__ __noinline__ void stage_out(unsigned char* st, E* dst, int64_t ld, int rows, int cols, int lane) {
    for (int r = 0; r < rows; ++r)
        if (lane < cols) dst[r * ld + lane] = *element<E>(st, r, lane);
}

// The pieces of a whole chunk, in flight in registers (8 of float32, 4 of 16 bits).
template <int EL> __device__ __forceinline__ void fetch_pieces(uint4* v, const Side& s, const Chunk& k, int lane) {
    constexpr int PER = 32 * EL / 16, N = 32 * PER / 32;  // pieces per row, pieces per lane
    const unsigned char* p = static_cast<const unsigned char*>(s.p) +
                             ((k.row0 + lane / PER) * s.sr + k.col0) * EL + (lane % PER) * 16;
    const int64_t step = s.sr * (EL * (32 / PER));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = *reinterpret_cast<const uint4*>(p + i * step);
}
// ... put into the staging area (the others straight from memory)
template <typename T>
__device__ __forceinline__ void stage_side(const uint4* v, bool f32, bool whole, const Side& s, const Chunk& k,
                                           unsigned char* st, int lane) {
    __syncwarp();
    if (sizeof(T) == 4 || f32) {
        if (whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) *at32(st, i * 4 + (lane >> 3), lane & 7) = v[i];
        } else {
            stage_in<float>(st, static_cast<const float*>(s.p) + k.row0 * s.sr + k.col0 * s.sc, s.sr, s.sc, k.rows, k.cols, lane);
        }
    } else {
        if (whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *at16(st, i * 8 + (lane >> 2), lane & 3) = v[i];
        } else {
            stage_in<uint16_t>(st, static_cast<const uint16_t*>(s.p) + k.row0 * s.sr + k.col0 * s.sc, s.sr, s.sc, k.rows, k.cols,
                               lane);
        }
    }
    __syncwarp();
}
// f(j, value) for the 32 staged values of this lane's row (read piece by piece: 32 registers
// for all of them would spill)
template <typename T, typename F>
__device__ __forceinline__ void with_side(bool f32, unsigned char* st, int lane, F f) {
    if (sizeof(T) == 4 || f32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 q = *reinterpret_cast<const float4*>(at32(st, lane, i));
            f(4 * i, q.x), f(4 * i + 1, q.y), f(4 * i + 2, q.z), f(4 * i + 3, q.w);
        }
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 q = *at16(st, lane, i);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 x = unpack2<T>(w[e]);
                f(8 * i + 2 * e, x.x), f(8 * i + 2 * e + 1, x.y);
            }
        }
    }
}
template <int EL>
__device__ __forceinline__ void store_pieces(unsigned char* st, void* out, int64_t ld, const Chunk& k, int lane) {
    constexpr int PER = 32 * EL / 16, N = 32 * PER / 32, RS = 32 / PER;
    unsigned char* p = static_cast<unsigned char*>(out) + ((k.row0 + lane / PER) * ld + k.col0) * EL + (lane % PER) * 16;
    const int64_t step = ld * (EL * RS);
#pragma unroll
    for (int i = 0; i < N; ++i)
        *reinterpret_cast<uint4*>(p + i * step) =
            EL == 4 ? *at32(st, i * RS + lane / PER, lane % PER) : *at16(st, i * RS + lane / PER, lane % PER);
}
template <typename T>
__device__ __forceinline__ void store_rows(const float* x, void* out, bool f32, int64_t ld, bool vec, const Chunk& k,
                                           unsigned char* st, int lane) {
    const bool whole = vec && k.rows == 32 && k.cols == 32;
    __syncwarp();
    if (sizeof(T) == 4 || f32) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4*>(at32(st, lane, i)) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        __syncwarp();
        if (whole) store_pieces<4>(st, out, ld, k, lane);
        else stage_out<float>(st, static_cast<float*>(out) + k.row0 * ld + k.col0, ld, k.rows, k.cols, lane);
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *at16(st, lane, i) = make_uint4(pack2<T>(x[8 * i], x[8 * i + 1]), pack2<T>(x[8 * i + 2], x[8 * i + 3]),
                                            pack2<T>(x[8 * i + 4], x[8 * i + 5]), pack2<T>(x[8 * i + 6], x[8 * i + 7]));
        __syncwarp();
        if (whole) store_pieces<2>(st, out, ld, k, lane);
        else stage_out<uint16_t>(st, static_cast<uint16_t*>(out) + k.row0 * ld + k.col0, ld, k.rows, k.cols, lane);
    }
}
// x op= the 32 values of a shared vector
template <typename F> __device__ __forceinline__ void with_vector(float* x, const float* v, F f) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        const float4 q = *reinterpret_cast<const float4*>(v + j);
        f(x[j], q.x), f(x[j + 1], q.y), f(x[j + 2], q.z), f(x[j + 3], q.w);
    }
}
// --------------------------------------------------------------------------
// The same chunks in fragment order (tmem_ld_frag32): four lanes hold a 32-byte piece of a
// float32 row, so they load and store without staging.  Float32 tiles staged both ways took
// the shared memory bandwidth that the tensor cores read their operands with; and a column's
// 32 rows lie in 8 lanes, so its sum takes 7 exchanges for 8 columns instead of 31 for 32.
// Element j = 16 b + 4 g + 2 i + e: row 16 b + 8 i + lane / 4, column 8 g + 2 (lane % 4) + e.
// --------------------------------------------------------------------------
__device__ __forceinline__ int frag_row(int j, int lane) { return (j >> 4) * 16 + ((j >> 1) & 1) * 8 + (lane >> 2); }
__device__ __forceinline__ int frag_col(int j, int lane) { return ((j >> 2) & 3) * 8 + (lane & 3) * 2 + (j & 1); }

template <typename E> struct Pair2;
template <> struct Pair2<float> { using type = float2; };
template <> struct Pair2<uint16_t> { using type = uint32_t; };

// v: 16 pairs (pair j / 2 of elements j, j + 1)
template <typename E>
__device__ __forceinline__ void frag_fetch(typename Pair2<E>::type* v, const Side& s, bool vec, const Chunk& k, int lane) {
    using P = typename Pair2<E>::type;
    const E* p = static_cast<const E*>(s.p) + (k.row0 + (lane >> 2)) * s.sr + (k.col0 + (lane & 3) * 2) * s.sc;
    if (vec && k.rows == 32 && k.cols == 32) {
#pragma unroll
        for (int q = 0; q < 16; ++q)
            v[q] = *reinterpret_cast<const P*>(p + ((q >> 3) * 16 + (q & 1) * 8) * s.sr + ((q >> 1) & 3) * 8);
    } else {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            E t[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = frag_row(2 * q, lane), c = frag_col(2 * q, lane) + e;
                t[e] = r < k.rows && c < k.cols ? p[(r - (lane >> 2)) * s.sr + (c - (lane & 3) * 2) * s.sc] : E(0);
            }
            v[q] = *reinterpret_cast<P*>(t);
        }
    }
}
template <typename E>
__device__ __forceinline__ void frag_put(const typename Pair2<E>::type* v, void* out, int64_t ld, bool vec, const Chunk& k,
                                         int lane) {
    using P = typename Pair2<E>::type;
    E* p = static_cast<E*>(out) + (k.row0 + (lane >> 2)) * ld + k.col0 + (lane & 3) * 2;
    if (vec && k.rows == 32 && k.cols == 32) {
#pragma unroll
        for (int q = 0; q < 16; ++q) *reinterpret_cast<P*>(p + ((q >> 3) * 16 + (q & 1) * 8) * ld + ((q >> 1) & 3) * 8) = v[q];
    } else {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const E* t = reinterpret_cast<const E*>(&v[q]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = frag_row(2 * q, lane), c = frag_col(2 * q, lane) + e;
                if (r < k.rows && c < k.cols) p[(r - (lane >> 2)) * ld + c - (lane & 3) * 2] = t[e];
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void frag_store(const float* z, void* out, bool f32, int64_t ld, bool vec, const Chunk& k, int lane) {
    if (sizeof(T) == 4 || f32) {
        frag_put<float>(reinterpret_cast<const float2*>(z), out, ld, vec, k, lane);
    } else if constexpr (sizeof(T) == 2) {
        uint32_t v[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) v[q] = pack2<T>(z[2 * q], z[2 * q + 1]);
        frag_put<uint16_t>(v, out, ld, vec, k, lane);
    }
}
// f(j, value) for the 32 fetched values
template <typename T, typename F> __device__ __forceinline__ void with_frag(bool f32, const uint32_t* v, F f) {
    if (sizeof(T) == 4 || f32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) f(j, __uint_as_float(v[j]));
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const float2 x = unpack2<T>(v[q]);
            f(2 * q, x.x), f(2 * q + 1, x.y);
        }
    }
}
// this lane's 8 columns of a vector, and x[j] op= the one of element j
template <typename T> __device__ __forceinline__ void frag_vector(float* v, const Side& s, const Chunk& k, int lane, float none) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const int c = (q >> 1) * 8 + (lane & 3) * 2 + (q & 1);
        v[q] = c < k.cols ? side_at<T>(s, 0, k.col0 + c) : none;
    }
}
__device__ __forceinline__ int frag_vec_of(int j) { return ((j >> 2) & 3) * 2 + (j & 1); }
// Column sums of a chunk over its 32 rows, in a fixed order: a lane's four rows, then the
// eight lanes of a column.  Lane l returns column frag_sum_col(l).
__device__ __forceinline__ int frag_sum_col(int lane) {
    const int q = ((lane >> 4) & 1) * 4 + ((lane >> 3) & 1) * 2 + ((lane >> 2) & 1);
    return (q >> 1) * 8 + (lane & 3) * 2 + (q & 1);
}
__device__ __forceinline__ float frag_column_sum(const float* z, int lane) {
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const int j = (q >> 1) * 4 + (q & 1);
        v[q] = (z[j] + z[j + 2]) + (z[j + 16] + z[j + 18]);
    }
#pragma unroll
    for (int o = 16, n = 4; o > 2; o >>= 1, n >>= 1) {
        const bool hi = (lane & o) != 0;
#pragma unroll
        for (int q = 0; q < n; ++q) {
            const float keep = hi ? v[q + n] : v[q], give = hi ? v[q] : v[q + n];
            v[q] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    return v[0];
}

template <typename T, int CG, bool A_MN, bool B_MN, int KIND, int MODE>
__global__ void __launch_bounds__(NTHR, 1)
    tc_kernel(const TcArgs a, const __grid_constant__ CUtensorMap ta0, const __grid_constant__ CUtensorMap ta1,
              const __grid_constant__ CUtensorMap tb0, const __grid_constant__ CUtensorMap tb1) {
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + a.stages * a.stage_bytes);
    unsigned char* tail = base + a.stages * a.stage_bytes + BAR_BYTES;  // staging, then [8 warps][scale, bias][32]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + N_BARS);
    volatile int* abort_f = reinterpret_cast<volatile int*>(tmem_slot + 1);

    constexpr int PLANES = MODE == 2 ? 3 : 1;
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
    auto unit_of = [&](int unit) {
        Unit t;
        unsigned u = (unsigned)unit;
        t.split = t.pair = 0;
        if (a.splits > 1) t.split = (int)(u % (unsigned)a.splits), u /= (unsigned)a.splits;
        if (a.pairs > 1) t.pair = (int)(u & 1u), u >>= 1;
        const unsigned row = u / (unsigned)a.tiles_n;
        t.n0 = (int64_t)(u - row * (unsigned)a.tiles_n) * (a.dual ? a.bn / 2 : a.bn);
        t.m0 = (int64_t)row * (128 * CG) + rank * 128;
        t.kb0 = t.split * a.kb_split;
        t.kb1 = t.kb0 + a.kb_split < a.kblocks ? t.kb0 + a.kb_split : a.kblocks;
        return t;
    };

    if (warp >= EPI_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_OTHER));
    if (warp == W_TMA) {
        // ============================ TMA producer ============================
        // One thread runs the loop: a warp-wide one with an election for each copy took longer
        // to issue a k-block than the tensor cores to multiply it.
        if (elect_one()) {
        int st = 0, it = 0;
        uint32_t phase = 1;  // (a fresh barrier's previous phase counts as complete)
        bool ok = true;
        for (int u = worker; u < a.units && ok; u += workers) {
            const Unit t = unit_of(u);
            for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                ok = mbar_wait(&bars[B_EMPTY + st], phase, abort_f);
                if (!ok) break;
                const int seg = kb >= a.kseg ? 1 : 0, k0 = (kb - seg * a.kseg) * BK;
                const CUtensorMap* ma = (a.pairs == 2 ? t.pair : seg) ? &ta1 : &ta0;
                unsigned char* sa = base + st * a.stage_bytes;
                {
                    uint64_t* full = &bars[B_FULL + st];
                    const uint32_t full0 = CG == 2 ? cluster_addr(full, 0) : 0u;
                    auto load = [&](unsigned char* dst, const CUtensorMap* m, int x, int y, int plane) {
                        if (CG == 2) tma_load_3d_pair(dst, m, full0, x, y, plane);
                        else tma_load_3d(dst, m, full, x, y, plane);
                    };
                    if (rank == 0) mbar_arrive_expect_tx(full, a.load_bytes);
#pragma unroll
                    for (int pl = 0; pl < PLANES; ++pl, sa += A_BYTES) {
                        unsigned char* sb = base + st * a.stage_bytes + a.b_at + pl * a.b_bytes;
                        if (A_MN) {
                            load(sa, ma, (int)t.m0, k0, pl);
                            load(sa + A_BYTES / 2, ma, (int)t.m0 + 64, k0, pl);
                        } else {
                            load(sa, ma, k0, (int)t.m0, pl);
                        }
                        if (KIND == E_GLU || KIND == E_GLU_BWD) {
                            if (CG == 2) {
                                load(sb, rank ? &tb1 : &tb0, k0, (int)t.n0, pl);
                            } else {
                                load(sb, &tb0, k0, (int)t.n0, pl);
                                load(sb + a.bn / 2 * 128, &tb1, k0, (int)t.n0, pl);
                            }
                        } else {
                            const CUtensorMap* mb = seg ? &tb1 : &tb0;
                            const int y = (int)t.n0 + (int)rank * a.b_rows;
                            if (B_MN) {
                                for (int i = 0; i < a.b_rows; i += 64) load(sb + i * 128, mb, y + i, k0, pl);
                            } else {
                                load(sb, mb, k0, y, pl);
                            }
                        }
                    }
                }
                if (++st == a.stages) st = 0, phase ^= 1;
            }
        }
        // every copy has landed before a CTA may exit (rank 0's barriers count the pair's)
        if (rank == 0)
            for (int s = 0; s < a.stages && s < it; ++s)
                mbar_wait(&bars[B_FULL + s], (((it - 1 - s) / a.stages)) & 1, nullptr);
        }
    } else if (warp == W_MMA) {
        // ============================ MMA issuer ==============================
        if (rank == 0 && elect_one()) {
            const uint64_t ad0 = sdesc_sw128(smem_addr(base), A_MN ? A_BYTES / 2 : 16, 1024);
            const uint64_t bd0 = sdesc_sw128(smem_addr(base + a.b_at), B_MN ? 8192 : 16, 1024);
            constexpr uint32_t ak = A_MN ? 2048 >> 4 : 32 >> 4, bk = B_MN ? 2048 >> 4 : 32 >> 4;
            auto mma = [&](uint32_t d, uint64_t ad, uint64_t bd, uint32_t acc) {
                if (CG == 2) umma_f16_ss_pair(d, ad, bd, a.idesc, acc);
                else umma_f16_ss(d, ad, bd, a.idesc, acc);
            };
            auto commit = [&](uint64_t* bar) {
                if (CG == 2) umma_commit_pair(bar);
                else umma_commit(bar);
            };
            int st = 0, buf = 0;
            uint32_t phase = 0, tphase = 1;
            bool ok = true;
            for (int u = worker; u < a.units && ok; u += workers) {
                const Unit t = unit_of(u);
                for (int f0 = t.kb0; f0 < t.kb1; f0 += a.flush) {
                    const int f1 = f0 + a.flush < t.kb1 ? f0 + a.flush : t.kb1;
                    const uint32_t d = tmem + buf * ACC_COLS;
                    ok = mbar_wait(&bars[B_TEMPTY + buf], tphase, abort_f);
                    if (!ok) break;
                    tc_fence_after();
                    for (int kb = f0; kb < f1; ++kb) {
                        ok = mbar_wait(&bars[B_FULL + st], phase, abort_f);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t so = (uint64_t)(st * (a.stage_bytes >> 4));
                        const uint64_t ad = ad0 + so, bd = bd0 + so;
                        const uint64_t bp = a.b_bytes >> 4;  // from one plane of B to the next
                        constexpr uint64_t ap = A_BYTES >> 4;
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) {
                            const uint32_t acc = kb > f0 || k > 0 ? 1u : 0u;
                            mma(d, ad + k * ak, bd + k * bk, acc);
                            if (PLANES == 3) {
                                mma(d + MINOR, ad + k * ak, bd + k * bk + 2 * bp, acc);
                                mma(d + MINOR, ad + k * ak + 2 * ap, bd + k * bk, 1u);
                                mma(d + MINOR, ad + k * ak + ap, bd + k * bk + bp, 1u);
                                mma(d + MINOR, ad + k * ak, bd + k * bk + bp, 1u);
                                mma(d + MINOR, ad + k * ak + ap, bd + k * bk, 1u);
                            }
                        }
                        commit(&bars[B_EMPTY + st]);
                        if (++st == a.stages) st = 0, phase ^= 1;
                    }
                    if (!ok) break;
                    commit(&bars[B_TFULL + buf]);
                    buf ^= 1;
                    if (buf == 0) tphase ^= 1;
                }
            }
            // every product has completed before TMEM is freed
            commit(&bars[B_DRAIN]);
            mbar_wait(&bars[B_DRAIN], 0, nullptr);
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_EPI));
        // ============================== epilogue ==============================
        constexpr bool DUAL = KIND == E_GLU || KIND == E_GLU_BWD, EXACT = MODE == 2;
        // chunks in fragment order: float32 in and out, and where columns are summed
        constexpr bool FRAG = MODE != 0 || KIND == E_LINEAR_BWD;
        constexpr bool VECS = KIND == E_LINEAR || KIND == E_LINEAR_BWD;
        // MODE 1, 2: chunks (of a pair of projections: one) whose sums a warp holds
        constexpr int CH = MODE == 0 || DUAL ? 1 : (MODE == 1 ? 4 : 2);
        const int q = warp & 3, h = warp >> 2;
        unsigned char* st = tail + warp * STAGING;
        float* vscale = reinterpret_cast<float*>(tail + EPI_WARPS * STAGING) + warp * 64;
        float* vbias = vscale + 32;
        const Epilogue& e = a.e;
        const int width = DUAL ? a.bn / 2 : a.bn;
        const bool has_side = KIND != E_STORE && KIND != E_GLU && e.res.p != nullptr;
        const bool side_f32 = sizeof(T) == 4 || e.res.f32, out_f32 = sizeof(T) == 4 || e.out_f32;
        int buf = 0;
        uint32_t phase = 0;
        auto wait_full = [&]() {
            const bool ok = mbar_wait_warp(&bars[B_TFULL + buf], phase, abort_f);
            tc_fence_after();
            return ok;
        };
        auto release = [&]() {  // this warp has read its part of the accumulator
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) mbar_arrive_cluster(cluster_addr(&bars[B_TEMPTY + buf], 0));
                else mbar_arrive(&bars[B_TEMPTY + buf]);
            }
            buf ^= 1;
            if (buf == 0) phase ^= 1;
        };
        for (int u = worker; u < a.units; u += workers) {
            const Unit t = unit_of(u);
            const int64_t row0 = t.m0 + q * 32;
            const bool live = row0 < a.M;
            const int rows = a.M - row0 < 32 ? (int)(a.M - row0) : 32;
            auto place = [&](int c) {
                Chunk k;
                k.row0 = row0, k.col0 = t.n0 + c * 32;
                k.rows = rows;
                k.cols = a.N - k.col0 < 32 ? (int)(a.N - k.col0) : 32;
                return k;
            };
            auto side_whole = [&](const Chunk& k) { return a.side_vec && k.rows == 32 && k.cols == 32; };
            uint4 side[8];           // the chunk's pieces of residual or gradient, in flight
            float ps = 0.f, pb = 0.f;  // this lane's column of scale and bias
            auto fetch = [&](int c) {
                const Chunk k = place(c);
                if (k.cols <= 0) return;
                if (FRAG) {
                    if (has_side) {
                        if (side_f32) frag_fetch<float>(reinterpret_cast<float2*>(side), e.res, a.side_vec, k, lane);
                        else frag_fetch<uint16_t>(reinterpret_cast<uint32_t*>(side), e.res, a.side_vec, k, lane);
                    }
                    return;
                }
                if (has_side && side_whole(k)) {
                    if (side_f32) fetch_pieces<4>(side, e.res, k, lane);
                    else fetch_pieces<2>(side, e.res, k, lane);
                }
                if (VECS) {
                    if (e.scale.p) ps = lane < k.cols ? side_at<T>(e.scale, 0, k.col0 + lane) : 1.f;
                    if (e.bias.p) pb = lane < k.cols ? side_at<T>(e.bias, 0, k.col0 + lane) : 0.f;
                }
            };
            // one chunk of sums: the epilogue in fragment order
            auto chunk_frag = [&](int c, float* z, float* w, bool more) {
                const Chunk k = place(c);
                if (!live || k.cols <= 0) return;
                const uint32_t* sv = reinterpret_cast<const uint32_t*>(side);
                if (KIND == E_STORE) {
                    if (a.splits > 1)
                        frag_store<T>(z, a.partial + ((int64_t)t.split * a.pairs + t.pair) * a.M * a.ldp, true, a.ldp, true, k,
                                      lane);
                    else
                        frag_store<T>(z, t.pair ? e.out2 : e.out, out_f32, e.ldo, a.out_vec, k, lane);
                    return;
                }
                float vs[VECS ? 8 : 1], vb[VECS ? 8 : 1];
                if (VECS && e.scale.p) frag_vector<T>(vs, e.scale, k, lane, 1.f);
                if (VECS && e.bias.p) {
                    frag_vector<T>(vb, e.bias, k, lane, 0.f);
#pragma unroll
                    for (int j = 0; j < 32; ++j) z[j] += vb[frag_vec_of(j)];
                }
                if (KIND == E_LINEAR) {
                    with_act(e.act, [&](auto A) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) z[j] = act16<A.value, EXACT>(z[j]);
                    });
                    if (e.scale.p) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) z[j] *= vs[frag_vec_of(j)];
                    }
                    if (has_side) with_frag<T>(side_f32, sv, [&](int j, float g) { z[j] += g; });
                    if (more) fetch(c + 2);
                    frag_store<T>(z, e.out, out_f32, e.ldo, a.out_vec, k, lane);
                } else if (KIND == E_LINEAR_BWD) {
                    float y[32];
                    with_act(e.act, [&](auto A) {
                        with_frag<T>(side_f32, sv, [&](int j, float g) {
                            float f, d;
                            act_grad16<A.value, EXACT>(z[j], f, d);
                            z[j] = g * d;
                            y[j] = g * f;
                        });
                    });
                    if (more) fetch(c + 2);
                    if (e.scale.p) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) z[j] *= vs[frag_vec_of(j)];
                    }
                    if (k.rows < 32) {  // rows past the last: no part in the sums, whatever the bias is
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (frag_row(j, lane) >= k.rows) z[j] = y[j] = 0.f;
                    }
                    frag_store<T>(z, e.out, out_f32, e.ldo, a.out_vec, k, lane);
                    const int col = frag_sum_col(lane);
                    const int64_t at = (row0 >> 5) * a.N + k.col0 + col;
                    if (e.part_bias) {
                        const float s = frag_column_sum(z, lane);
                        if (col < k.cols) e.part_bias[at] = s;
                    }
                    if (e.part_scale) {
                        const float s = frag_column_sum(y, lane);
                        if (col < k.cols) e.part_scale[at] = s;
                    }
                } else if (KIND == E_GLU) {
                    with_act(e.act, [&](auto A) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) z[j] = act16<A.value, EXACT>(z[j]) * w[j];
                    });
                    frag_store<T>(z, e.out, out_f32, e.ldo, a.out_vec, k, lane);
                } else {
                    with_act(e.act, [&](auto A) {
                        with_frag<T>(side_f32, sv, [&](int j, float g) {
                            float f, d;
                            act_grad16<A.value, EXACT>(z[j], f, d);
                            z[j] = g * w[j] * d;
                            w[j] = g * f;
                        });
                    });
                    if (more) fetch(c + 2);
                    frag_store<T>(z, e.out, out_f32, e.ldo, a.out_vec, k, lane);
                    frag_store<T>(w, e.out2, out_f32, e.ldo, a.out_vec, k, lane);
                }
            };
            // and with a lane for a row, through the staging area
            auto chunk_rows = [&](int c, float* z, float* w, bool more) {
                const Chunk k = place(c);
                if (!live || k.cols <= 0) return;
                if (has_side) stage_side<T>(side, side_f32, side_whole(k), e.res, k, st, lane);
                if (VECS) {
                    __syncwarp();
                    vscale[lane] = ps;
                    vbias[lane] = pb;
                    __syncwarp();
                }
                if (more) fetch(c + 2);
                if (KIND == E_LINEAR) {
                    if (e.bias.p) with_vector(z, vbias, [](float& x, float v) { x += v; });
                    with_act(e.act, [&](auto A) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) z[j] = act16<A.value, EXACT>(z[j]);
                    });
                    if (e.scale.p) with_vector(z, vscale, [](float& x, float v) { x *= v; });
                    if (has_side) with_side<T>(side_f32, st, lane, [&](int j, float g) { z[j] += g; });
                } else if (KIND == E_GLU) {
                    with_act(e.act, [&](auto A) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) z[j] = act16<A.value, EXACT>(z[j]) * w[j];
                    });
                } else if (KIND == E_GLU_BWD) {
                    with_act(e.act, [&](auto A) {
                        with_side<T>(false, st, lane, [&](int j, float g) {
                            float f, d;
                            act_grad16<A.value, EXACT>(z[j], f, d);
                            z[j] = g * w[j] * d;
                            w[j] = g * f;
                        });
                    });
                }
                store_rows<T>(z, t.pair ? e.out2 : e.out, out_f32, e.ldo, a.out_vec, k, st, lane);
                if (KIND == E_GLU_BWD) store_rows<T>(w, e.out2, out_f32, e.ldo, a.out_vec, k, st, lane);
            };
            if constexpr (MODE != 0) {
                float sz[CH][32], sw[DUAL ? 32 : 1];  // the unit's accumulations, added up
#pragma unroll
                for (int j = 0; j < 32; ++j) {
#pragma unroll
                    for (int cc = 0; cc < CH; ++cc) sz[cc][j] = 0.f;
                    if (DUAL) sw[j] = 0.f;
                }
                bool ok = true;
                for (int f0 = t.kb0; f0 < t.kb1; f0 += a.flush) {
                    ok = wait_full();
                    if (!ok) break;
                    const uint32_t acc = tmem + buf * ACC_COLS + ((uint32_t)(q * 32) << 16);
                    auto add = [&](float* sum, int col) {
                        float z[32];
                        tmem_ld_frag32(acc + col, reinterpret_cast<uint32_t*>(z));
                        if (MODE == 2) {
                            float y[32];
                            tmem_ld_frag32(acc + MINOR + col, reinterpret_cast<uint32_t*>(y));
                            tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(z));
                            tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(y));
#pragma unroll
                            for (int j = 0; j < 32; ++j) sum[j] += isfinite(z[j]) ? z[j] + y[j] : z[j];
                        } else {
                            tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(z));
#pragma unroll
                            for (int j = 0; j < 32; ++j) sum[j] += z[j];
                        }
                    };
#pragma unroll
                    for (int cc = 0; cc < CH; ++cc)
                        if ((h + 2 * cc) * 32 < width) add(sz[cc], (h + 2 * cc) * 32);
                    if (DUAL && h * 32 < width) add(sw, width + h * 32);
                    release();
                }
                if (!ok) break;
                if (live && h * 32 < width) fetch(h);  // (here, or its registers would live through the sums)
#pragma unroll
                for (int cc = 0; cc < CH; ++cc) {
                    const int c = h + 2 * cc;
                    if (c * 32 < width) chunk_frag(c, sz[cc], sw, cc + 1 < CH && (c + 2) * 32 < width);
                }
            } else {
                if (live && h * 32 < width) fetch(h);
                if (!wait_full()) break;
                const uint32_t acc = tmem + buf * ACC_COLS + ((uint32_t)(q * 32) << 16);
                if (h * 32 >= width) release();
                for (int c = h; c * 32 < width; c += 2) {
                    const bool more = (c + 2) * 32 < width;
                    float z[32], w[DUAL ? 32 : 1];
                    const bool frag = FRAG || (KIND == E_STORE && a.splits > 1);
                    if (frag) {
                        tmem_ld_frag32(acc + c * 32, reinterpret_cast<uint32_t*>(z));
                    } else {
                        tmem_ld32(acc + c * 32, reinterpret_cast<uint32_t*>(z));
                        if (DUAL) tmem_ld32(acc + width + c * 32, reinterpret_cast<uint32_t*>(w));
                    }
                    tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(z));
                    if (DUAL) tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(w));
                    if (!more) release();
                    if (frag) chunk_frag(c, z, w, more);
                    else chunk_rows(c, z, w, more);
                }
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

// How a product's sums are kept: 0 one accumulation (16-bit results), 1 added up in registers
// every 512 indices (float32 results of 16-bit operands), 2 float32 operands, every 256.
int mode_of(const Product& p, int dt) {
    if (dt == MABA_F32) return 2;
    return p.e.kind == E_LINEAR && p.e.out_f32 ? 1 : 0;
}

// The tile and the splits with the least estimated time.  Per k-block and SM: the larger of
// the products (128 x bn x 64 at 4,096 per cycle) and the loads (60 bytes per cycle from L2);
// a unit that is not hidden under another adds its fill and epilogue.  The registers that
// hold a unit's sums bound bn in modes 1 and 2.  Splits also bound what one accumulation
// truncates: at most 16,384 indices.
Plan plan_of(const Product& p, int mode) {
    const bool dual = p.form == F_DUAL, store = p.e.kind == E_STORE;
    const bool b_mn = store;
    const int64_t kblocks = ceil_div(p.K, BK) * (p.form == F_SUM ? 2 : 1);
    const int64_t pairs = p.form == F_PAIR ? 2 : 1;
    const int planes = mode == 2 ? 3 : 1, terms = mode == 2 ? 6 : 1;
    int64_t fewest = store && mode == 0 ? ceil_div(kblocks, 256) : 1;
    Plan best;
    double least = 1e300;
    for (int cg = 1; cg <= 2; ++cg) {
        const int most = mode == 2 ? 128 : (cg == 2 ? 256 : 192);
        for (int bn = dual ? 64 : 32; bn <= most; bn += dual ? 64 : 32) {
            const int64_t tiles = ceil_div(p.M, 128 * cg) * ceil_div(p.N, dual ? bn / 2 : bn) * pairs;
            const int64_t slots = sm_count() / cg;
            const double mma = 2.0 * bn * terms, load = planes * (A_BYTES + b_bytes_of(cg, bn, b_mn)) / 60.0;
            const double kcost = mma > load ? mma : load;
            for (int64_t splits = fewest; splits <= (store ? fewest + 15 : 1) && splits <= kblocks; ++splits) {
                const int64_t units = tiles * splits;
                const double waves = (double)ceil_div(units, slots);
                const double kb = (double)ceil_div(kblocks, splits);
                double t = waves * kb * kcost + 2000.0 + 12.0 * bn;
                // the partial sums, written and read: bytes at ~3,500 per cycle over the GPU, and a launch
                if (splits > 1) t += 2000.0 + 8.0 * (double)splits * pairs * p.M * p.N / 3500.0;
                if (t < least) least = t, best = Plan{cg, bn, (int)splits};
            }
        }
    }
    return best;
}

// One operand's map: rows x contraction (x planes), read K-major (contraction contiguous) or
// MN-major.
bool operand_map(CUtensorMap* m, int dt, const Matrix& x, int planes, int64_t rows, int64_t k, bool mn, int box_rows) {
    const int64_t dims[3] = {mn ? rows : k, mn ? k : rows, planes};
    const int64_t ld = dims[1] > 1 ? (mn ? x.sk : x.sr) : (dims[0] + 7) / 8 * 8;
    const int64_t strides[2] = {ld, planes > 1 ? x.sp : ld};
    const uint32_t box[3] = {(uint32_t)BK, (uint32_t)(mn ? BK : box_rows), 1};
    return make_map(m, dt, x.p, 3, dims, strides, box);
}

bool aligned(const void* p, int64_t ld, int el, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (ld * el) % bytes == 0;
}

using Kernel = void (*)(const TcArgs, const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap);

// The register split assumes REG_LAUNCH registers per thread at launch; with fewer, the
// epilogue's increase would never complete, so such a build is not launched (nullptr).
template <typename T, int CG, bool A_MN, bool B_MN, int KIND, int MODE> Kernel checked() {
    static const bool ok = [] {
        cudaFuncAttributes fa{};
        return cudaFuncGetAttributes(&fa, tc_kernel<T, CG, A_MN, B_MN, KIND, MODE>) == cudaSuccess && fa.numRegs == REG_LAUNCH;
    }();
    return ok ? tc_kernel<T, CG, A_MN, B_MN, KIND, MODE> : nullptr;
}

template <typename T, int CG> Kernel kernel_of(const Product& p, int mode) {
    constexpr int M = sizeof(T) == 4 ? 2 : 0;
    if constexpr (M == 0)
        if (mode == 1) return checked<T, CG, false, false, E_LINEAR, 1>();
    switch (p.e.kind) {
        case E_LINEAR: return checked<T, CG, false, false, E_LINEAR, M>();
        case E_LINEAR_BWD: return checked<T, CG, false, false, E_LINEAR_BWD, M>();
        case E_GLU: return checked<T, CG, false, false, E_GLU, M>();
        case E_GLU_BWD: return checked<T, CG, false, false, E_GLU_BWD, M>();
        default: return p.a_mn ? checked<T, CG, true, true, E_STORE, M>() : checked<T, CG, false, true, E_STORE, M>();
    }
}

}  // namespace

bool tc_readable(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t col_stride) {
    if (col_stride != 1 && cols > 1) return false;
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return false;
    return rows == 1 || (ld % 8 == 0 && ld >= cols);
}

int tc_splits(const Product& p, int dt) {
    const int64_t kblocks = ceil_div(p.K, BK) * (p.form == F_SUM ? 2 : 1);
    return (int)ceil_div(kblocks, ceil_div(kblocks, plan_of(p, mode_of(p, dt)).splits));  // none is empty
}

template <typename T> int tc_product(const Product& p, float* partial, int64_t ldp, cudaStream_t s) {
    if (encode_fn() == nullptr) return set_error(MABA_ERR_CUDA, "dense: cuTensorMapEncodeTiled not found");
    constexpr int dt = sizeof(T) == 4 ? MABA_F32 : (std::is_same<T, __nv_bfloat16>::value ? MABA_BF16 : MABA_F16);
    constexpr int planes = dt == MABA_F32 ? 3 : 1, odt = dt == MABA_F16 ? MABA_F16 : MABA_BF16;
    const int mode = mode_of(p, dt);
    const Plan pl = plan_of(p, mode);
    const bool dual = p.form == F_DUAL, store = p.e.kind == E_STORE, a_mn = p.a_mn, b_mn = store;
    TcArgs a{};
    a.M = p.M, a.N = p.N;
    a.kseg = (int)ceil_div(p.K, BK);
    a.kblocks = a.kseg * (p.form == F_SUM ? 2 : 1);
    a.pairs = p.form == F_PAIR ? 2 : 1;
    a.dual = dual;
    a.kb_split = (int)ceil_div(a.kblocks, pl.splits);
    a.splits = (int)ceil_div(a.kblocks, a.kb_split);
    a.bn = pl.bn;
    a.b_rows = b_rows_of(pl.cg, pl.bn);
    a.tiles_n = (int)ceil_div(p.N, dual ? pl.bn / 2 : pl.bn);
    const int64_t units = ceil_div(p.M, 128 * pl.cg) * a.tiles_n * a.pairs * a.splits;
    if (units > 0x7fffffff) return set_error(MABA_ERR_UNSUPPORTED, "dense: %lld tiles", (long long)units);
    a.units = (int)units;
    const uint32_t bb = b_bytes_of(pl.cg, pl.bn, b_mn);
    a.flush = mode == 0 ? a.kblocks : (mode == 1 ? 512 / BK : 256 / BK);
    a.b_at = planes * A_BYTES;
    a.b_bytes = (bb + 1023) / 1024 * 1024;
    a.stage_bytes = planes * (A_BYTES + a.b_bytes);
    a.load_bytes = planes * (A_BYTES + bb) * pl.cg;
    const uint32_t tail = BAR_BYTES + (mode == 0 && p.e.kind != E_LINEAR_BWD ? ROW_TAIL : 0);
    const uint32_t room = SMEM_MAX - 1024 - tail;
    a.stages = (int)(room / a.stage_bytes);
    if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
    const size_t smem = 1024 + (size_t)a.stages * a.stage_bytes + tail;
    a.idesc = idesc_f16(128 * pl.cg, pl.bn, odt == MABA_BF16, a_mn, b_mn);
    a.e = p.e;
    const bool out_f32 = planes == 3 || p.e.out_f32;
    const int sl = p.e.res.f32 ? 4 : 2, ol = out_f32 ? 4 : 2;
    // pieces of 16 bytes, or pairs of elements in fragment order
    const bool frag = mode != 0 || p.e.kind == E_LINEAR_BWD;
    a.side_vec = p.e.res.p && p.e.res.sc == 1 && aligned(p.e.res.p, p.e.res.sr, sl, frag ? 2 * sl : 16);
    const int ob = frag ? 2 * ol : 16;
    a.out_vec = aligned(p.e.out, p.e.ldo, ol, ob) && (!p.e.out2 || aligned(p.e.out2, p.e.ldo, ol, ob));
    a.partial = partial;
    a.ldp = ldp;
    // (before the maps: this call binds the device's context to the thread, which encoding a
    // map needs and autograd's threads may not have)
    const Kernel kern = pl.cg == 2 ? kernel_of<T, 2>(p, mode) : kernel_of<T, 1>(p, mode);
    if (kern == nullptr) return set_error(MABA_ERR_UNSUPPORTED, "dense(tcgen05): built with another register count");
    cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) return set_error(MABA_ERR_CUDA, "dense(tcgen05): %s", cudaGetErrorString(err));
    CUtensorMap m[4];
    const int na = p.form == F_SUM || p.form == F_PAIR ? 2 : 1, nb = p.form == F_SUM || dual ? 2 : 1;
    const int box = dual ? pl.bn / 2 : a.b_rows;
    bool ok = true;
    for (int i = 0; i < 2; ++i) {
        ok = ok && operand_map(&m[i], odt, p.a[i < na ? i : 0], planes, p.M, p.K, a_mn, 128);
        ok = ok && operand_map(&m[2 + i], odt, p.b[i < nb ? i : 0], planes, p.N, p.K, b_mn, box);
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
template int tc_product<float>(const Product&, float*, int64_t, cudaStream_t);
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
