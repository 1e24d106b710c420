// Float32 products on the CUDA cores: any strides, float32 sums.
//
// A CTA computes a 128 x 128 tile of C (of a pair of projections 128 x 64 of each: the tile's
// columns 0..63 belong to B0, 64..127 to B1) over its share of the contraction, 16 indices at a
// time.  Both operand tiles lie contraction-major in two shared-memory buffers; the next tile is
// on its way into registers under the current one's arithmetic.  A thread owns rows and columns
// {4 t, 64 + 4 t} + 0..3, so gate and up of a pair sit in one thread, and multiplies two columns
// by one instruction (fma.f32x2).
//
// What bounds it: whole tiles on 296 places, and issue.  4,096 x 640 -> 1,544 takes 286 us, 28.3
// TFLOP/s, forward and gradients of the gated block of 2,048 x 640 -> 2 x 1,248 866 us; library
// products in float32 with separate activations take 212 and 602.  The first has 416 tiles, of
// which the last column's 32 hold 8 of 128 columns; a k index costs a thread 32 packed multiply-adds,
// 8 moves that repeat a row's value and 4 shared-memory loads.  A contraction below 1,024 is not split
// under an epilogue, so few rows leave most SMs idle: 16, 64 and 256 rows of 640 -> 1,544 take 111,
// 112 and 131 us (13 and 26 CTAs), library products 16, 17 and 24.  A 64 x 128 tile, four CTAs to an
// SM, 8 indices at a time, took 319 and 863.
#include "dense.cuh"

namespace maba {
namespace dense {
namespace {

constexpr int BM = 4 * TC_ROWS, BN = 128, BK = 16, LD = BN + 4, NTHR = 256, PER_SM = 2;

__device__ __forceinline__ unsigned long long both(float a) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(a));
    return r;
}
__device__ __forceinline__ void fma_pair(unsigned long long& c, unsigned long long a, unsigned long long b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}

// A thread's piece of 64 rows x 16 of the contraction: four elements along the contraction (kfast) or
// along the rows, whichever is the shorter stride.  A piece that is whole, contiguous and on 16
// bytes is one load; elements out of range are 0.
struct Piece {
    const float* p;  // its first element at contraction index 0
    int rows;        // kfast: 1 if its row is inside; else how many of the four are
    bool kfast, vec;
};
__device__ __forceinline__ Piece piece_of(const Matrix& m, int64_t r0, int64_t rows, int tid) {
    Piece c;
    c.kfast = m.sk <= m.sr;
    c.vec = (c.kfast ? m.sk == 1 && (m.sr & 3) == 0 : m.sr == 1 && (m.sk & 3) == 0) &&
            (reinterpret_cast<uintptr_t>(m.p) & 15u) == 0;
    const int64_t r = r0 + (c.kfast ? tid >> 2 : (tid & 15) * 4);
    const int64_t left = rows - r, most = c.kfast ? 1 : 4;
    c.rows = left <= 0 ? 0 : (int)(left < most ? left : most);
    c.p = static_cast<const float*>(m.p) + r * m.sr;
    return c;
}
__device__ __forceinline__ float4 load_piece(const Piece& c, const Matrix& m, int64_t k0, int64_t K, int tid) {
    const int64_t k = k0 + (c.kfast ? (tid & 3) * 4 : tid >> 4);
    const int64_t left = K - k;
    const int n = left <= 0 ? 0 : (c.kfast ? (c.rows ? (left < 4 ? (int)left : 4) : 0) : c.rows);
    const float* p = c.p + k * m.sk;
    if (c.vec && n == 4) return *reinterpret_cast<const float4*>(p);
    const int64_t step = c.kfast ? m.sk : m.sr;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? p[j * step] : 0.f;
    return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_piece(const float4& v, bool kfast, float* s, int tid) {
    if (kfast) {
        float* t = s + (tid & 3) * 4 * LD + (tid >> 2);
        t[0] = v.x, t[LD] = v.y, t[2 * LD] = v.z, t[3 * LD] = v.w;
    } else {
        *reinterpret_cast<float4*>(s + (tid >> 4) * LD + (tid & 15) * 4) = v;
    }
}
// four results of a row: one store where they are whole and on 16 bytes
__device__ __forceinline__ void put4(float* p, const float* v, int64_t n) {
    if (n >= 4 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < n) p[j] = v[j];
    }
}

template <bool DUAL>
__global__ void __launch_bounds__(NTHR, PER_SM)
    simt_kernel(const Product p, int tiles_n, int splits, float* partial, int64_t ldp) {
    __shared__ __align__(16) float As[2][BK * LD], Bs[2][BK * LD];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t tm = blockIdx.x / tiles_n, m0 = tm * BM, n0 = (int64_t)(blockIdx.x % tiles_n) * (DUAL ? 64 : BN);
    const int pair = p.form == F_PAIR ? blockIdx.z : 0;
    const int64_t nk = (p.K + BK - 1) / BK, total = nk * (p.form == F_SUM ? 2 : 1);
    const int64_t k_lo = total * blockIdx.y / splits, k_hi = total * (blockIdx.y + 1) / splits;

    Piece a0, a1, b0, b1;
    auto segment = [&](int sg) {
        const int i = p.form == F_PAIR ? pair : sg;
        a0 = piece_of(p.a[i], m0, p.M, tid);
        a1 = piece_of(p.a[i], m0 + 64, p.M, tid);
        b0 = piece_of(p.b[i], n0, p.N, tid);
        b1 = piece_of(p.b[DUAL ? 1 : i], DUAL ? n0 : n0 + 64, p.N, tid);
    };
    float4 va0, va1, vb0, vb1;
    int seg = k_lo >= nk ? 1 : 0;
    segment(seg);
    auto load = [&](int64_t it) {
        if (seg == 0 && it >= nk) segment(seg = 1);
        const int64_t k0 = (it - seg * nk) * BK;
        const int i = p.form == F_PAIR ? pair : seg;
        va0 = load_piece(a0, p.a[i], k0, p.K, tid), va1 = load_piece(a1, p.a[i], k0, p.K, tid);
        vb0 = load_piece(b0, p.b[i], k0, p.K, tid), vb1 = load_piece(b1, p.b[DUAL ? 1 : i], k0, p.K, tid);
    };
    auto store = [&](int buf) {  // (of the tile that load() brought last: the same segment)
        store_piece(va0, a0.kfast, As[buf], tid), store_piece(va1, a1.kfast, As[buf] + 64, tid);
        store_piece(vb0, b0.kfast, Bs[buf], tid), store_piece(vb1, b1.kfast, Bs[buf] + 64, tid);
    };
    unsigned long long acc[8][4] = {};
    if (k_lo < k_hi) {
        load(k_lo);
        store(0);
    }
    __syncthreads();
    for (int64_t it = k_lo; it < k_hi; ++it) {
        const int buf = (int)(it - k_lo) & 1;
        if (it + 1 < k_hi) load(it + 1);
#pragma unroll
        for (int k = 0; k < BK; ++k) {
            float x[8];
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(&As[buf][k * LD + ty * 4]);
            *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(&As[buf][k * LD + 64 + ty * 4]);
            const ulonglong2 y0 = *reinterpret_cast<const ulonglong2*>(&Bs[buf][k * LD + tx * 4]);
            const ulonglong2 y1 = *reinterpret_cast<const ulonglong2*>(&Bs[buf][k * LD + 64 + tx * 4]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned long long xx = both(x[i]);
                fma_pair(acc[i][0], xx, y0.x), fma_pair(acc[i][1], xx, y0.y);
                fma_pair(acc[i][2], xx, y1.x), fma_pair(acc[i][3], xx, y1.y);
            }
        }
        if (it + 1 < k_hi) store(buf ^ 1);  // (its last readers passed the barrier before this step)
        __syncthreads();
    }

    const Epilogue& e = p.e;
    const int64_t rows_out = p.form == F_PAIR ? 2 * p.M : p.M;
    float sum_b[16] = {}, sum_s[16] = {};  // of the thread's rows in either half of the tile
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t m = m0 + (i >> 2) * 64 + ty * 4 + (i & 3);
        if (m >= p.M) continue;
        float z[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 v = *reinterpret_cast<const float2*>(&acc[i][j]);
            z[2 * j] = v.x, z[2 * j + 1] = v.y;
        }
        if (DUAL) {
            const int64_t n = n0 + tx * 4;
            if (n >= p.N) continue;
            float first[4], second[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (e.kind == E_GLU) {
                    first[j] = act_f(z[j], e.act) * z[j + 4];
                } else {
                    const float g = n + j < p.N ? side_at<float>(e.res, m, n + j) : 0.f;
                    float y, d;
                    act_grad_f(z[j], e.act, y, d);
                    first[j] = g * z[j + 4] * d, second[j] = g * y;
                }
            }
            put4(static_cast<float*>(e.out) + m * e.ldo + n, first, p.N - n);
            if (e.kind == E_GLU_BWD) put4(static_cast<float*>(e.out2) + m * e.ldo + n, second, p.N - n);
            continue;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t n = n0 + h * 64 + tx * 4;
            if (n >= p.N) continue;
            float* v = z + 4 * h;
            if (e.kind != E_STORE) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (n + j >= p.N) continue;
                    if (e.bias.p) v[j] += side_at<float>(e.bias, 0, n + j);
                    const float s = e.scale.p ? side_at<float>(e.scale, 0, n + j) : 1.f;
                    const float g = e.res.p ? side_at<float>(e.res, m, n + j) : 0.f;
                    if (e.kind == E_LINEAR) {
                        v[j] = act_f(v[j], e.act);
                        if (e.scale.p) v[j] *= s;
                        if (e.res.p) v[j] += g;
                    } else {
                        float y, d;
                        act_grad_f(v[j], e.act, y, d);
                        v[j] = g * d;
                        if (e.scale.p) v[j] *= s;
                        sum_b[(i >> 2) * 8 + 4 * h + j] += v[j], sum_s[(i >> 2) * 8 + 4 * h + j] += g * y;
                    }
                }
            }
            float* out = splits > 1 ? partial + ((int64_t)blockIdx.y * rows_out + m + pair * p.M) * ldp
                                    : static_cast<float*>(pair ? e.out2 : e.out) + m * e.ldo;
            put4(out + n, v, p.N - n);
        }
    }
    if (e.kind != E_LINEAR_BWD || !(e.part_bias || e.part_scale)) return;
    // column sums of TC_ROWS rows: each thread's, then those of the block's 8 thread rows, in order
    float* red = As[0];  // [16][128], free after the last barrier
#pragma unroll
    for (int which = 0; which < 4; ++which) {
        float* dst = which & 1 ? e.part_scale : e.part_bias;
        const int half = which >> 1, q0 = (tid >> 7) * 8;
        const int64_t block = tm * (BM / TC_ROWS) + half * 2 + (tid >> 7), n = n0 + (tid & 127);
        if (!dst) continue;  // (the CTA's threads alike)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            red[ty * 128 + (j >> 2) * 64 + tx * 4 + (j & 3)] = which & 1 ? sum_s[half * 8 + j] : sum_b[half * 8 + j];
        __syncthreads();
        if (n < p.N && block * TC_ROWS < p.M) {
            float s = 0.f;
            for (int q = q0; q < q0 + 8; ++q) s += red[q * 128 + (tid & 127)];
            dst[block * p.N + n] = s;
        }
        __syncthreads();
    }
}

}  // namespace

// A plain product whose tiles do not fill the GPU splits its contraction,
// into parts of at least 128 indices; so does an epilogue's with few tiles and a long one, and
// the epilogue follows; that also keeps one chain of additions short.
Plan simt_plan(const Product& p) {
    Plan plan;
    const int64_t tiles = ceil_div(p.M, BM) * ceil_div(p.N, p.form == F_DUAL ? 64 : BN) * (p.form == F_PAIR ? 2 : 1);
    const int64_t k = p.K * (p.form == F_SUM ? 2 : 1), slots = PER_SM * (int64_t)sm_count();
    if (p.e.kind != E_STORE && (p.K < 1024 || 4 * tiles > slots)) return plan;
    int64_t n = slots / tiles;
    if (n > k / 128) n = k / 128;
    if (n > 16) n = 16;
    plan.splits = n > 1 ? (int)n : 1;
    plan.finish = p.e.kind != E_STORE && plan.splits > 1;
    return plan;
}

int simt_product(const Product& p, int splits, float* partial, int64_t ldp, cudaStream_t s) {
    const int64_t tn = ceil_div(p.N, p.form == F_DUAL ? 64 : BN), tm = ceil_div(p.M, BM);
    if (tm * tn > 0x7fffffff) return set_error(MABA_ERR_UNSUPPORTED, "dense: %lld tiles", (long long)(tm * tn));
    const dim3 grid((unsigned)(tm * tn), (unsigned)splits, p.form == F_PAIR ? 2 : 1);
    if (p.form == F_DUAL) simt_kernel<true><<<grid, NTHR, 0, s>>>(p, (int)tn, splits, partial, ldp);
    else simt_kernel<false><<<grid, NTHR, 0, s>>>(p, (int)tn, splits, partial, ldp);
    return check_launch("dense(simt)");
}

}  // namespace dense
}  // namespace maba
