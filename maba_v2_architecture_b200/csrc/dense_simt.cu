// Products on the CUDA cores: any type, any strides, float32 sums.
//
// A CTA computes a 128 x 128 tile of C (or 128 x 64 pairs of the gated block: the tile's
// columns 0..63 belong to B0, 64..127 to B1) over its share of the contraction, 16 indices
// at a time; both operand tiles are kept contraction-major in two shared-memory buffers and
// the next tile is loaded into registers under the current one's arithmetic.  A thread owns
// rows {4 ty, 64 + 4 ty} + 0..3 and columns {4 tx, 64 + 4 tx} + 0..3, so gate and up of a
// pair sit in one thread.  A column's sum over a tile's rows (bias and scale gradients) is
// added in a fixed order: thread rows first, then the 16 thread rows of the CTA.
#include "dense.cuh"

namespace maba {
namespace dense {
namespace {

constexpr int BM = SIMT_ROWS, BN = 128, BK = 16, LD = BM + 4, NTHR = 256;

struct Tile {  // one operand tile in flight: rows [r0, r0 + 128) x contraction [k0, k0 + 16)
    float v[8];
};

// The 8 elements of thread tid; out-of-range elements are 0.  vec: float rows, unit
// contraction stride and 16-byte alignment; otherwise the unit-stride axis (if any) runs
// along the threads.
template <typename T>
__device__ __forceinline__ void load_tile(Tile& t, const T* p, int64_t sr, int64_t sk, int64_t r0, int64_t rows,
                                          int64_t k0, int64_t K, bool vec, int tid) {
    if (sizeof(T) == 4 && vec && k0 + BK <= K) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = tid + i * NTHR;
            const int64_t r = r0 + (e >> 2);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) x = *reinterpret_cast<const float4*>(p + r * sr + k0 + (e & 3) * 4);
            t.v[4 * i] = x.x, t.v[4 * i + 1] = x.y, t.v[4 * i + 2] = x.z, t.v[4 * i + 3] = x.w;
        }
        return;
    }
    const bool kfast = sk == 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = tid + i * NTHR;
        const int64_t r = r0 + (kfast ? e / BK : e % BM), k = k0 + (kfast ? e % BK : e / BM);
        t.v[i] = r < rows && k < K ? Cvt<T>::to_f(p[r * sr + k * sk]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store_tile(const Tile& t, float* s, int64_t sk, int64_t k0, int64_t K, bool vec, int tid) {
    if (sizeof(T) == 4 && vec && k0 + BK <= K) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = tid + i * NTHR;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[((e & 3) * 4 + j) * LD + (e >> 2)] = t.v[4 * i + j];
        }
        return;
    }
    const bool kfast = sk == 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = tid + i * NTHR;
        if (kfast) s[(e % BK) * LD + e / BK] = t.v[i];
        else s[(e / BM) * LD + e % BM] = t.v[i];
    }
}

template <typename T> __device__ __forceinline__ bool vec_ok(const Matrix& m) {
    return sizeof(T) == 4 && m.sk == 1 && (m.sr & 3) == 0 && (reinterpret_cast<uintptr_t>(m.p) & 15u) == 0;
}

template <typename T>
__global__ void __launch_bounds__(NTHR) simt_kernel(const Product p, int tiles_n, int splits, float* partial, int64_t ldp) {
    __shared__ float As[2][BK * LD], Bs[2][BK * LD];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const bool dual = p.form == F_DUAL;
    const int bn = dual ? 64 : BN;
    const int64_t tm = blockIdx.x / tiles_n, m0 = tm * BM;
    const int64_t n0 = (int64_t)(blockIdx.x % tiles_n) * bn;
    const int pair = p.form == F_PAIR ? blockIdx.z : 0;
    const int nseg = p.form == F_SUM ? 2 : 1;
    const int64_t nk = (p.K + BK - 1) / BK, total = nk * nseg;
    const int64_t k_lo = total * blockIdx.y / splits, k_hi = total * (blockIdx.y + 1) / splits;

    float acc[8][8] = {};
    Tile ta, tb;
    const bool va0 = vec_ok<T>(p.a[0]), va1 = vec_ok<T>(p.a[1]), vb0 = vec_ok<T>(p.b[0]), vb1 = vec_ok<T>(p.b[1]);
    auto seg_of = [&](int64_t it) { return it >= nk ? 1 : 0; };
    auto load = [&](int64_t it) {
        const int sg = seg_of(it), ia = p.form == F_PAIR ? pair : sg;
        const int64_t k0 = (it - sg * nk) * BK;
        const Matrix& A = p.a[ia];
        load_tile<T>(ta, static_cast<const T*>(A.p), A.sr, A.sk, m0, p.M, k0, p.K, ia ? va1 : va0, tid);
        if (!dual) {
            const Matrix& B = p.b[sg];
            load_tile<T>(tb, static_cast<const T*>(B.p), B.sr, B.sk, n0, p.N, k0, p.K, sg ? vb1 : vb0, tid);
        } else {
            // rows 0..63 of the tile from B0, 64..127 from B1 (both laid out alike)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = tid + i * NTHR;
                const bool kfast = p.b[0].sk == 1;
                const int rr = kfast ? e / BK : e % BM;
                const Matrix& B = p.b[rr >> 6];
                const int64_t r = n0 + (rr & 63), k = k0 + (kfast ? e % BK : e / BM);
                tb.v[i] = r < p.N && k < p.K ? Cvt<T>::to_f(static_cast<const T*>(B.p)[r * B.sr + k * B.sk]) : 0.f;
            }
        }
    };
    auto store = [&](int64_t it, int buf) {
        const int sg = seg_of(it), ia = p.form == F_PAIR ? pair : sg;
        const int64_t k0 = (it - sg * nk) * BK;
        store_tile<T>(ta, As[buf], p.a[ia].sk, k0, p.K, ia ? va1 : va0, tid);
        store_tile<T>(tb, Bs[buf], p.b[dual ? 0 : sg].sk, k0, p.K, !dual && (sg ? vb1 : vb0), tid);
    };
    if (k_lo < k_hi) {
        load(k_lo);
        store(k_lo, 0);
    }
    __syncthreads();
    for (int64_t it = k_lo; it < k_hi; ++it) {
        const int buf = (int)(it - k_lo) & 1;
        if (it + 1 < k_hi) load(it + 1);
#pragma unroll
        for (int k = 0; k < BK; ++k) {
            float a[8], b[8];
            *reinterpret_cast<float4*>(a) = *reinterpret_cast<const float4*>(&As[buf][k * LD + ty * 4]);
            *reinterpret_cast<float4*>(a + 4) = *reinterpret_cast<const float4*>(&As[buf][k * LD + 64 + ty * 4]);
            *reinterpret_cast<float4*>(b) = *reinterpret_cast<const float4*>(&Bs[buf][k * LD + tx * 4]);
            *reinterpret_cast<float4*>(b + 4) = *reinterpret_cast<const float4*>(&Bs[buf][k * LD + 64 + tx * 4]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        if (it + 1 < k_hi) store(it + 1, buf ^ 1);
        __syncthreads();
    }

    const Epilogue& e = p.e;
    const int64_t rows_out = p.form == F_PAIR ? 2 * p.M : p.M;
    float sum_b[8] = {}, sum_s[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t m = m0 + (i >> 2) * 64 + ty * 4 + (i & 3);
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t n = n0 + (dual ? tx * 4 + (j & 3) : (j >> 2) * 64 + tx * 4 + (j & 3));
            if (dual && j >= 4) continue;
            float z = acc[i][j];
            T* out = static_cast<T*>(e.out) + m * e.ldo + n;
            float* outf = static_cast<float*>(e.out) + m * e.ldo + n;
            if (e.kind == E_STORE) {
                if (n >= p.N) continue;
                const int64_t mo = m + pair * p.M;
                if (splits > 1) partial[((int64_t)blockIdx.y * rows_out + mo) * ldp + n] = z;
                else static_cast<T*>(pair ? e.out2 : e.out)[m * e.ldo + n] = Cvt<T>::from_f(z);
            } else if (e.kind == E_LINEAR) {
                if (n >= p.N) continue;
                if (e.bias.p) z += side_at<T>(e.bias, 0, n);
                z = act_f(z, e.act);
                if (e.scale.p) z *= side_at<T>(e.scale, 0, n);
                if (e.res.p) z += side_at<T>(e.res, m, n);
                if (e.out_f32) *outf = z;
                else *out = Cvt<T>::from_f(z);
            } else if (e.kind == E_LINEAR_BWD) {
                if (n >= p.N) continue;
                if (e.bias.p) z += side_at<T>(e.bias, 0, n);
                const float g = side_at<T>(e.res, m, n);
                float y, d;
                act_grad_f(z, e.act, y, d);
                float dz = g * d;
                if (e.scale.p) dz *= side_at<T>(e.scale, 0, n);
                sum_b[j] += dz;
                sum_s[j] += g * y;
                *out = Cvt<T>::from_f(dz);
            } else {
                const float u = acc[i][j + 4 < 8 ? j + 4 : j];
                if (n >= p.N) continue;
                if (e.kind == E_GLU) {
                    *out = Cvt<T>::from_f(act_f(z, e.act) * u);
                } else {
                    const float da = side_at<T>(e.res, m, n);
                    float y, d;
                    act_grad_f(z, e.act, y, d);
                    *out = Cvt<T>::from_f(da * u * d);
                    static_cast<T*>(e.out2)[m * e.ldo + n] = Cvt<T>::from_f(da * y);
                }
            }
        }
    }
    if (e.kind == E_LINEAR_BWD && (e.part_bias || e.part_scale)) {
        float* red = As[0];  // [16][128], free after the last barrier
        for (int which = 0; which < 2; ++which) {
            float* dst = which ? e.part_scale : e.part_bias;
            if (!dst) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) red[ty * 128 + (j >> 2) * 64 + tx * 4 + (j & 3)] = which ? sum_s[j] : sum_b[j];
            __syncthreads();
            if (tid < 128 && n0 + tid < p.N) {
                float s = 0.f;
                for (int q = 0; q < 16; ++q) s += red[q * 128 + tid];
                dst[tm * p.N + n0 + tid] = s;
            }
            __syncthreads();
        }
    }
}

}  // namespace

template <typename T> int simt_product(const Product& p, int splits, float* partial, int64_t ldp, cudaStream_t s) {
    const int bn = p.form == F_DUAL ? 64 : BN;
    const int64_t tn = ceil_div(p.N, bn), tm = ceil_div(p.M, BM);
    if (tm * tn > 0x7fffffff) return set_error(MABA_ERR_UNSUPPORTED, "dense: %lld tiles", (long long)(tm * tn));
    dim3 grid((unsigned)(tm * tn), (unsigned)splits, p.form == F_PAIR ? 2 : 1);
    simt_kernel<T><<<grid, NTHR, 0, s>>>(p, (int)tn, splits, partial, ldp);
    return check_launch("dense(simt)");
}
template int simt_product<float>(const Product&, int, float*, int64_t, cudaStream_t);

}  // namespace dense
}  // namespace maba
