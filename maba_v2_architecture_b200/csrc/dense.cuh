// Dense products of the model's blocks: the linear map with its epilogue and the
// gated feed-forward block, forward and backward.
//
//   linear   z = x W^T + b,  out = r + s * phi(z)
//            dz = g * s * phi'(z);  dx = dz W;  dW = dz^T x;  db = sum_m dz;  ds = sum_m g * phi(z)
//   ffn      a = phi(x Wg^T) * (x Wu^T)
//            dg = da * u * phi'(g);  du = da * phi(g);  dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x
//
// Every product of both operators is one Product: C[M,N] = A B^T summed in float32 over
// the contraction index, with an epilogue on the float32 sums.
#pragma once
#include "common.cuh"

namespace maba {
namespace dense {

enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

// What a Product's operands form.
enum Form {
    F_SINGLE = 0,  // C = A0 B0^T
    F_DUAL = 1,    // two products of one A: columns j of B0 and of B1 meet in the epilogue
    F_SUM = 2,     // C = A0 B0^T + A1 B1^T
    F_PAIR = 3,    // C0 = A0 B0^T and C1 = A1 B1^T (epilogue E_STORE)
};

enum EpiKind {
    E_LINEAR = 0,      // out = res + scale * act(z + bias)
    E_LINEAR_BWD = 1,  // out = dz from g = res; column sums of dz and of g * act(z + bias) per row tile
    E_GLU = 2,         // out = act(z0) * z1
    E_GLU_BWD = 3,     // out = dg, out2 = du from da = res
    E_STORE = 4,       // out = z, or float32 partial sums [split][M (2 M of F_PAIR)][N]
};

// An operand of a Product, of the operands' type.
struct Matrix {
    const void* p = nullptr;
    int64_t sr = 0, sk = 0;  // element strides along the rows and along the contraction
};

// A vector or a matrix that an epilogue reads: float32 or the operands' type, any strides.
struct Side {
    const void* p = nullptr;
    int64_t sr = 0, sc = 0;
    int f32 = 0;
};

struct Epilogue {
    int kind = E_STORE, act = ACT_NONE, out_f32 = 0;
    void* out = nullptr;   // row-major, unit column stride
    void* out2 = nullptr;  // laid out like out: du of E_GLU_BWD, C1 of F_PAIR
    int64_t ldo = 0;
    Side bias, scale, res;
    float* part_bias = nullptr;   // E_LINEAR_BWD: [row blocks][N] column sums of dz
    float* part_scale = nullptr;  // and of g * act(z + bias)
    int sums_f32 = 0;             // they end in a float32 gradient
};

struct Product {
    int form = F_SINGLE;
    Matrix a[2], b[2];
    int64_t M = 0, N = 0, K = 0;
    bool a_mn = false, b_mn = false;  // E_STORE: an operand's rows, not its contraction, are contiguous
    Epilogue e;
};

// phi and phi' in float32, the exponential and erf CUDA's.  silu and its slope are within a few ulp of
// their own size down to z = -87, where 1 / (1 + e^-z) leaves float32's normal range (__expf's error
// grows with |z|: 27 ulp at -60).  gelu and its slope are off by about an ulp of |z| and of 1 + |z|: for
// z < 0 the sum 1 + erf cancels, and beside that __expf's error in the slope's second term is nothing.
__device__ __forceinline__ float act_f(float z, int act) {
    if (act == ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
    if (act == ACT_SILU) return __fdiv_rn(z, 1.f + expf(-z));
    if (act == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    return z;
}
// phi(z) and phi'(z) together
__device__ __forceinline__ void act_grad_f(float z, int act, float& y, float& d) {
    if (act == ACT_RELU) {
        y = z > 0.f ? z : (z != z ? z : 0.f);
        d = z > 0.f ? 1.f : 0.f;
    } else if (act == ACT_SILU) {
        const float s = __fdiv_rn(1.f, 1.f + expf(-z));
        y = z * s;
        d = s * (1.f + z * (1.f - s));
    } else if (act == ACT_GELU) {
        const float phi = 0.5f * (1.f + erff(z * 0.70710678118654752f));
        y = z * phi;
        d = phi + z * 0.39894228040143268f * __expf(-0.5f * z * z);
    } else {
        y = z;
        d = 1.f;
    }
}

template <typename T> __device__ __forceinline__ float side_at(const Side& s, int64_t r, int64_t c) {
    const int64_t i = r * s.sr + c * s.sc;
    return s.f32 ? static_cast<const float*>(s.p)[i] : Cvt<T>::to_f(static_cast<const T*>(s.p)[i]);
}

// Partial sums of a split product: float32 [split][rows][ldp], rows = M (2 M of F_PAIR).
inline int64_t partials_ld(int64_t cols) { return (cols + 3) / 4 * 4; }
inline int64_t partials_bytes(int64_t splits, int64_t rows, int64_t cols) { return splits * rows * partials_ld(cols) * 4; }

// dense_skinny.cu: forward products of few rows, any strides.
bool skinny_takes(const Product& p, int dt);
template <typename T> int skinny_product(const Product& p, cudaStream_t s);

// dense_tc.cu: 16-bit operands on the tensor cores, laid out as tc_readable() accepts them;
// column sums per TC_ROWS rows; T is their type.
constexpr int TC_ROWS = 32;
struct Plan {
    int cg = 1, bn = 32;  // CTAs per tile, columns of the MMA
    int splits = 1;       // of the contraction
    bool finish = false;  // the splits' sums get the epilogue in a kernel of its own (split_sums)
};
bool tc_readable(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t col_stride);
Plan tc_plan(const Product& p);
Product split_sums(const Product& p);  // the same sums as a plain product, two for F_DUAL
// End, in elements, of the partial sums [parts][rows][ldp] where the tensor-memory copies store them.
int64_t partials_reach(int64_t rows, int64_t cols, int64_t ldp, int64_t parts);
template <typename T>
int tc_product(const Product& p, const Plan& plan, float* partial, int64_t ldp, cudaStream_t s);
int device_error_take(cudaStream_t s, int* out);

// dense_simt.cu: float32 operands, any strides; column sums per TC_ROWS rows too.
Plan simt_plan(const Product& p);
int simt_product(const Product& p, int splits, float* partial, int64_t ldp, cudaStream_t s);

}  // namespace dense
}  // namespace maba
