// C entries of the dense operators (maba_linear*, maba_gated_ffn*): argument checks, the
// products each one consists of, their workspace, and the small kernels between them
// (operand copies, sums of split contractions, column sums).
//
// A call first lays its workspace out with a Scratch; the *_workspace_size entries run the
// same code without launching, so size and use cannot differ.  Nothing is accumulated with
// atomics: results do not depend on the order in which CTAs run.
#include "dense.cuh"

namespace maba {
namespace dense {
namespace {

// Bump allocation over the caller's workspace; dry runs (base == nullptr) only add up.
struct Scratch {
    unsigned char* base = nullptr;
    size_t used = 0;
    void* take(size_t bytes) {
        void* p = base ? base + used : nullptr;
        used += (bytes + 255) & ~size_t(255);
        return p;
    }
};

struct Ctx {
    int dt;            // operand type
    bool dry;          // workspace query: no launches
    Scratch ws;
    cudaStream_t s;
};

inline size_t esize(int dt) { return dt == MABA_F32 ? 4 : 2; }

#define DENSE_DISPATCH(DT, ...)                                                  \
    [&]() -> int {                                                               \
        if ((DT) == MABA_F32) { using T = float; return __VA_ARGS__(); }         \
        if ((DT) == MABA_F16) { using T = __half; return __VA_ARGS__(); }        \
        using T = __nv_bfloat16;                                                 \
        return __VA_ARGS__();                                                    \
    }()

// ---------------------------------------------------------------------------
// small kernels
// ---------------------------------------------------------------------------
// dst [rows][ld] (T) = src (T or float32, any strides)
template <typename T>
__global__ void __launch_bounds__(256) copy_kernel(Side src, int64_t rows, int64_t cols, T* dst, int64_t ld) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cols, c = i - r * cols;
        dst[r * ld + c] = Cvt<T>::from_f(side_at<T>(src, r, c));
    }
}

// dst [3][rows][ld] (bf16) = x1, x2, x3 with x = x1 + x2 + x3: each the nearest bf16 of what
// the ones before left, so the three hold all 24 bits of x (the largest finite float32 would
// round to infinity: it is truncated).  An infinity or NaN is x1 alone.
__global__ void __launch_bounds__(256)
    planes_kernel(const float* __restrict__ src, int64_t sr, int64_t sc, int64_t rows, int64_t cols, __nv_bfloat16* dst,
                  int64_t ld, int64_t plane) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cols, c = i - r * cols;
        const float x = src[r * sr + c * sc];
        __nv_bfloat16 x1 = __float2bfloat16_rn(x), x2 = __float2bfloat16_rn(0.f), x3 = x2;
        if (isfinite(x)) {
            if (!isfinite(__bfloat162float(x1))) x1 = __float2bfloat16_rz(x);
            const float r1 = x - __bfloat162float(x1);
            x2 = __float2bfloat16_rn(r1);
            x3 = __float2bfloat16_rn(r1 - __bfloat162float(x2));
        }
        __nv_bfloat16* d = dst + r * ld + c;
        d[0] = x1, d[plane] = x2, d[2 * plane] = x3;
    }
}

// out = sum over splits of partial [splits][rows][ldp]; rows from `half` on go to out2
template <typename T>
__global__ void __launch_bounds__(256)
    sum_splits_kernel(const float* __restrict__ partial, int64_t ldp, int splits, int64_t rows, int64_t cols, T* out,
                      T* out2, int64_t half, int64_t ld) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cols, c = i - r * cols;
        float z = 0.f;
        for (int q = 0; q < splits; ++q) z += partial[(q * rows + r) * ldp + c];
        T* o = r < half ? out + r * ld : out2 + (r - half) * ld;
        o[c] = Cvt<T>::from_f(z);
    }
}

// part[blk][n] = sum of g over rows [128 blk, 128 blk + 128), added in row order
constexpr int CS_ROWS = 128;
template <typename T>
__global__ void __launch_bounds__(256) colsum_kernel(Side g, int64_t rows, int64_t cols, float* part) {
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int w = threadIdx.x >> 5;
    __shared__ float red[8][32];
    const int64_t r0 = (int64_t)blockIdx.y * CS_ROWS;
    float s = 0.f;
    if (c < cols)
        for (int64_t r = r0 + w; r < rows && r < r0 + CS_ROWS; r += 8) s += side_at<T>(g, r, c);
    red[w][threadIdx.x & 31] = s;
    __syncthreads();
    if (w == 0 && c < cols) {
        float t = 0.f;
        for (int q = 0; q < 8; ++q) t += red[q][threadIdx.x];
        part[(int64_t)blockIdx.y * cols + c] = t;
    }
}

// out[n] = sum over blocks of part [blocks][cols]
template <typename T>
__global__ void __launch_bounds__(256)
    colsum_finish_kernel(const float* __restrict__ part, int64_t blocks, int64_t cols, void* out, int64_t so, int out_f32) {
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int w = threadIdx.x >> 5;
    __shared__ float red[8][32];
    float s = 0.f;
    if (c < cols)
        for (int64_t b = w; b < blocks; b += 8) s += part[b * cols + c];
    red[w][threadIdx.x & 31] = s;
    __syncthreads();
    if (w == 0 && c < cols) {
        float t = 0.f;
        for (int q = 0; q < 8; ++q) t += red[q][threadIdx.x];
        if (out_f32) static_cast<float*>(out)[c * so] = t;
        else static_cast<T*>(out)[c * so] = Cvt<T>::from_f(t);
    }
}

inline unsigned grid1d(int64_t n) {
    const int64_t g = ceil_div(n, 256), cap = 8 * (int64_t)sm_count();
    return (unsigned)(g < cap ? (g > 0 ? g : 1) : cap);
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
int run(Ctx& c, const Product& p) {
    if (skinny_takes(p, c.dt)) {
        if (c.dry) return MABA_OK;
        return DENSE_DISPATCH(c.dt, [&] { return skinny_product<T>(p, c.s); });
    }
    // a plain product whose tiles do not fill the GPU splits its contraction; the partial
    // sums are float32 and added in split order
    const int splits = tc_splits(p, c.dt);
    const int64_t rows = p.form == F_PAIR ? 2 * p.M : p.M, ldp = (p.N + 3) / 4 * 4;
    float* partial = splits > 1 ? static_cast<float*>(c.ws.take((size_t)splits * rows * ldp * 4)) : nullptr;
    if (c.dry) return MABA_OK;
    return DENSE_DISPATCH(c.dt, [&] {
        MABA_TRY(tc_product<T>(p, partial, ldp, c.s));
        if (splits == 1) return (int)MABA_OK;
        sum_splits_kernel<T><<<grid1d(rows * p.N), 256, 0, c.s>>>(partial, ldp, splits, rows, p.N, static_cast<T*>(p.e.out),
                                                                  static_cast<T*>(p.e.out2), p.M, p.e.ldo);
        return check_launch("dense(split sums)");
    });
}

int copy_matrix(Ctx& c, const Side& src, int64_t rows, int64_t cols, void* dst, int64_t ld) {
    if (c.dry) return MABA_OK;
    return DENSE_DISPATCH(c.dt, [&] {
        copy_kernel<T><<<grid1d(rows * cols), 256, 0, c.s>>>(src, rows, cols, static_cast<T*>(dst), ld);
        return check_launch("dense(copy)");
    });
}

int column_sums(Ctx& c, const Side& g, int64_t rows, int64_t cols, float* part) {
    if (c.dry) return MABA_OK;
    return DENSE_DISPATCH(c.dt, [&] {
        const dim3 grid((unsigned)ceil_div(cols, 32), (unsigned)ceil_div(rows, CS_ROWS));
        colsum_kernel<T><<<grid, 256, 0, c.s>>>(g, rows, cols, part);
        return check_launch("dense(column sums)");
    });
}

int finish_columns(Ctx& c, const float* part, int64_t blocks, int64_t cols, const maba_tensor* out) {
    if (c.dry) return MABA_OK;
    return DENSE_DISPATCH(c.dt, [&] {
        colsum_finish_kernel<T><<<(unsigned)ceil_div(cols, 32), 256, 0, c.s>>>(part, blocks, cols, out->data,
                                                                               out->stride[0], out->dtype == MABA_F32);
        return check_launch("dense(column sums)");
    });
}

// ---------------------------------------------------------------------------
// argument checks
// ---------------------------------------------------------------------------
bool given(const maba_tensor* t) { return t != nullptr && t->ndim > 0; }

int want_matrix(const maba_tensor* t, const char* name, int64_t rows, int64_t cols, int dt, bool f32_ok, bool dense_rows) {
    if (!given(t)) return set_error(MABA_ERR_INVALID, "%s: tensor is required", name);
    if (t->ndim != 2) return set_error(MABA_ERR_INVALID, "%s: expected 2 dims, got %d", name, t->ndim);
    if ((rows >= 0 && t->shape[0] != rows) || (cols >= 0 && t->shape[1] != cols))
        return set_error(MABA_ERR_INVALID, "%s: shape [%lld, %lld], expected [%lld, %lld]", name, (long long)t->shape[0],
                         (long long)t->shape[1], (long long)rows, (long long)cols);
    if (t->dtype != dt && !(f32_ok && t->dtype == MABA_F32))
        return set_error(MABA_ERR_DTYPE, "%s: dtype %s, expected %s%s", name, dtype_name(t->dtype), dtype_name(dt),
                         f32_ok ? " or float32" : "");
    if (t->stride[0] < 0 || t->stride[1] < 0) return set_error(MABA_ERR_INVALID, "%s: negative stride", name);
    if (dense_rows && t->shape[0] > 0 &&
        ((t->stride[1] != 1 && t->shape[1] > 1) || (t->shape[0] > 1 && t->stride[0] < t->shape[1])))
        return set_error(MABA_ERR_INVALID, "%s: rows must have unit stride and not overlap", name);
    if (t->data == nullptr && t->shape[0] > 0 && t->shape[1] > 0)
        return set_error(MABA_ERR_INVALID, "%s: no data", name);
    return MABA_OK;
}

int want_vector(const maba_tensor* t, const char* name, int64_t n, int dt) {
    if (t->ndim != 1 || t->shape[0] != n || t->data == nullptr)
        return set_error(MABA_ERR_INVALID, "%s: expected [%lld]", name, (long long)n);
    if (t->dtype != dt && t->dtype != MABA_F32)
        return set_error(MABA_ERR_DTYPE, "%s: dtype %s, expected %s or float32", name, dtype_name(t->dtype), dtype_name(dt));
    if (t->stride[0] < 0) return set_error(MABA_ERR_INVALID, "%s: negative stride", name);
    return MABA_OK;
}

int want_operands(const maba_tensor* x, const maba_tensor* w, const char* wname, int act, int act_min) {
    if (!given(x)) return set_error(MABA_ERR_INVALID, "x: tensor is required");
    if (x->dtype != MABA_F32 && x->dtype != MABA_F16 && x->dtype != MABA_BF16)
        return set_error(MABA_ERR_DTYPE, "x: dtype %s, expected float32, float16 or bfloat16", dtype_name(x->dtype));
    if (act < act_min || act > ACT_GELU) return set_error(MABA_ERR_INVALID, "activation %d", act);
    MABA_TRY(want_matrix(x, "x", -1, -1, x->dtype, false, false));
    MABA_TRY(want_matrix(w, wname, -1, x->shape[1], x->dtype, false, false));
    if (x->shape[1] <= 0 || w->shape[0] <= 0)
        return set_error(MABA_ERR_INVALID, "%s: [%lld, %lld] has no features", wname, (long long)w->shape[0],
                         (long long)x->shape[1]);
    // coordinates of the tensor-memory loads and tile counts are 32-bit
    const int64_t lim = int64_t(1) << 31;
    if (x->shape[0] >= lim || x->shape[1] >= lim || w->shape[0] >= lim)
        return set_error(MABA_ERR_UNSUPPORTED, "sizes of 2^31 or more");
    return MABA_OK;
}

Side side2(const maba_tensor* t) {
    return given(t) ? Side{t->data, t->stride[0], t->stride[1], t->dtype == MABA_F32} : Side{};
}
Side side1(const maba_tensor* t) { return given(t) ? Side{t->data, 0, t->stride[0], t->dtype == MABA_F32} : Side{}; }

// ---------------------------------------------------------------------------
// the operators
// ---------------------------------------------------------------------------
// A matrix as an operand.  The tensor-memory loads of the 16-bit products want rows on
// 16-byte boundaries; what is not laid out so is copied once per call, and a float32 matrix
// is split into its planes.  One copy serves both directions of a matrix: K-major along its
// rows, MN-major across them.
int operand(Ctx& c, const Side& t, int64_t rows, int64_t cols, Matrix& m) {
    m = Matrix{t.p, t.sr, t.sc, 0};
    if (!t.f32 && tc_readable(t.p, rows, cols, t.sr, t.sc)) return MABA_OK;
    const int64_t ld = (cols + 7) / 8 * 8, plane = rows * ld;
    void* to = c.ws.take((size_t)(c.dt == MABA_F32 ? 3 : 1) * plane * 2);
    m = Matrix{to, ld, 1, plane};
    if (c.dt != MABA_F32) return copy_matrix(c, t, rows, cols, to, ld);
    if (c.dry) return MABA_OK;
    planes_kernel<<<grid1d(rows * cols), 256, 0, c.s>>>(static_cast<const float*>(t.p), t.sr, t.sc, rows, cols,
                                                        static_cast<__nv_bfloat16*>(to), ld, plane);
    return check_launch("dense(planes)");
}
int operand(Ctx& c, const maba_tensor* t, Matrix& m, bool as_is = false) {
    m = Matrix{t->data, t->stride[0], t->stride[1], 0};
    return as_is ? (int)MABA_OK : operand(c, side2(t), t->shape[0], t->shape[1], m);
}
// What an epilogue of this call wrote, [rows][ld] in the operands' type.
int own_operand(Ctx& c, void* p, int64_t ld, int64_t rows, int64_t cols, Matrix& m) {
    return operand(c, Side{p, ld, 1, c.dt == MABA_F32}, rows, cols, m);
}
Matrix transposed(const Matrix& m) { return Matrix{m.p, m.sk, m.sr, m.sp}; }

struct LinearArgs {
    const maba_tensor *x, *w, *bias, *scale, *res, *out;              // forward
    const maba_tensor *g, *dx, *dw, *dbias, *dscale;                  // backward
    int act;
};

int linear_forward(Ctx& c, const LinearArgs& a) {
    Product p;
    p.M = a.x->shape[0], p.K = a.x->shape[1], p.N = a.w->shape[0];
    if (p.M == 0) return MABA_OK;
    p.e.kind = E_LINEAR;
    const bool as_is = skinny_takes(p, c.dt);
    MABA_TRY(operand(c, a.x, p.a[0], as_is));
    MABA_TRY(operand(c, a.w, p.b[0], as_is));
    p.e.act = a.act;
    p.e.bias = side1(a.bias), p.e.scale = side1(a.scale), p.e.res = side2(a.res);
    if (a.out) p.e.out = a.out->data, p.e.ldo = a.out->stride[0], p.e.out_f32 = a.out->dtype == MABA_F32;
    return run(c, p);
}

int zero_rows(Ctx& c, const maba_tensor* t) {
    if (c.dry || !given(t) || t->data == nullptr) return MABA_OK;
    const size_t es = t->dtype == MABA_F32 ? 4 : 2;
    const bool mat = t->ndim == 2;
    const int64_t rows = t->shape[0], cols = mat ? t->shape[1] : 1;
    const cudaError_t e = cudaMemset2DAsync(t->data, (size_t)(rows > 1 ? t->stride[0] : cols) * es, 0, (size_t)cols * es,
                                            (size_t)rows, c.s);
    return e == cudaSuccess ? MABA_OK : set_error(MABA_ERR_CUDA, "dense(zero): %s", cudaGetErrorString(e));
}

// dx = sum of d_i W_i and dW_i = d_i^T x for one or two (d, W)
int dx_product(Ctx& c, int64_t M, int64_t N, int n, const Matrix* d, const Matrix* w, const maba_tensor* dx) {
    Product p;
    p.form = n == 2 ? F_SUM : F_SINGLE;
    p.M = M, p.N = dx->shape[1], p.K = N;
    for (int i = 0; i < n; ++i) p.a[i] = d[i], p.b[i] = transposed(w[i]);
    p.e.out = dx->data, p.e.ldo = dx->stride[0];
    return run(c, p);
}
int dw_product(Ctx& c, int64_t M, int n, const Matrix* d, const Matrix& x, const maba_tensor* const* dw) {
    Product p;
    p.form = n == 2 ? F_PAIR : F_SINGLE;
    p.M = dw[0]->shape[0], p.N = dw[0]->shape[1], p.K = M;
    for (int i = 0; i < n; ++i) p.a[i] = transposed(d[i]);
    p.b[0] = transposed(x);
    p.a_mn = true;
    p.e.out = dw[0]->data, p.e.ldo = dw[0]->stride[0];
    if (n == 2) p.e.out2 = dw[1]->data;
    return run(c, p);
}

int linear_backward(Ctx& c, const LinearArgs& a) {
    const int64_t M = a.x->shape[0], K = a.x->shape[1], N = a.w->shape[0];
    const bool need_dx = given(a.dx), need_dw = given(a.dw), need_db = given(a.dbias), need_ds = given(a.dscale);
    if (M == 0) {  // sums over no rows
        MABA_TRY(zero_rows(c, a.dw));
        MABA_TRY(zero_rows(c, a.dbias));
        return zero_rows(c, a.dscale);
    }
    if (!need_dx && !need_dw && !need_db && !need_ds) return MABA_OK;
    const bool through = a.act == ACT_NONE && !given(a.scale);  // dz = g
    const int64_t blocks = ceil_div(M, through ? CS_ROWS : TC_ROWS);
    float* pb = need_db ? static_cast<float*>(c.ws.take((size_t)blocks * N * 4)) : nullptr;
    float* ps = need_ds ? static_cast<float*>(c.ws.take((size_t)blocks * N * 4)) : nullptr;
    Matrix x, w, d;
    if (!through || need_dw) MABA_TRY(operand(c, a.x, x));
    if (!through || need_dx) MABA_TRY(operand(c, a.w, w));
    if (!through) {
        // z again, rather than a copy kept by the forward pass: a 16-bit z would add its own
        // rounding to phi'(z), and a float32 one costs more traffic than the product
        const int64_t ld = (N + 7) / 8 * 8;
        Product p;
        p.M = M, p.N = N, p.K = K;
        p.a[0] = x, p.b[0] = w;
        p.e.kind = E_LINEAR_BWD;
        p.e.act = a.act;
        p.e.bias = side1(a.bias), p.e.scale = side1(a.scale), p.e.res = side2(a.g);
        p.e.out = c.ws.take((size_t)M * ld * esize(c.dt)), p.e.ldo = ld;
        p.e.part_bias = pb, p.e.part_scale = ps;
        MABA_TRY(run(c, p));
        if (need_dx || need_dw) MABA_TRY(own_operand(c, p.e.out, ld, M, N, d));
    } else {
        if (need_db) MABA_TRY(column_sums(c, side2(a.g), M, N, pb));
        // the products take one type: a float32 gradient is rounded to x's here
        if (need_dx || need_dw) MABA_TRY(operand(c, a.g, d));
    }
    if (need_db) MABA_TRY(finish_columns(c, pb, blocks, N, a.dbias));
    if (need_ds) MABA_TRY(finish_columns(c, ps, blocks, N, a.dscale));
    if (need_dx) MABA_TRY(dx_product(c, M, N, 1, &d, &w, a.dx));
    if (need_dw) MABA_TRY(dw_product(c, M, 1, &d, x, &a.dw));
    return MABA_OK;
}

struct FfnArgs {
    const maba_tensor *x, *wg, *wu, *out;   // forward
    const maba_tensor *g, *dx, *dwg, *dwu;  // backward
    int act;
};

int ffn_product(Ctx& c, const FfnArgs& a, Product& p) {
    p.form = F_DUAL;
    p.M = a.x->shape[0], p.K = a.x->shape[1], p.N = a.wg->shape[0];
    p.e.act = a.act;
    p.e.kind = given(a.g) ? E_GLU_BWD : E_GLU;
    if (p.M == 0) return MABA_OK;
    const bool as_is = skinny_takes(p, c.dt);
    MABA_TRY(operand(c, a.x, p.a[0], as_is));
    MABA_TRY(operand(c, a.wg, p.b[0], as_is));
    return operand(c, a.wu, p.b[1], as_is);
}

int ffn_forward(Ctx& c, const FfnArgs& a) {
    Product p;
    MABA_TRY(ffn_product(c, a, p));
    if (p.M == 0) return MABA_OK;
    if (a.out) p.e.out = a.out->data, p.e.ldo = a.out->stride[0];
    return run(c, p);
}

int ffn_backward(Ctx& c, const FfnArgs& a) {
    const int64_t M = a.x->shape[0];
    if (M == 0) {
        MABA_TRY(zero_rows(c, a.dwg));
        return zero_rows(c, a.dwu);
    }
    if (!given(a.dx) && !given(a.dwg) && !given(a.dwu)) return MABA_OK;
    Product p;
    MABA_TRY(ffn_product(c, a, p));
    const int64_t ld = (p.N + 7) / 8 * 8;
    // dg and du in the operands' type: the matrix units multiply 16-bit operands, so this is
    // the one rounding between the two passes
    p.e.res = side2(a.g);
    p.e.out = c.ws.take((size_t)M * ld * esize(c.dt)), p.e.ldo = ld;
    p.e.out2 = c.ws.take((size_t)M * ld * esize(c.dt));
    MABA_TRY(run(c, p));
    Matrix d[2];
    MABA_TRY(own_operand(c, p.e.out, ld, M, p.N, d[0]));
    MABA_TRY(own_operand(c, p.e.out2, ld, M, p.N, d[1]));
    if (given(a.dx)) MABA_TRY(dx_product(c, M, p.N, 2, d, p.b, a.dx));
    const maba_tensor* dw[2] = {a.dwg, a.dwu};
    if (given(a.dwg) && given(a.dwu) && a.dwg->stride[0] == a.dwu->stride[0])
        return dw_product(c, M, 2, d, p.a[0], dw);
    for (int i = 0; i < 2; ++i)
        if (given(dw[i])) MABA_TRY(dw_product(c, M, 1, d + i, p.a[0], dw + i));
    return MABA_OK;
}

int check_linear(const LinearArgs& a, bool backward) {
    MABA_TRY(want_operands(a.x, a.w, "weight", a.act, ACT_NONE));
    const int dt = a.x->dtype;
    const int64_t M = a.x->shape[0], K = a.x->shape[1], N = a.w->shape[0];
    if (given(a.bias)) MABA_TRY(want_vector(a.bias, "bias", N, dt));
    if (given(a.scale)) MABA_TRY(want_vector(a.scale, "scale", N, dt));
    if (!backward) {
        if (given(a.res)) MABA_TRY(want_matrix(a.res, "residual", M, N, dt, true, false));
        return want_matrix(a.out, "out", M, N, dt, true, true);
    }
    MABA_TRY(want_matrix(a.g, "grad", M, N, dt, true, false));
    if (given(a.dx)) MABA_TRY(want_matrix(a.dx, "dx", M, K, dt, false, true));
    if (given(a.dw)) MABA_TRY(want_matrix(a.dw, "dw", N, K, dt, false, true));
    if (given(a.dbias)) {
        MABA_TRY(want_vector(a.dbias, "dbias", N, dt));
        if (!given(a.bias)) return set_error(MABA_ERR_INVALID, "dbias without bias");
    }
    if (given(a.dscale)) {
        MABA_TRY(want_vector(a.dscale, "dscale", N, dt));
        if (!given(a.scale)) return set_error(MABA_ERR_INVALID, "dscale without scale");
    }
    return MABA_OK;
}

int check_ffn(const FfnArgs& a, bool backward) {
    MABA_TRY(want_operands(a.x, a.wg, "w_gate", a.act, ACT_RELU));
    const int dt = a.x->dtype;
    const int64_t M = a.x->shape[0], K = a.x->shape[1], N = a.wg->shape[0];
    MABA_TRY(want_matrix(a.wu, "w_up", N, K, dt, false, false));
    if (!backward) return want_matrix(a.out, "out", M, N, dt, false, true);
    MABA_TRY(want_matrix(a.g, "grad", M, N, dt, false, false));
    if (given(a.dx)) MABA_TRY(want_matrix(a.dx, "dx", M, K, dt, false, true));
    if (given(a.dwg)) MABA_TRY(want_matrix(a.dwg, "dw_gate", N, K, dt, false, true));
    if (given(a.dwu)) MABA_TRY(want_matrix(a.dwu, "dw_up", N, K, dt, false, true));
    return MABA_OK;
}

template <typename Args, typename F> size_t query(const Args& a, F op) {
    Ctx c{a.x->dtype, true, {}, nullptr};
    return op(c, a) == MABA_OK ? c.ws.used : 0;
}

template <typename Args, typename F>
int execute(const Args& a, F op, const char* name, void* workspace, size_t bytes, void* stream) {
    const size_t need = query(a, op);
    if (need > 0 && (workspace == nullptr || bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))
        return set_error(MABA_ERR_WORKSPACE, "%s: needs a 256-byte aligned workspace of %zu bytes, got %zu", name, need, bytes);
    Ctx c{a.x->dtype, false, {static_cast<unsigned char*>(workspace), 0}, as_stream(stream)};
    return op(c, a);
}

}  // namespace
}  // namespace dense
}  // namespace maba

using namespace maba;
using namespace maba::dense;

extern "C" int maba_linear(const maba_tensor* x, const maba_tensor* weight, const maba_tensor* bias, int32_t activation,
                           const maba_tensor* scale, const maba_tensor* residual, const maba_tensor* out, void* workspace,
                           size_t workspace_bytes, void* stream) {
    LinearArgs a{};
    a.x = x, a.w = weight, a.bias = bias, a.scale = scale, a.res = residual, a.out = out, a.act = activation;
    MABA_TRY(check_linear(a, false));
    return execute(a, linear_forward, "linear", workspace, workspace_bytes, stream);
}

extern "C" size_t maba_linear_workspace_size(const maba_tensor* x, const maba_tensor* weight, const maba_tensor* out) {
    LinearArgs a{};
    a.x = x, a.w = weight, a.out = out;
    if (check_linear(a, false) != MABA_OK) return 0;
    return query(a, linear_forward);
}

extern "C" int maba_linear_backward(const maba_tensor* grad, const maba_tensor* x, const maba_tensor* weight,
                                    const maba_tensor* bias, int32_t activation, const maba_tensor* scale,
                                    const maba_tensor* dx, const maba_tensor* dw, const maba_tensor* dbias,
                                    const maba_tensor* dscale, void* workspace, size_t workspace_bytes, void* stream) {
    LinearArgs a{};
    a.g = grad, a.x = x, a.w = weight, a.bias = bias, a.scale = scale, a.act = activation;
    a.dx = dx, a.dw = dw, a.dbias = dbias, a.dscale = dscale;
    MABA_TRY(check_linear(a, true));
    return execute(a, linear_backward, "linear_backward", workspace, workspace_bytes, stream);
}

extern "C" size_t maba_linear_backward_workspace_size(const maba_tensor* grad, const maba_tensor* x,
                                                      const maba_tensor* weight, const maba_tensor* bias,
                                                      int32_t activation, const maba_tensor* scale, const maba_tensor* dx,
                                                      const maba_tensor* dw, const maba_tensor* dbias,
                                                      const maba_tensor* dscale) {
    LinearArgs a{};
    a.g = grad, a.x = x, a.w = weight, a.bias = bias, a.scale = scale, a.act = activation;
    a.dx = dx, a.dw = dw, a.dbias = dbias, a.dscale = dscale;
    if (check_linear(a, true) != MABA_OK) return 0;
    return query(a, linear_backward);
}

extern "C" int maba_gated_ffn(const maba_tensor* x, const maba_tensor* w_gate, const maba_tensor* w_up, int32_t activation,
                              const maba_tensor* out, void* workspace, size_t workspace_bytes, void* stream) {
    FfnArgs a{};
    a.x = x, a.wg = w_gate, a.wu = w_up, a.out = out, a.act = activation;
    MABA_TRY(check_ffn(a, false));
    return execute(a, ffn_forward, "gated_ffn", workspace, workspace_bytes, stream);
}

extern "C" size_t maba_gated_ffn_workspace_size(const maba_tensor* x, const maba_tensor* w_gate, const maba_tensor* w_up,
                                                const maba_tensor* out) {
    FfnArgs a{};
    a.x = x, a.wg = w_gate, a.wu = w_up, a.out = out, a.act = ACT_SILU;
    if (check_ffn(a, false) != MABA_OK) return 0;
    return query(a, ffn_forward);
}

extern "C" int maba_gated_ffn_backward(const maba_tensor* grad, const maba_tensor* x, const maba_tensor* w_gate,
                                       const maba_tensor* w_up, int32_t activation, const maba_tensor* dx,
                                       const maba_tensor* dw_gate, const maba_tensor* dw_up, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    FfnArgs a{};
    a.g = grad, a.x = x, a.wg = w_gate, a.wu = w_up, a.act = activation, a.dx = dx, a.dwg = dw_gate, a.dwu = dw_up;
    MABA_TRY(check_ffn(a, true));
    return execute(a, ffn_backward, "gated_ffn_backward", workspace, workspace_bytes, stream);
}

extern "C" size_t maba_gated_ffn_backward_workspace_size(const maba_tensor* grad, const maba_tensor* x,
                                                         const maba_tensor* w_gate, const maba_tensor* w_up,
                                                         const maba_tensor* dx, const maba_tensor* dw_gate,
                                                         const maba_tensor* dw_up) {
    FfnArgs a{};
    a.g = grad, a.x = x, a.wg = w_gate, a.wu = w_up, a.act = ACT_SILU, a.dx = dx, a.dwg = dw_gate, a.dwu = dw_up;
    if (check_ffn(a, true) != MABA_OK) return 0;
    return query(a, ffn_backward);
}
