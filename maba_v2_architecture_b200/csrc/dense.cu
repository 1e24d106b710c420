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


#define DENSE_DISPATCH16(DT, ...)                                                \
    [&]() -> int {                                                               \
        if ((DT) == MABA_F16) { using T = __half; return __VA_ARGS__(); }        \
        using T = __nv_bfloat16;                                                 \
        return __VA_ARGS__();                                                    \
    }()
#define DENSE_DISPATCH(DT, ...)                                                  \
    [&]() -> int {                                                               \
        if ((DT) == MABA_F32) { using T = float; return __VA_ARGS__(); }         \
        if ((DT) == MABA_F16) { using T = __half; return __VA_ARGS__(); }        \
        using T = __nv_bfloat16;                                                 \
        return __VA_ARGS__();                                                    \
    }()

template <typename... KArgs, typename... Args>
int launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args... args) {
    kern<<<grid, block, smem, s>>>(static_cast<KArgs>(args)...);
    return check_launch("dense");
}

// A grid's second dimension holds 65,535 blocks: the kernels that use it walk on by gridDim.y
unsigned grid_y(int64_t blocks) { return (unsigned)(blocks < 32768 ? blocks : 32768); }

// ---------------------------------------------------------------------------
// small kernels
// ---------------------------------------------------------------------------
// Matrices made readable for the tensor-memory copies, up to four in one launch: dst [rows][ld] of
// a 16-bit type = src (that type or float32, any strides), or float32 = float32.  Tiles of 32 x 64;
// where the source's columns are not contiguous they pass through shared memory, so that both
// sides run along their contiguous axis.
struct Job {
    Side src;
    int64_t rows = 0, cols = 0;
    void* dst = nullptr;
    int64_t ld = 0;
    int f32 = 0;  // a float32 copy
};
struct Jobs {
    Job j[4];
    int n = 0;
};
template <typename T> __device__ __forceinline__ void put_pair(const Job& b, int64_t at, float x, float y) {
    if (b.f32) {
        *reinterpret_cast<float2*>(static_cast<float*>(b.dst) + at) = make_float2(x, y);
        return;
    }
    const T v[2] = {Cvt<T>::from_f(x), Cvt<T>::from_f(y)};
    *reinterpret_cast<uint32_t*>(static_cast<T*>(b.dst) + at) = *reinterpret_cast<const uint32_t*>(v);
}
template <typename T> __global__ void __launch_bounds__(256) prepare_kernel(const Jobs jobs) {
    __shared__ float tile[32][65];
    const Job& b = jobs.j[blockIdx.y];
    const unsigned tiles_c = (unsigned)((b.cols + 63) / 64);
    const int64_t tiles = (b.rows + 31) / 32 * tiles_c;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t tr = tiles >> 32 ? t / tiles_c : (unsigned)t / tiles_c, r0 = tr * 32, c0 = (t - tr * tiles_c) * 64;
        const int64_t c = c0 + lane * 2, rw = r0 + w * 4;
        if (b.src.sc == 1) {
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = rw + i < b.rows && c < b.cols ? side_at<T>(b.src, rw + i, c) : 0.f;
                y[i] = rw + i < b.rows && c + 1 < b.cols ? side_at<T>(b.src, rw + i, c + 1) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)  // (ld is a multiple of 8: the pair fits)
                if (rw + i < b.rows && c < b.cols) put_pair<T>(b, (rw + i) * b.ld + c, x[i], y[i]);
            continue;
        }
        const bool along = b.src.sc <= b.src.sr;  // lanes along the columns
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = along ? w * 4 + (i >> 1) : lane, q = along ? (i & 1) * 32 + lane : w * 8 + i;
            if (r0 + r < b.rows && c0 + q < b.cols) tile[r][q] = side_at<T>(b.src, r0 + r, c0 + q);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (rw + i < b.rows && c < b.cols)
                put_pair<T>(b, (rw + i) * b.ld + c, tile[w * 4 + i][lane * 2], c + 1 < b.cols ? tile[w * 4 + i][lane * 2 + 1] : 0.f);
        __syncthreads();
    }
}

// out = sum over splits of partial [splits][rows][ldp]; rows from `half` on go to out2.  A
// thread adds four columns; ldp is a multiple of 4.
template <typename T>
__global__ void __launch_bounds__(256)
    sum_splits_kernel(const float* __restrict__ partial, int64_t ldp, int splits, int64_t rows, int64_t cols, T* out,
                      T* out2, int64_t half, int64_t ld) {
    const int64_t c = ((int64_t)blockIdx.x * 32 + (threadIdx.x & 31)) * 4;
    if (c >= cols) return;
    for (int64_t r = (int64_t)blockIdx.y * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.y * 8) {
        const float* p = partial + r * ldp + c;
        float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int q = 0; q < splits; ++q) {
            const float4 v = *reinterpret_cast<const float4*>(p + q * rows * ldp);
            z.x += v.x, z.y += v.y, z.z += v.z, z.w += v.w;
        }
        T* o = (r < half ? out + r * ld : out2 + (r - half) * ld) + c;
        const float zz[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < cols) o[e] = Cvt<T>::from_f(zz[e]);
    }
}

// The epilogue on split sums, partial [splits][1 or 2][M][ldp]: a block has 32 columns of 32 rows
template <typename T>
__global__ void __launch_bounds__(256)
    finish_kernel(const float* __restrict__ partial, int64_t ldp, int splits, int64_t M, int64_t N, const Epilogue e) {
    __shared__ float red[2][8][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t n = (int64_t)blockIdx.x * 32 + lane;
    const bool dual = e.kind == E_GLU || e.kind == E_GLU_BWD;
    for (int64_t blk = blockIdx.y; blk * 32 < M; blk += gridDim.y) {
        float sb = 0.f, ss = 0.f;
        for (int64_t m = blk * 32 + w; m < M && m < blk * 32 + 32; m += 8) {
            if (n >= N) break;
            float z = 0.f, u = 0.f;
            const float* p = partial + m * ldp + n;
            const int64_t one = M * ldp, step = dual ? 2 * one : one;
            for (int q0 = 0; q0 < splits; q0 += 8) {  // eight loads in flight, added in order
                float v[8], w[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    v[q] = q0 + q < splits ? p[(q0 + q) * step] : 0.f;
                    w[q] = dual && q0 + q < splits ? p[(q0 + q) * step + one] : 0.f;
                }
#pragma unroll
                for (int q = 0; q < 8; ++q) z += v[q], u += w[q];
            }
            const int64_t at = m * e.ldo + n;
            float r[2];
            if (e.kind == E_LINEAR) {
                if (e.bias.p) z += side_at<T>(e.bias, 0, n);
                r[0] = act_f(z, e.act);
                if (e.scale.p) r[0] *= side_at<T>(e.scale, 0, n);
                if (e.res.p) r[0] += side_at<T>(e.res, m, n);
            } else if (e.kind == E_GLU) {
                r[0] = act_f(z, e.act) * u;
            } else {
                if (e.bias.p) z += side_at<T>(e.bias, 0, n);
                const float g = side_at<T>(e.res, m, n);
                float y, d;
                act_grad_f(z, e.act, y, d);
                r[0] = g * d * (dual ? u : (e.scale.p ? side_at<T>(e.scale, 0, n) : 1.f));
                r[1] = g * y;
                sb += r[0], ss += r[1];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (i == 1 && e.kind != E_GLU_BWD) break;
                void* out = i ? e.out2 : e.out;
                if (e.out_f32) {
                    static_cast<float*>(out)[at] = r[i];
                } else {
                    static_cast<T*>(out)[at] = Cvt<T>::from_f(r[i]);
                }
            }
        }
        if (e.kind != E_LINEAR_BWD || !(e.part_bias || e.part_scale)) continue;
        red[0][w][lane] = sb, red[1][w][lane] = ss;
        __syncthreads();
        float* part = w == 0 ? e.part_bias : e.part_scale;
        if (w < 2 && part && n < N) {
            float t = 0.f;
            for (int q = 0; q < 8; ++q) t += red[w][q][lane];
            part[blk * N + n] = t;
        }
        __syncthreads();
    }
}

// part[blk][n] = sum of g over rows [128 blk, 128 blk + 128): eight warps take every eighth row each,
// and their sums are added in turn
constexpr int CS_ROWS = 128;
template <typename T>
__global__ void __launch_bounds__(256) colsum_kernel(Side g, int64_t rows, int64_t cols, float* part) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    __shared__ float red[8][32];
    for (int64_t blk = blockIdx.y; blk * CS_ROWS < rows; blk += gridDim.y) {
        const int64_t r0 = blk * CS_ROWS;
        float s = 0.f;
        if (c < cols)
            for (int64_t r = r0 + w; r < rows && r < r0 + CS_ROWS; r += 8) s += side_at<T>(g, r, c);
        red[w][lane] = s;
        __syncthreads();
        if (w == 0 && c < cols) {
            float t = 0.f;
            for (int q = 0; q < 8; ++q) t += red[q][lane];
            part[blk * cols + c] = t;
        }
        __syncthreads();
    }
}

// out[n] = sum over blocks of part [blocks][cols], for one or two vectors (blockIdx.y): 32
// threads add a column's blocks in turn, then their sums in order
struct Columns {
    const float* part[2];
    void* out[2];
    int64_t so[2];
    int f32[2];
};
template <typename T>
__global__ void __launch_bounds__(1024) colsum_finish_kernel(const Columns v, int64_t blocks, int64_t cols) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, i = blockIdx.y;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    __shared__ float red[32][33];
    float s = 0.f;
    if (c < cols) {
        const float* p = v.part[i] + c;
#pragma unroll 8
        for (int64_t b = w; b < blocks; b += 32) s += p[b * cols];
    }
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < cols) {
        float t = 0.f;
        for (int q = 0; q < 32; ++q) t += red[q][lane];
        if (v.f32[i]) static_cast<float*>(v.out[i])[c * v.so[i]] = t;
        else static_cast<T*>(v.out[i])[c * v.so[i]] = Cvt<T>::from_f(t);
    }
}

struct Ctx {
    int dt;    // operand type
    bool dry;  // workspace query: no launches
    Scratch ws;
    cudaStream_t s;
    Jobs jobs;  // operand copies not launched yet
    Plan plans[4];  // of the call's products, made by the workspace query and used in its order
    int n_plans = 0, next_plan = 0;
};

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
    const Plan plan = c.dry ? (c.plans[c.n_plans++] = c.dt == MABA_F32 ? simt_plan(p) : tc_plan(p)) : c.plans[c.next_plan++];
    const Product sums = plan.finish ? split_sums(p) : p;
    const int64_t rows = sums.form == F_PAIR ? 2 * p.M : p.M, ldp = partials_ld(p.N);
    float* partial = plan.splits > 1 ? static_cast<float*>(c.ws.take((size_t)partials_bytes(plan.splits, rows, p.N))) : nullptr;
    if (c.dry) return MABA_OK;
    if (c.dt == MABA_F32) MABA_TRY(simt_product(sums, plan.splits, partial, ldp, c.s));
    else MABA_TRY(DENSE_DISPATCH16(c.dt, [&] { return tc_product<T>(sums, plan, partial, ldp, c.s); }));
    if (plan.splits == 1) return MABA_OK;
    return DENSE_DISPATCH(c.dt, [&] {
        if (plan.finish)
            return launch(finish_kernel<T>, dim3((unsigned)ceil_div(p.N, 32), grid_y(ceil_div(p.M, 32))), dim3(256), 0, c.s,
                          partial, ldp, plan.splits, p.M, p.N, p.e);
        return launch(sum_splits_kernel<T>, dim3((unsigned)ceil_div(p.N, 128), grid_y(ceil_div(rows, 8))), dim3(256), 0, c.s,
                      partial, ldp, plan.splits, rows, p.N, static_cast<T*>(p.e.out), static_cast<T*>(p.e.out2), p.M, p.e.ldo);
    });
}

// Launches the copies that operand() has noted.
int prepare(Ctx& c) {
    const int n = c.jobs.n;
    if (n == 0) return MABA_OK;
    int64_t most = 1;
    for (int i = 0; i < n; ++i) {
        const int64_t t = ceil_div(c.jobs.j[i].rows, 32) * ceil_div(c.jobs.j[i].cols, 64);
        most = t > most ? t : most;
    }
    const int64_t cap = 16 * (int64_t)sm_count();
    const dim3 grid((unsigned)(most < cap ? most : cap), (unsigned)n);
    const Jobs jobs = c.jobs;
    c.jobs.n = 0;
    if (c.dry) return MABA_OK;
    return DENSE_DISPATCH16(c.dt, [&] {
        return launch(prepare_kernel<T>, grid, dim3(256), 0, c.s, jobs);
    });
}

int column_sums(Ctx& c, const Side& g, int64_t rows, int64_t cols, float* part) {
    if (c.dry) return MABA_OK;
    return DENSE_DISPATCH(c.dt, [&] {
        const dim3 grid((unsigned)ceil_div(cols, 32), grid_y(ceil_div(rows, CS_ROWS)));
        return launch(colsum_kernel<T>, grid, dim3(256), 0, c.s, g, rows, cols, part);
    });
}

int finish_columns(Ctx& c, const float* pb, const maba_tensor* db, const float* ps, const maba_tensor* ds, int64_t blocks,
                   int64_t cols) {
    Columns v{};
    int n = 0;
    for (int i = 0; i < 2; ++i) {
        const maba_tensor* t = i ? ds : db;
        if (!(i ? ps : pb)) continue;
        v.part[n] = i ? ps : pb, v.out[n] = t->data, v.so[n] = t->stride[0], v.f32[n] = t->dtype == MABA_F32;
        ++n;
    }
    if (n == 0) return MABA_OK;
    return DENSE_DISPATCH(c.dt, [&] {
        return launch(colsum_finish_kernel<T>, dim3((unsigned)ceil_div(cols, 32), (unsigned)n), dim3(1024), 0, c.s, v, blocks,
                          cols);
    });
}

// ---------------------------------------------------------------------------
// argument checks
// ---------------------------------------------------------------------------
bool given(const maba_tensor* t) { return t != nullptr && t->ndim > 0; }

int want_matrix(const maba_tensor* t, const char* name, int64_t rows, int64_t cols, int dt, bool f32_ok, bool dense_rows) {
    if (!given(t)) return set_error(MABA_ERR_INVALID, "%s: tensor is required", name);
    if (t->ndim != 2) return set_error(MABA_ERR_INVALID, "%s: expected 2 dims, got %d", name, t->ndim);
    if (t->shape[0] < 0 || t->shape[1] < 0) return set_error(MABA_ERR_INVALID, "%s: negative size", name);
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
// a gradient: its elements lie apart
int want_vector_out(const maba_tensor* t, const char* name, int64_t n, int dt) {
    MABA_TRY(want_vector(t, name, n, dt));
    return n > 1 && t->stride[0] < 1 ? set_error(MABA_ERR_INVALID, "%s: elements must not overlap", name) : MABA_OK;
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
// 16-byte boundaries; what is not laid out so is copied once per call (noted here, launched by
// prepare()).  One copy serves both directions of a matrix: K-major along its rows, MN-major
// across them.  The float32 products read the caller's matrix.
void operand(Ctx& c, const maba_tensor* t, Matrix& m, bool as_is = false) {
    const Side src = side2(t);
    const int64_t rows = t->shape[0], cols = t->shape[1];
    m = Matrix{src.p, src.sr, src.sc};
    if (as_is || c.dt == MABA_F32 || (!src.f32 && tc_readable(src.p, rows, cols, src.sr, src.sc))) return;
    const int64_t ld = (cols + 7) / 8 * 8;
    void* to = c.ws.take((size_t)rows * ld * 2);
    m = Matrix{to, ld, 1};
    c.jobs.j[c.jobs.n++] = Job{src, rows, cols, to, ld, 0};
}
// A matrix that an epilogue of the tensor-core products reads: copied where its rows are not on
// 16-byte boundaries (a broadcast one too).
Side side_of(Ctx& c, const maba_tensor* t, bool as_is = false) {
    const Side src = side2(t);
    if (!given(t) || as_is || c.dt == MABA_F32) return src;
    const int64_t rows = t->shape[0], cols = t->shape[1], per = src.f32 ? 4 : 8;
    if (src.sc == 1 && (rows == 1 || (src.sr % per == 0 && src.sr >= cols)) && (reinterpret_cast<uintptr_t>(src.p) & 15u) == 0)
        return src;
    const int64_t ld = (cols + 7) / 8 * 8;
    void* to = c.ws.take((size_t)rows * ld * (src.f32 ? 4 : 2));
    c.jobs.j[c.jobs.n++] = Job{src, rows, cols, to, ld, src.f32};
    return Side{to, ld, 1, src.f32};
}
// A gradient that an epilogue writes as an operand of the next products.
Matrix written_operand(Ctx& c, int64_t rows, int64_t cols) {
    const int64_t ld = (cols + 7) / 8 * 8;
    return Matrix{c.ws.take((size_t)rows * ld * (c.dt == MABA_F32 ? 4 : 2)), ld, 1};
}
Matrix transposed(const Matrix& m) { return Matrix{m.p, m.sk, m.sr}; }

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
    operand(c, a.x, p.a[0], as_is);
    operand(c, a.w, p.b[0], as_is);
    p.e.res = side_of(c, a.res, as_is);
    MABA_TRY(prepare(c));
    p.e.act = a.act;
    p.e.bias = side1(a.bias), p.e.scale = side1(a.scale);
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
    p.b_mn = true;
    p.e.out = dx->data, p.e.ldo = dx->stride[0];
    return run(c, p);
}
int dw_product(Ctx& c, int64_t M, int n, const Matrix* d, const Matrix& x, const maba_tensor* const* dw) {
    Product p;
    p.form = n == 2 ? F_PAIR : F_SINGLE;
    p.M = dw[0]->shape[0], p.N = dw[0]->shape[1], p.K = M;
    for (int i = 0; i < n; ++i) p.a[i] = transposed(d[i]);
    p.b[0] = p.b[1] = transposed(x);
    p.a_mn = p.b_mn = true;
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
    if (!through || need_dw) operand(c, a.x, x);
    if (!through || need_dx) operand(c, a.w, w);
    // (the products take one type: where dz = g, a float32 gradient is rounded to x's here)
    if (through && (need_dx || need_dw)) operand(c, a.g, d);
    Side g;
    if (!through) g = side_of(c, a.g);
    MABA_TRY(prepare(c));
    if (!through) {
        // z again, rather than a copy kept by the forward pass: a 16-bit z would add its own
        // rounding to phi'(z), and a float32 one costs more traffic than the product
        d = written_operand(c, M, N);
        Product p;
        p.M = M, p.N = N, p.K = K;
        p.a[0] = x, p.b[0] = w;
        p.e.kind = E_LINEAR_BWD;
        p.e.act = a.act;
        p.e.bias = side1(a.bias), p.e.scale = side1(a.scale), p.e.res = g;
        p.e.out = const_cast<void*>(d.p), p.e.ldo = d.sr;
        p.e.part_bias = pb, p.e.part_scale = ps;
        p.e.sums_f32 = (need_db && a.dbias->dtype == MABA_F32) || (need_ds && a.dscale->dtype == MABA_F32);
        MABA_TRY(run(c, p));
    } else if (need_db) {
        MABA_TRY(column_sums(c, side2(a.g), M, N, pb));
    }
    if (!c.dry) MABA_TRY(finish_columns(c, pb, a.dbias, ps, a.dscale, blocks, N));
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
    operand(c, a.x, p.a[0], as_is);
    operand(c, a.wg, p.b[0], as_is);
    operand(c, a.wu, p.b[1], as_is);
    p.e.res = side_of(c, a.g);
    return prepare(c);
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
    // dg and du in the operands' type: the one rounding between the two passes where that has 16 bits,
    // which is what the tensor cores multiply; none in float32
    const Matrix d[2] = {written_operand(c, M, p.N), written_operand(c, M, p.N)};
    p.e.out = const_cast<void*>(d[0].p), p.e.out2 = const_cast<void*>(d[1].p), p.e.ldo = d[0].sr;
    MABA_TRY(run(c, p));
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
        MABA_TRY(want_vector_out(a.dbias, "dbias", N, dt));
        if (!given(a.bias)) return set_error(MABA_ERR_INVALID, "dbias without bias");
    }
    if (given(a.dscale)) {
        MABA_TRY(want_vector_out(a.dscale, "dscale", N, dt));
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

template <typename Args, typename F> Ctx query(const Args& a, F op) {
    Ctx c{};
    c.dt = a.x->dtype, c.dry = true;
    if (op(c, a) != MABA_OK) c.ws.used = 0;
    return c;
}

template <typename Args, typename F>
int execute(const Args& a, F op, const char* name, void* workspace, size_t bytes, void* stream) {
    Ctx c = query(a, op);
    const size_t need = c.ws.used;
    if (need > 0 && (workspace == nullptr || bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))
        return set_error(MABA_ERR_WORKSPACE, "%s: needs a 256-byte aligned workspace of %zu bytes, got %zu", name, need, bytes);
    c.dry = false;
    c.ws = Scratch{static_cast<unsigned char*>(workspace), 0};
    c.s = as_stream(stream);
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

extern "C" size_t maba_linear_workspace_size(const maba_tensor* x, const maba_tensor* weight, const maba_tensor* residual,
                                             const maba_tensor* out) {
    LinearArgs a{};
    a.x = x, a.w = weight, a.res = residual, a.out = out;
    if (check_linear(a, false) != MABA_OK) return 0;
    return query(a, linear_forward).ws.used;
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
    return query(a, linear_backward).ws.used;
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
    return query(a, ffn_forward).ws.used;
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
    return query(a, ffn_backward).ws.used;
}

extern "C" int maba_selftest_split_layout(int64_t rows, int64_t cols, int32_t splits, int32_t pairs, int64_t* reserved,
                                          int64_t* reached) {
    if (rows < 1 || cols < 1 || splits < 1 || pairs < 1 || reserved == nullptr || reached == nullptr)
        return set_error(MABA_ERR_INVALID, "selftest_split_layout: sizes must be positive");
    *reserved = partials_bytes(splits, rows * pairs, cols);
    *reached = 4 * partials_reach(rows, cols, partials_ld(cols), (int64_t)splits * pairs);
    return MABA_OK;
}
