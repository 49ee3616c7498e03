// A dense layer with what follows it, and its gradients:
//   z = x W^T + b,   y = act(z) + residual;   dz = dy act'(z),   dx = dz W,   dW = dz^T x,   db = sum over rows of dz
//
// The products are fgl_row_product.hip's (fp32 on the bf16 matrix cores: fgl_split_product.hip) and fgl_wgrad.hip's; the forward one stores act(z) + residual
// from its accumulators, and act': a bit a value for relu, the slope itself for gelu and silu (in bf16 as fp16, whose eleven bits, down to 2^-29, leave dz with the one rounding that the
// matrix cores ask for: gradients off by 2.36e-3 in the 2-norm, results rounded once alone by 1.66e-3, torch's layer in bf16 2.43e-3; with z kept in bf16 2.5e-3.  dz in two bf16 parts would
// leave the results' rounding alone, for twice the products and a pass over n x out values more in each of three kernels).  The backward pass forms dz in one pass over dy
// (none where there is no activation: dz is dy).
//
// KEEP8: the rows of x are held in 8 bits a value (fgl_keep8.hpp) for dW, which fgl_wgrad8.hip forms from them; dx and db need no x.  db comes with dW, or alone from
// fgl_column_sums.hip (60 K x 256 fp32 17 us, where dW with it takes 82).
//
// What bounds it: the products (their files say); dz the pass over memory (2.4 M x 64 bf16 173 us, 5.3 TB/s; 107 K x 256 fp32 60 us, 5.5 TB/s), and so the rows in 8 bits.
#include "fgl_activation.hpp"
#include "fgl_column_sums.hpp"
#include "fgl_common.hpp"
#include "fgl_keep8.hpp"
#include "fgl_kernels.hpp"
#include "fgl_row_product.hpp"
#include "fgl_wgrad8.hpp"

#include <type_traits>

namespace fgl {

constexpr int kLinearMost = 4096;  // columns of x and y
constexpr int kPackRows = 16;      // of a workgroup
constexpr int kPackLoads = 4;      // of a lane, on their way together

struct LinearState {
    uint32_t* mask;  // relu: [n][mask_ld]
    void* slope;     // gelu, silu: [n][ldz] fp32, or fp16 times kSlopeScale for bf16
    uint8_t* codes;  // KEEP8, behind those, which are all that there is without it: [n][k8_columns(dim)]
    uint8_t* steps;  // KEEP8: [k8_columns(dim) / 32][w8_step_ld(n)]
    int64_t mask_ld, ldz;
    size_t bytes;
};

static LinearState linear_state(void* base, int64_t n, int dim, int out, int dtype, int act, bool keep8)
{
    Carver c(base);
    LinearState s;
    memset(&s, 0, sizeof(s));
    s.mask_ld = (out + 31) / 32;
    s.ldz = (out + 1) / 2 * 2;
    if (act == kActRelu) s.mask = c.take<uint32_t>((size_t)n * (size_t)s.mask_ld);
    else if (act != kActNone) s.slope = c.take<uint8_t>((size_t)n * (size_t)s.ldz * (dtype == FGL_F32 ? 4 : 2));
    if (keep8) {
        s.codes = c.take<uint8_t>((size_t)n * (size_t)k8_columns(dim));
        s.steps = c.take<uint8_t>((size_t)(k8_columns(dim) / 32) * (size_t)w8_step_ld(n));
    }
    s.bytes = c.used();
    return s;
}

template <typename T>
constexpr int kLinV = 16 / (int)sizeof(T);
template <typename T>
using LinVec = T __attribute__((ext_vector_type(kLinV<T>), aligned(sizeof(T))));

template <typename T>
__device__ __forceinline__ LinVec<T> lin_load(const T* p, int left)
{
    LinVec<T> v;
    if (left >= kLinV<T>) {
        v = *reinterpret_cast<const LinVec<T>*>(p);
    } else {
#pragma unroll
        for (int e = 0; e < kLinV<T>; ++e) {
            v[e] = (T)0.0f;
            if (e < left) v[e] = p[e];
        }
    }
    return v;
}

// Rows in 8 bits a value.  A workgroup takes 16 rows, a lane 16 bytes of one at a time, so that 32 columns are those of 8 lanes (bf16: 4); steps are
// gathered in LDS, since those of a column of rows are neighbours.  (64 rows a workgroup and a load at a time: 8192 x 602 fp32 25 us, 8 so, 87 K x 512 bf16 34, 28.)
template <typename T>
__global__ __launch_bounds__(kBlock) void pack8_kernel(const T* __restrict__ x, int64_t ldx, int64_t n, int d, int code_ld, uint8_t* __restrict__ codes,
                                                      uint8_t* __restrict__ steps, int64_t step_ld)
{
    constexpr int V = kLinV<T>, kGroup = 32 / V;
    __shared__ uint8_t s_step[kLinearMost / 32][kPackRows];
    typedef uint32_t Codes __attribute__((ext_vector_type(V / 4)));
    const int64_t row0 = (int64_t)blockIdx.x * kPackRows;
    const int per_row = code_ld / V, rows = n - row0 < kPackRows ? (int)(n - row0) : kPackRows;
    const int items = rows * per_row;
    for (int i0 = (int)threadIdx.x; i0 - (int)threadIdx.x < items; i0 += kBlock * kPackLoads) {  // (the lanes of a group are all in or all out)
        LinVec<T> v[kPackLoads];
        int r[kPackLoads], c[kPackLoads];
#pragma unroll
        for (int k = 0; k < kPackLoads; ++k) {
            const int i = i0 + k * kBlock;
            r[k] = i / per_row;
            c[k] = (i - r[k] * per_row) * V;
            v[k] = lin_load(x + (row0 + r[k]) * ldx + c[k], i < items ? d - c[k] : 0);
        }
#pragma unroll
        for (int k = 0; k < kPackLoads; ++k) {
            uint32_t most = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const uint32_t m = __float_as_uint((float)v[k][e]) & 0x7FFFFFFFu;
                most = most > m ? most : m;
            }
            most = group_max<kGroup>(most) >> 23;
            const uint32_t step = most == 0xFF ? kStepNone : k8_step((int)most - 127);
            const float inverse = step == kStepNone ? 0.0f : k8_inverse(step);
            Codes q;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const uint32_t code = k8_code((float)v[k][e], inverse);
                if (e % 4 == 0) q[e / 4] = code;
                else q[e / 4] |= code << 8 * (e % 4);
            }
            q ^= kSigned;
            if (i0 + k * kBlock < items) {
                *reinterpret_cast<Codes*>(codes + (row0 + r[k]) * code_ld + c[k]) = q;
                if (c[k] % 32 == 0) s_step[c[k] / 32][r[k]] = (uint8_t)step;
            }
        }
    }
    __syncthreads();
    const int columns = code_ld / 32;
    for (int i = (int)threadIdx.x; i < columns * kPackRows; i += kBlock) {
        const int c = i / kPackRows, r = i % kPackRows;
        if (r < rows) steps[c * step_ld + row0 + r] = s_step[c][r];
    }
}

// dz = dy act'(z); rows of the slopes and of dz are ldz apart, those of dy lddy.  2^log_lanes neighbouring lanes take the loads of a row, and a lane those of
// kSlopeRows rows at a time.
constexpr int kSlopeRows = 4;
template <typename T>
using SlopeOf = std::conditional_t<sizeof(T) == 4, float, _Float16>;

template <typename T, bool MASK>
__global__ __launch_bounds__(kBlock) void slope_kernel(const T* __restrict__ dy, int64_t lddy, const SlopeOf<T>* __restrict__ slope, const uint32_t* __restrict__ mask,
                                                      int64_t mask_ld, int64_t n, int d, int64_t ldz, T* __restrict__ dz, int log_lanes)
{
    constexpr int V = kLinV<T>;
    const int l = (int)threadIdx.x & ((1 << log_lanes) - 1), rows = kBlock >> log_lanes;
    const int64_t first = (int64_t)blockIdx.x * rows * kSlopeRows + (threadIdx.x >> log_lanes);
    for (int c = l * V; c < d; c += V << log_lanes) {
        const int left = d - c;
        LinVec<T> g[kSlopeRows];
        LinVec<SlopeOf<T>> s[kSlopeRows];
        uint32_t bits[kSlopeRows];
#pragma unroll
        for (int i = 0; i < kSlopeRows; ++i) {
            const int64_t row = first + i * rows < n ? first + i * rows : n - 1;
            g[i] = lin_load(dy + row * lddy + c, left);
            if constexpr (MASK) bits[i] = mask[row * mask_ld + c / 32] >> (c % 32);
            else s[i] = lin_load(slope + row * ldz + c, left);
        }
#pragma unroll
        for (int i = 0; i < kSlopeRows; ++i) {
            LinVec<T> q;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (MASK) q[e] = bits[i] >> e & 1u ? g[i][e] : (T)0.0f;
                else q[e] = (T)((float)g[i][e] * ((float)s[i][e] * (sizeof(T) == 4 ? 1.0f : 1.0f / kSlopeScale)));
            }
            if (first + i * rows >= n) break;
            T* to = dz + (first + i * rows) * ldz + c;
            if (left >= V) {
                *reinterpret_cast<LinVec<T>*>(to) = q;
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < left) to[e] = q[e];
            }
        }
    }
}

template <typename T>
static int launch_slope(const void* dy, int64_t lddy, const LinearState& s, int act, int64_t n, int d, void* dz, hipStream_t stream)
{
    int log_lanes = 0;
    while (log_lanes < 6 && (kLinV<T> << log_lanes) < d) ++log_lanes;
    const int64_t blocks = ceil_div(n, (int64_t)(kBlock >> log_lanes) * kSlopeRows);
    const dim3 grid((unsigned)blocks);  // (n below 2^31, 16 rows and more a workgroup)
    if (act == kActRelu)
        hipLaunchKernelGGL((slope_kernel<T, true>), grid, dim3(kBlock), 0, stream, static_cast<const T*>(dy), lddy, (const SlopeOf<T>*)nullptr, s.mask, s.mask_ld, n, d, s.ldz,
                           static_cast<T*>(dz), log_lanes);
    else
        hipLaunchKernelGGL((slope_kernel<T, false>), grid, dim3(kBlock), 0, stream, static_cast<const T*>(dy), lddy, static_cast<const SlopeOf<T>*>(s.slope),
                           (const uint32_t*)nullptr, (int64_t)0, n, d, s.ldz, static_cast<T*>(dz), log_lanes);
    FGL_CHECK_LAUNCH("slope_kernel");
    return FGL_OK;
}

// What the backward pass carves from its workspace: dz (where there is an activation), the sums of the weight's gradient, or of the bias's alone
struct LinearWorkspace {
    void* dz;
    void* sums;
    size_t sums_bytes, bytes;
};
// The bias's gradient is the one that it has beside the weight's
static ColumnSplit linear_column_split(int64_t n, int dim, int out, int dtype, bool keep8)
{
    return keep8 ? wgrad8_column_split(n, out, dim, dtype) : wgrad_column_split(n, out, dim, dtype);
}
static LinearWorkspace linear_workspace(void* base, int64_t n, int dim, int out, int dtype, int act, bool keep8, bool need_w, bool need_b)
{
    Carver c(base);
    LinearWorkspace w;
    memset(&w, 0, sizeof(w));
    const size_t size = dtype == FGL_F32 ? 4 : 2;
    if (act != kActNone) w.dz = c.take<uint8_t>((size_t)n * (size_t)((out + 1) / 2 * 2) * size);
    if (need_w || need_b) {
        if (!need_w) w.sums_bytes = column_sums_workspace_bytes(linear_column_split(n, dim, out, dtype, keep8), out);
        else w.sums_bytes = keep8 ? wgrad8_workspace_bytes(n, out, dim, dtype) : fgl_weight_grad_workspace_bytes_for(n, out, dim, dtype);
        w.sums = c.take<uint8_t>(w.sums_bytes);
    }
    w.bytes = c.used();
    return w;
}

static bool linear_sizes(int64_t n, int dim, int out, int dtype, int act)
{
    return n >= 0 && n <= 0x7FFFFFFF && dim >= 1 && dim <= kLinearMost && out >= 1 && out <= kLinearMost && (dtype == FGL_F32 || dtype == FGL_BF16) && act >= kActNone &&
           act <= kActSilu;
}

#define FGL_LINEAR_ROWS(p_, ld_, cols_)                                                                                                                  \
    FGL_REQUIRE((ld_) >= (cols_) && (ld_) < (1 << 24), "linear: row stride %lld of %d columns", (long long)(ld_), (int)(cols_));                         \
    FGL_REQUIRE(dtype == FGL_F32 || ((ld_) % 2 == 0 && (uintptr_t)(p_) % 4 == 0), "linear: bf16 rows must start on 4-byte boundaries")

}  // namespace fgl

using namespace fgl;

FGL_EXPORT size_t fgl_linear_state_bytes(int64_t n, int dim, int out, int dtype, int act, int keep8)
{
    return linear_sizes(n, dim, out, dtype, act) ? linear_state(nullptr, n, dim, out, dtype, act, keep8 != 0).bytes : 0;
}

FGL_EXPORT size_t fgl_linear_workspace_bytes(int64_t n, int dim, int out, int dtype, int act, int keep8, int want_w, int want_b)
{
    return linear_sizes(n, dim, out, dtype, act) ? linear_workspace(nullptr, n, dim, out, dtype, act, keep8 != 0, want_w != 0, want_b != 0).bytes : 0;
}

FGL_EXPORT int fgl_linear(const void* d_x, int64_t ldx, const void* d_w, int64_t ldw, const void* d_bias, const void* d_residual, int64_t ldr, int64_t n, int dim, int out,
                          int dtype, int act, int keep8, void* d_y, int64_t ldy, void* d_state, size_t state_bytes, void* stream)
{
    FGL_REQUIRE(linear_sizes(n, dim, out, dtype, act), "linear: %lld rows of %d by %d columns, dtype %d, activation %d", (long long)n, dim, out, dtype, act);
    FGL_LINEAR_ROWS(d_x, ldx, dim);
    FGL_LINEAR_ROWS(d_w, ldw, dim);
    FGL_REQUIRE(ldy >= out && ldy < (1 << 24) && (d_residual == nullptr || (ldr >= out && ldr < (1 << 24))), "linear: row strides %lld and %lld of %d columns", (long long)ldy,
                (long long)ldr, out);
    if (n == 0) return FGL_OK;
    FGL_REQUIRE(d_x && d_w && d_y, "linear: null pointer");
    RowProductArgs g;
    memset(&g, 0, sizeof(g));
    g.side[0] = RowProductSide{d_x, d_w, ldx, ldw, dim};
    g.bias = d_bias; g.c = d_y; g.ldc = ldy; g.m = n; g.n = out;
    g.then.act = act; g.then.residual = d_residual; g.then.ldr = d_residual != nullptr ? ldr : 0;
    hipStream_t s = as_stream(stream);
    if (d_state != nullptr) {
        const LinearState kept = linear_state(d_state, n, dim, out, dtype, act, keep8 != 0);
        if (state_bytes < kept.bytes || ((uintptr_t)d_state & 255) != 0) {
            set_error("linear: state of %zu bytes at a multiple of 256 bytes, %zu given", kept.bytes, state_bytes);
            return FGL_ERR_WORKSPACE;
        }
        if (act == kActRelu) {
            g.then.mask = kept.mask;
            g.then.mask_ld = kept.mask_ld;
        } else if (act != kActNone) {
            g.then.slope = kept.slope;
            g.then.lds = kept.ldz;
        }
        if (keep8) {
            const dim3 grid((unsigned)ceil_div(n, kPackRows));
            if (dtype == FGL_F32)
                hipLaunchKernelGGL(pack8_kernel<float>, grid, dim3(kBlock), 0, s, static_cast<const float*>(d_x), ldx, n, dim, (int)k8_columns(dim), kept.codes, kept.steps,
                                   w8_step_ld(n));
            else
                hipLaunchKernelGGL(pack8_kernel<__bf16>, grid, dim3(kBlock), 0, s, static_cast<const __bf16*>(d_x), ldx, n, dim, (int)k8_columns(dim), kept.codes, kept.steps,
                                   w8_step_ld(n));
            FGL_CHECK_LAUNCH("pack8_kernel");
        }
    }
    return row_product_then(g, true, dtype, s);
}

FGL_EXPORT int fgl_linear_backward(const void* d_dy, int64_t lddy, const void* d_x, int64_t ldx, const void* d_w, int64_t ldw, int64_t n, int dim, int out, int dtype,
                                   int act, int keep8, const void* d_state, size_t state_bytes, void* d_dx, int64_t lddx, void* d_dw, void* d_db, void* d_ws, size_t ws_bytes,
                                   void* stream)
{
    FGL_REQUIRE(linear_sizes(n, dim, out, dtype, act) && n >= 1, "linear_backward: %lld rows of %d by %d columns, dtype %d, activation %d", (long long)n, dim, out, dtype, act);
    const bool sums = d_dw != nullptr || d_db != nullptr;
    if (d_dx == nullptr && !sums) return FGL_OK;
    FGL_REQUIRE(d_dy != nullptr && (d_dx == nullptr || d_w != nullptr) && (d_dw == nullptr || keep8 || d_x != nullptr), "linear_backward: null pointer");
    if (act == kActNone) {  // (dy is an operand itself then)
        FGL_LINEAR_ROWS(d_dy, lddy, out);
    } else {
        FGL_REQUIRE(lddy >= out, "linear_backward: row stride smaller than the row length");
    }
    FGL_REQUIRE(d_dx == nullptr || (ldw >= dim && lddx >= dim && ldw < (1 << 24) && lddx < (1 << 24)), "linear_backward: row strides %lld and %lld of %d columns", (long long)ldw,
                (long long)lddx, dim);
    if (d_dw != nullptr && !keep8) {
        FGL_LINEAR_ROWS(d_x, ldx, dim);
    }
    LinearState kept;
    memset(&kept, 0, sizeof(kept));
    const bool codes = keep8 && d_dw != nullptr;  // (nothing else reads them)
    if (codes || act != kActNone) {
        kept = linear_state(const_cast<void*>(d_state), n, dim, out, dtype, act, codes);
        if (d_state == nullptr || state_bytes < kept.bytes || ((uintptr_t)d_state & 255) != 0) {
            set_error("linear_backward: state of %zu bytes at a multiple of 256 bytes, %zu given", kept.bytes, state_bytes);
            return FGL_ERR_WORKSPACE;
        }
    }
    const LinearWorkspace w = linear_workspace(d_ws, n, dim, out, dtype, act, keep8 != 0, d_dw != nullptr, d_db != nullptr);
    if (w.bytes > 0 && (d_ws == nullptr || ws_bytes < w.bytes || ((uintptr_t)d_ws & 255) != 0)) {
        set_error("linear_backward: workspace of %zu bytes at a multiple of 256 bytes, %zu given", w.bytes, ws_bytes);
        return FGL_ERR_WORKSPACE;
    }
    hipStream_t s = as_stream(stream);
    const void* dz = d_dy;
    int64_t lddz = lddy;
    if (act != kActNone) {
        const int rc = dtype == FGL_F32 ? launch_slope<float>(d_dy, lddy, kept, act, n, out, w.dz, s) : launch_slope<__bf16>(d_dy, lddy, kept, act, n, out, w.dz, s);
        if (rc != FGL_OK) return rc;
        dz = w.dz;
        lddz = kept.ldz;
    }
    if (d_dx != nullptr) {
        RowProductArgs g;
        memset(&g, 0, sizeof(g));
        g.side[0] = RowProductSide{dz, d_w, lddz, ldw, out};
        g.c = d_dx; g.ldc = lddx; g.m = n; g.n = dim;
        const int rc = row_product_then(g, false, dtype, s);
        if (rc != FGL_OK) return rc;
    }
    if (!sums) return FGL_OK;
    if (d_dw == nullptr) return launch_column_sums(dz, lddz, n, out, dtype, linear_column_split(n, dim, out, dtype, keep8 != 0), d_db, w.sums, w.sums_bytes, s);
    if (keep8) return launch_wgrad8(dz, lddz, kept.codes, kept.steps, n, out, dim, dtype, d_dw, dim, d_db, w.sums, w.sums_bytes, s);
    return fgl_weight_grad(dz, lddz, d_x, ldx, n, out, dim, dtype, d_dw, dim, d_db, w.sums, w.sums_bytes, stream);
}
