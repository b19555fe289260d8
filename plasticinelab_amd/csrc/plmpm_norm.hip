// Norms before and after a block, with the block's gate and residual scale, in one pass (include/plmpm_policy.h: plmpm_norm):
//
//   y = x + scale * f(gate) * post * uh,  uh = u ru,  ru = 1 / sqrt(mean(u^2) + eps)
//   z = pre * yh,                         yh = y ry,  ry = 1 / sqrt(mean(y^2) + eps)
// backward, with q = dz * pre:
//   dy' = dy + ry (q - yh mean(q yh))       dx = dy'       w = dy' * scale * f * post      du = ru (w - uh mean(w uh))
//   dgate = dy' * scale * post * uh * f'    dscale = sum dy' f post uh     dpost = sum dy' scale f uh     dpre = sum dz yh
//
// A row stays in the registers of TPR threads (eight columns each) between its sums, so every input is read once; nothing but the
// inputs themselves is kept for the backward pass, which makes y and both norms again (x in place of y: the same bytes, and unrounded).
// z comes from the unrounded y.  A thread keeps its columns over the rows that its workgroup walks: the three weights are loaded
// once, and the three column sums grow in registers (32 bits) and leave as one partial row a workgroup; a second kernel adds those in a
// fixed order.
#include <algorithm>

#include "plmpm_nn.h"

using namespace plbnn;

namespace {

constexpr int kCols = 8;                // columns a thread
constexpr int kMaxRowThreads = 1024;
constexpr int kMaxWidth = kCols * kMaxRowThreads;
constexpr int kMaxBlocks = 512;         // workgroups of a backward launch: one partial row of column sums each

struct NormArgs {
    const void *x, *u, *gate, *scale, *post, *pre, *dy, *dz;
    void *y, *z, *dx, *du, *dgate;
    float* part;                        // [workgroups][3][width]: dscale, dpost, dpre
    int64_t rows, sx, su, sg, sdy, sdz;
    int D, tpr, fn, wt;
    float eps;
};

// sum over the `tpr` (a power of two) neighbouring threads that hold a row; `lds`: one float a wave, another buffer for each sum of a row
__device__ __forceinline__ float row_sum(float v, int tpr, float* lds) {
    const int top = tpr < 64 ? tpr : 64;
    for (int m = 1; m < top; m <<= 1) v += __shfl_xor(v, m);
    if (tpr <= 64) return v;
    const int wave = threadIdx.x >> 6, per = tpr >> 6, first = wave & ~(per - 1);
    if ((threadIdx.x & 63) == 0) lds[wave] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < per; ++w) v += lds[first + w];
    return v;
}

__device__ __forceinline__ void gate_of(int fn, float g, float& f, float& df) {
    if (fn == PLMPM_GATE_IDENTITY) { f = g; df = 1.0f; return; }
    const float s = sigmoid_fast(g);
    if (fn == PLMPM_GATE_SIGMOID) { f = s; df = s * (1.0f - s); }
    else { f = g * s; df = s * fmaf(g, 1.0f - s, 1.0f); }
}

// column of element k of piece j: pieces of VW neighbouring columns, TPR pieces apart
template <int VW> __device__ __forceinline__ int column(int tpr, int j) { return (j * tpr + (int)(threadIdx.x & (tpr - 1))) * VW; }

template <int VW> __device__ __forceinline__ void load_weight(const void* w, int dtype, int D, int tpr, float* out) {
#pragma unroll
    for (int j = 0; j < kCols / VW; ++j) {
        const int c = column<VW>(tpr, j);
#pragma unroll
        for (int k = 0; k < VW; ++k) out[j * VW + k] = w ? 0.0f : 1.0f;
        if (!w || c >= D) continue;
        if (dtype == PLMPM_NN_F32) { Vec<float, VW> v; v.load((const float*)w + c); v.get(out + j * VW); }
        else if (dtype == PLMPM_NN_BF16) { Vec<bf16, VW> v; v.load((const bf16*)w + c); v.get(out + j * VW); }
        else { Vec<f16, VW> v; v.load((const f16*)w + c); v.get(out + j * VW); }
    }
}
template <class T, int VW> __device__ __forceinline__ void load_row(const void* p, int64_t row, int64_t stride, int D, int tpr, float* out) {
#pragma unroll
    for (int j = 0; j < kCols / VW; ++j) {
        const int c = column<VW>(tpr, j);
        Vec<T, VW> v;
        if (p && c < D) v.load((const T*)p + row * stride + c);
        else v.zero();
        v.get(out + j * VW);
    }
}
template <class T, int VW> __device__ __forceinline__ void store_row(void* p, int64_t row, int D, int tpr, const float* in) {
#pragma unroll
    for (int j = 0; j < kCols / VW; ++j) {
        const int c = column<VW>(tpr, j);
        if (c >= D) continue;
        Vec<T, VW> v;
        v.set(in + j * VW);
        v.store((T*)p + row * D + c);
    }
}

template <class TX, class TU, int VW>
__global__ __launch_bounds__(1024) void k_norm_forward(NormArgs A) {
    __shared__ float lds[2][16];
    const int tpr = A.tpr, group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const float inv = 1.0f / (float)A.D;
    float scale[kCols], post[kCols], pre[kCols];
    load_weight<VW>(A.scale, A.wt, A.D, tpr, scale);
    load_weight<VW>(A.post, A.wt, A.D, tpr, post);
    load_weight<VW>(A.pre, A.wt, A.D, tpr, pre);
    for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows; base += (int64_t)gridDim.x * groups) {
        const bool there = base + group < A.rows;              // every thread takes part in the sums
        const int64_t row = there ? base + group : A.rows - 1;
        float y[kCols], u[kCols], g[kCols];
        load_row<TX, VW>(A.x, row, A.sx, A.D, tpr, y);
        if (A.u) {
            load_row<TU, VW>(A.u, row, A.su, A.D, tpr, u);
            load_row<TU, VW>(A.gate, row, A.sg, A.D, tpr, g);
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < kCols; ++k) s = fmaf(u[k], u[k], s);
            const float ru = __builtin_amdgcn_rsqf(fmaf(row_sum(s, tpr, lds[0]), inv, A.eps));
#pragma unroll
            for (int k = 0; k < kCols; ++k) {
                float f = 1.0f, df;
                if (A.gate) gate_of(A.fn, g[k], f, df);
                y[k] = fmaf(scale[k] * f, post[k] * (u[k] * ru), y[k]);
            }
            if (there) store_row<TX, VW>(A.y, row, A.D, tpr, y);
        }
        if (A.z) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < kCols; ++k) s = fmaf(y[k], y[k], s);
            const float ry = __builtin_amdgcn_rsqf(fmaf(row_sum(s, tpr, lds[1]), inv, A.eps));
#pragma unroll
            for (int k = 0; k < kCols; ++k) y[k] = pre[k] * (y[k] * ry);
            if (there) store_row<TU, VW>(A.z, row, A.D, tpr, y);
        }
        if (tpr > 64 && !(A.u && A.z)) __syncthreads();        // with one sum a row its buffer is written again at once; with two, the other's barrier lies between
    }
}

template <class TX, class TU, int VW>
__global__ __launch_bounds__(1024) void k_norm_backward(NormArgs A) {
    __shared__ float lds[4][16], fold[kCols * 256];
    const int tpr = A.tpr, group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const float inv = 1.0f / (float)A.D;
    float scale[kCols], post[kCols], pre[kCols], sums[3][kCols];
    load_weight<VW>(A.scale, A.wt, A.D, tpr, scale);
    load_weight<VW>(A.post, A.wt, A.D, tpr, post);
    load_weight<VW>(A.pre, A.wt, A.D, tpr, pre);
#pragma unroll
    for (int k = 0; k < kCols; ++k) sums[0][k] = sums[1][k] = sums[2][k] = 0.0f;
    for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows; base += (int64_t)gridDim.x * groups) {
        const bool there = base + group < A.rows;
        const int64_t row = there ? base + group : A.rows - 1;
        float y[kCols], uh[kCols], g[kCols], dy[kCols], dz[kCols], f[kCols], df[kCols], ru = 0.0f;
        load_row<TX, VW>(A.x, row, A.sx, A.D, tpr, y);
        load_row<TU, VW>(A.u, row, A.su, A.D, tpr, uh);
        load_row<TU, VW>(A.gate, row, A.sg, A.D, tpr, g);
        load_row<TX, VW>(A.dy, row, A.sdy, A.D, tpr, dy);
        load_row<TU, VW>(A.dz, row, A.sdz, A.D, tpr, dz);
        if (A.u) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < kCols; ++k) s = fmaf(uh[k], uh[k], s);
            ru = __builtin_amdgcn_rsqf(fmaf(row_sum(s, tpr, lds[0]), inv, A.eps));
#pragma unroll
            for (int k = 0; k < kCols; ++k) {
                uh[k] *= ru;
                f[k] = 1.0f;
                df[k] = 0.0f;
                if (A.gate) gate_of(A.fn, g[k], f[k], df[k]);
                y[k] = fmaf(scale[k] * f[k], post[k] * uh[k], y[k]);
            }
        }
        if (A.dz) {
            float s = 0.0f, t = 0.0f;
#pragma unroll
            for (int k = 0; k < kCols; ++k) {
                s = fmaf(y[k], y[k], s);
                t = fmaf(dz[k] * pre[k], y[k], t);
            }
            const float ry = __builtin_amdgcn_rsqf(fmaf(row_sum(s, tpr, lds[1]), inv, A.eps));
            const float mean = row_sum(t, tpr, lds[2]) * inv * ry;
#pragma unroll
            for (int k = 0; k < kCols; ++k) {
                const float yh = y[k] * ry;
                if (there) sums[2][k] = fmaf(dz[k], yh, sums[2][k]);
                dy[k] = fmaf(ry, fmaf(-yh, mean, dz[k] * pre[k]), dy[k]);
            }
        }
        if (there) store_row<TX, VW>(A.dx, row, A.D, tpr, dy);
        if (A.u) {
            float w[kCols], s = 0.0f;
#pragma unroll
            for (int k = 0; k < kCols; ++k) {
                w[k] = dy[k] * scale[k] * f[k];
                const float vh = post[k] * uh[k];
                if (there) {
                    sums[0][k] = fmaf(dy[k] * f[k], vh, sums[0][k]);
                    sums[1][k] = fmaf(w[k], uh[k], sums[1][k]);
                }
                g[k] = dy[k] * scale[k] * vh * df[k];
                w[k] *= post[k];
                s = fmaf(w[k], uh[k], s);
            }
            const float mean = row_sum(s, tpr, lds[3]) * inv;
#pragma unroll
            for (int k = 0; k < kCols; ++k) w[k] = ru * fmaf(-uh[k], mean, w[k]);
            if (there) {
                store_row<TU, VW>(A.du, row, A.D, tpr, w);
                if (A.gate) store_row<TU, VW>(A.dgate, row, A.D, tpr, g);
            }
        } else if (tpr > 64) __syncthreads();                  // the two sums of this row share one barrier's worth of distance to the next row's
    }
    // a workgroup's column sums: rows side by side in it are folded through LDS first
    for (int n = 0; n < 3; ++n) {
        if (groups > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kCols; ++k) fold[k * 256 + threadIdx.x] = sums[n][k];
            __syncthreads();
            if (group == 0)
#pragma unroll
                for (int k = 0; k < kCols; ++k)
                    for (int o = 1; o < groups; ++o) sums[n][k] += fold[k * 256 + o * tpr + threadIdx.x];
        }
        if (group == 0) {
            float* to = A.part + ((int64_t)blockIdx.x * 3 + n) * A.D;
#pragma unroll
            for (int j = 0; j < kCols / VW; ++j)
#pragma unroll
                for (int k = 0; k < VW; ++k) {
                    const int c = column<VW>(tpr, j) + k;
                    if (c < A.D) to[c] = sums[n][j * VW + k];
                }
        }
    }
}

// the partial rows added up, 64 columns a workgroup, 16 strips of rows joined in a fixed order; blockIdx.y: which of the three
__global__ __launch_bounds__(1024) void k_column_sums(const float* part, int blocks, int D, void* dscale, void* dpost, void* dpre, int wt) {
    __shared__ float strip[16][64];
    const int col = threadIdx.x & 63, s = threadIdx.x >> 6, d = blockIdx.x * 64 + col, n = blockIdx.y;
    void* out = n == 0 ? dscale : n == 1 ? dpost : dpre;
    if (!out) return;
    float sum = 0.0f;
    if (d < D)
        for (int r = s; r < blocks; r += 16) sum += part[((int64_t)r * 3 + n) * D + d];
    strip[s][col] = sum;
    __syncthreads();
    if (s || d >= D) return;
    for (int k = 1; k < 16; ++k) sum += strip[k][col];
    if (wt == PLMPM_NN_F32) ((float*)out)[d] = sum;
    else if (wt == PLMPM_NN_BF16) from_f(sum, ((bf16*)out)[d]);
    else from_f(sum, ((f16*)out)[d]);
}

int row_threads(int64_t width) {
    int tpr = 4;
    while (tpr * kCols < width) tpr *= 2;
    return tpr;
}
int block_of(int tpr) { return tpr > 256 ? tpr : 256; }
int blocks_of(const plmpm_norm* n) {
    const int groups = block_of(row_threads(n->width)) / row_threads(n->width);
    const int64_t need = (n->rows + groups - 1) / groups;
    return (int)std::min<int64_t>(need, kMaxBlocks);
}

int check(const plmpm_norm* n, bool backward) {
    NN_REQUIRE(n, "norm: null argument");
    const int tx = n->x_dtype, tu = n->u_dtype;
    NN_REQUIRE(tx >= 0 && tx <= PLMPM_NN_F16 && tu >= 0 && tu <= PLMPM_NN_F16 && n->w_dtype >= 0 && n->w_dtype <= PLMPM_NN_F16, "norm: unknown dtype");
    NN_REQUIRE(tx == tu || tx == PLMPM_NN_F32, "norm: u has x's type, or 16 bits next to a float x");
    NN_REQUIRE(n->rows >= 0 && n->width >= 0, "norm: negative size");
    NN_REQUIRE(n->width <= kMaxWidth, "norm: width %lld, at most %d", (long long)n->width, kMaxWidth);
    NN_REQUIRE(n->gate_fn >= 0 && n->gate_fn <= PLMPM_GATE_SILU, "norm: unknown gate function %d", n->gate_fn);
    NN_REQUIRE(n->eps >= 0 && n->eps < 1e30, "norm: eps has to be zero or above, and finite");
    if (!n->rows || !n->width) return 0;
    NN_REQUIRE(n->x, "norm: x is needed");
    NN_REQUIRE(n->u || (!n->gate && !n->scale && !n->post), "norm: gate, scale and post go with u");
    if (backward) {
        NN_REQUIRE(n->dx && (!n->u || n->du) && (!n->gate || n->dgate), "norm backward: dx, du (with u) and dgate (with gate) are needed");
        NN_REQUIRE(!n->dz || n->pre, "norm backward: dz goes with pre");
    } else {
        NN_REQUIRE((!n->u || n->y) && (!n->z || n->pre) && (n->u || n->z), "norm forward: y goes with u, z with pre, and one of them is needed");
    }
    for (const void* p : {n->x, n->dy, (const void*)n->y, (const void*)n->dx}) NN_REQUIRE((uintptr_t)p % dtype_size(tx) == 0, "norm: a pointer is not aligned to its type");
    for (const void* p : {n->u, n->gate, n->dz, (const void*)n->z, (const void*)n->du, (const void*)n->dgate})
        NN_REQUIRE((uintptr_t)p % dtype_size(tu) == 0, "norm: a pointer is not aligned to its type");
    for (const void* p : {n->scale, n->post, n->pre}) NN_REQUIRE((uintptr_t)p % dtype_size(n->w_dtype) == 0, "norm: a pointer is not aligned to its type");
    return 0;
}

// columns an access: 8 (16 bytes of a 16-bit type), 2, or 1, by what widths, pointers and strides keep to
int vector_of(const plmpm_norm* n, bool backward) {
    const int zx = dtype_size(n->x_dtype), zu = dtype_size(n->u_dtype), zw = dtype_size(n->w_dtype);
    for (int vw : {8, 2}) {
        bool ok = n->width % vw == 0;
        const auto keeps = [&](const void* p, int64_t stride, int size) { if (p) ok = ok && aligned_to(p, stride, size) >= std::min(16, vw * size); };
        keeps(n->x, n->stride_x, zx);
        keeps(n->u, n->stride_u, zu);
        keeps(n->gate, n->stride_gate, zu);
        for (const void* p : {n->scale, n->post, n->pre}) keeps(p, n->width, zw);
        if (backward) {
            keeps(n->dy, n->stride_dy, zx);
            keeps(n->dz, n->stride_dz, zu);
            keeps(n->dx, n->width, zx);
            keeps(n->du, n->width, zu);
            keeps(n->dgate, n->width, zu);
        } else {
            keeps(n->y, n->width, zx);
            keeps(n->z, n->width, zu);
        }
        if (ok) return vw;
    }
    return 1;
}

template <class TX, class TU, int VW> void launch(const NormArgs& A, bool backward, int blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks), block((unsigned)block_of(A.tpr));
    if (backward) hipLaunchKernelGGL((k_norm_backward<TX, TU, VW>), grid, block, 0, st, A);
    else hipLaunchKernelGGL((k_norm_forward<TX, TU, VW>), grid, block, 0, st, A);
}
template <class TX, class TU> void launch(const NormArgs& A, int vw, bool backward, int blocks, hipStream_t st) {
    if (vw == 8) launch<TX, TU, 8>(A, backward, blocks, st);
    else if (vw == 2) launch<TX, TU, 2>(A, backward, blocks, st);
    else launch<TX, TU, 1>(A, backward, blocks, st);
}

int run(const plmpm_norm* n, bool backward, hipStream_t st) {
    if (check(n, backward)) return -1;
    if (!n->width) return 0;
    if (!n->rows && !backward) return 0;
    size_t need = 0;
    if (backward && plmpm_norm_workspace(n, &need)) return -1;
    NN_REQUIRE(n->workspace_bytes >= need && (n->workspace || !need), "norm: the workspace has %zu bytes, %zu are needed", n->workspace_bytes, need);
    NormArgs A{};
    A.x = n->x; A.u = n->u; A.gate = n->gate; A.scale = n->scale; A.post = n->post; A.pre = n->pre; A.dy = n->dy; A.dz = n->dz;
    A.y = n->y; A.z = n->z; A.dx = n->dx; A.du = n->du; A.dgate = n->dgate; A.part = (float*)n->workspace;
    A.rows = n->rows; A.sx = n->stride_x; A.su = n->stride_u; A.sg = n->stride_gate; A.sdy = n->stride_dy; A.sdz = n->stride_dz;
    A.D = (int)n->width; A.fn = n->gate_fn; A.wt = n->w_dtype; A.eps = (float)n->eps;
    A.tpr = row_threads(n->width);
    const int vw = vector_of(n, backward), blocks = blocks_of(n);
    if (blocks) {
        if (n->x_dtype == PLMPM_NN_BF16) launch<bf16, bf16>(A, vw, backward, blocks, st);
        else if (n->x_dtype == PLMPM_NN_F16) launch<f16, f16>(A, vw, backward, blocks, st);
        else if (n->u_dtype == PLMPM_NN_F32) launch<float, float>(A, vw, backward, blocks, st);
        else if (n->u_dtype == PLMPM_NN_BF16) launch<float, bf16>(A, vw, backward, blocks, st);
        else launch<float, f16>(A, vw, backward, blocks, st);
    }
    if (backward && (n->dscale || n->dpost || n->dpre))      // (without rows the weights' gradients are zeros)
        hipLaunchKernelGGL(k_column_sums, dim3((unsigned)((A.D + 63) / 64), 3), dim3(1024), 0, st, (const float*)A.part, blocks, A.D, n->dscale, n->dpost, n->dpre, A.wt);
    NN_LAUNCHED(backward ? "norm backward" : "norm forward");
    return 0;
}

}  // namespace

extern "C" {

int plmpm_norm_workspace(const plmpm_norm* n, size_t* bytes) {
    NN_REQUIRE(n && bytes, "norm: null argument");
    NN_REQUIRE(n->rows >= 0 && n->width >= 0 && n->width <= kMaxWidth, "norm: rows %lld x width %lld: negative, or wider than %d", (long long)n->rows, (long long)n->width, kMaxWidth);
    *bytes = n->width ? (size_t)blocks_of(n) * 3 * n->width * sizeof(float) : 0;
    return 0;
}
int plmpm_norm_forward(const plmpm_norm* n, void* hip_stream) { return run(n, false, (hipStream_t)hip_stream); }
int plmpm_norm_backward(const plmpm_norm* n, void* hip_stream) { return run(n, true, (hipStream_t)hip_stream); }

}  // extern "C"
