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
constexpr int kForwardBlocks = 1024;

struct NormArgs {
    const void *x, *u, *gate, *scale, *post, *pre, *dy, *dz;
    void *y, *z, *dx, *du, *dgate;
    float* part;                        // [workgroups][3][width]: dscale, dpost, dpre
    int64_t rows, sx, su, sg, sdy, sdz;
    int D, tpr, fn, wt;
    float eps;
};

// K sums over the `tpr` (a power of two) neighbouring threads that hold a row, in one exchange; `lds`: K floats a wave, another buffer for each
// exchange of a row
template <int K> __device__ __forceinline__ void row_sums(float (&v)[K], int tpr, float (*lds)[K]) {
    lane_sums<K>(v, tpr < 64 ? tpr : 64);
    if (tpr <= 64) return;
    const int wave = threadIdx.x >> 6, per = tpr >> 6, from = (wave & ~(per - 1)) + (int)(threadIdx.x & (per - 1));
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) lds[wave][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lds[from][k];
    lane_sums<K>(v, per);
}

// f(g) in place of g, and its derivative (one question a row, not one an element)
template <int VW> __device__ __forceinline__ void gates_of(int fn, float (&g)[VW], float (&df)[VW]) {
    if (fn == PLMPM_GATE_IDENTITY) {
#pragma unroll
        for (int k = 0; k < VW; ++k) df[k] = 1.0f;
    } else if (fn == PLMPM_GATE_SIGMOID) {
#pragma unroll
        for (int k = 0; k < VW; ++k) { const float both = both_sides(g[k]); g[k] = side_of(both); df[k] = product_of(both); }
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) { const float s = sigmoid_fast(g[k]); df[k] = s * fmaf(g[k], 1.0f - s, 1.0f); g[k] *= s; }
    }
}
template <int VW> __device__ __forceinline__ void gates_of(int fn, float (&g)[VW]) {
    if (fn == PLMPM_GATE_IDENTITY) return;
    if (fn == PLMPM_GATE_SIGMOID) {
#pragma unroll
        for (int k = 0; k < VW; ++k) g[k] = sigmoid_fast(g[k]);
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) g[k] *= sigmoid_fast(g[k]);
    }
}
// no gate counts as ones
template <int VW> __device__ __forceinline__ void open_gates(float (&g)[VW]) {
#pragma unroll
    for (int k = 0; k < VW; ++k) g[k] = 1.0f;
}

// The columns of a thread.  VW = 8: eight neighbouring ones in one access; where the width is no multiple of eight, the last thread with columns of
// its own takes the row's last eight, and `skip` of them are its neighbour's too: both compute and store the same values there, and only the
// neighbour counts them in sums.  Threads behind the width read the same place and count nothing.  Addresses are then those of elements, not of
// 16 bytes (global memory takes that; 2999 x 1214, fp16, forward and backward: 12.3 + 28.7 us, with accesses of 4 bytes 13.5 + 28.6).
// VW = 1, rows of less than eight: a column each, the threads behind them idle.
template <int VW, bool EVEN> struct Columns {
    int first, skip;                    // first column; how many of the VW are not this thread's to count
    bool mine;                          // it has one at all
    __device__ __forceinline__ Columns(int D, int tpr) {
        first = (int)(threadIdx.x & (tpr - 1)) * VW;
        const int over = EVEN ? 0 : first + VW - D;
        mine = EVEN || first < D;
        skip = over <= 0 ? 0 : over < VW ? over : VW;
        first -= EVEN ? 0 : over > 0 ? over : 0;
    }
    // sum of term(k, sum) over the columns that count
    template <class F> __device__ __forceinline__ float sum(F term) const {
        float s = 0.0f;
        if (EVEN || skip == 0)
#pragma unroll
            for (int k = 0; k < VW; ++k) s = term(k, s);
        else
#pragma unroll
            for (int k = 0; k < VW; ++k) s = k >= skip ? term(k, s) : s;
        return s;
    }
};

template <int VW, bool ALL, bool EVEN> __device__ __forceinline__ void load_weight(const void* w, int dtype, const Columns<VW, EVEN>& at, float* out) {
#pragma unroll
    for (int k = 0; k < VW; ++k) out[k] = 1.0f;
    if (!ALL && !w) return;
    if (dtype == PLMPM_NN_F32) { Vec<float, VW, !EVEN && VW == 8> v; v.load((const float*)w + at.first); v.get(out); }
    else if (dtype == PLMPM_NN_BF16) { Vec<bf16, VW, !EVEN && VW == 8> v; v.load((const bf16*)w + at.first); v.get(out); }
    else { Vec<f16, VW, !EVEN && VW == 8> v; v.load((const f16*)w + at.first); v.get(out); }
}
// a thread's columns of a row, loaded before the first use
template <class T, int VW, bool ALL, bool EVEN> struct Row {
    Vec<T, VW, !EVEN && VW == 8> v;
    // row `base` is the workgroup's, `mine` rows behind it this thread's (the host sees to it that the offset fits 32 bits)
    __device__ __forceinline__ void load(const void* p, int64_t base, int mine, int64_t stride, const Columns<VW, EVEN>& at) {
        if (ALL || p) v.load(at_offset((T*)p + base * stride, ((unsigned)mine * (unsigned)stride + (unsigned)at.first) * (unsigned)sizeof(T)));
        else v.zero();
    }
    // unpacked where it is used, each time: in between only the elements as they came are held
    __device__ __forceinline__ void get(float* out) {
        v.forget();
        v.get(out);
    }
};
template <class T, int VW, bool EVEN> __device__ __forceinline__ void store_row(void* p, int64_t base, int mine, int D, const Columns<VW, EVEN>& at, const float* in) {
    if (!at.mine) return;
    Vec<T, VW, !EVEN && VW == 8> v;
    v.set(in);
    v.store(at_offset((T*)p + base * D, ((unsigned)mine * (unsigned)D + (unsigned)at.first) * (unsigned)sizeof(T)));
}

// ALL: every tensor is there; EVEN: the width is what the threads hold (TPR x 8), everything keeps to 16 bytes and the rows come out even.  A condition around a load keeps the
// compiler from counting what is in flight (it then waits for everything) and holds registers: with conditions 8192 x 4096 backward
// took 220 us, without 157.
template <class TX, class TU, int VW, bool ALL, bool EVEN>
__global__ __launch_bounds__(1024) void k_norm_forward(NormArgs A) {
    __shared__ float lds[2][16][1];
    const int tpr = A.tpr, group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const int64_t step = (int64_t)gridDim.x * groups;
    const float inv = 1.0f / (float)A.D;
    const Columns<VW, EVEN> at(A.D, tpr);
    float scale[VW], post[VW], pre[VW];
    load_weight<VW, ALL, EVEN>(A.scale, A.wt, at, scale);
    load_weight<VW, ALL, EVEN>(A.post, A.wt, at, post);
    load_weight<VW, ALL, EVEN>(A.pre, A.wt, at, pre);
    Row<TX, VW, ALL, EVEN> rx;
    Row<TU, VW, ALL, EVEN> ru, rg;
    const auto fetch = [&](int64_t base) {
        const int mine = EVEN || base + group < A.rows ? group : (int)(A.rows - 1 - base);
        rx.load(A.x, base, mine, A.sx, at);
        ru.load(A.u, base, mine, A.su, at);
        rg.load(A.gate, base, mine, A.sg, at);
    };
    for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows; base += step) {
        const bool there = EVEN || base + group < A.rows;              // every thread takes part in the sums
        float y[VW], u[VW], g[VW];
        fetch(base);
        rx.get(y);
        ru.get(u);
        rg.get(g);
        if (ALL || A.u) {
            float s[1] = {at.sum([&](int k, float p) { return fmaf(u[k], u[k], p); })};
            row_sums<1>(s, tpr, lds[0]);
            const float r = __builtin_amdgcn_rsqf(fmaf(s[0], inv, A.eps));
            if (ALL || A.gate) gates_of(A.fn, g);
            else open_gates(g);
#pragma unroll
            for (int k = 0; k < VW; ++k) y[k] = fmaf(scale[k] * g[k], post[k] * (u[k] * r), y[k]);
            if (there) store_row<TX, VW, EVEN>(A.y, base, group, A.D, at, y);
        }
        if (ALL || A.z) {
            float s[1] = {at.sum([&](int k, float p) { return fmaf(y[k], y[k], p); })};
            row_sums<1>(s, tpr, lds[1]);
            const float r = __builtin_amdgcn_rsqf(fmaf(s[0], inv, A.eps));
#pragma unroll
            for (int k = 0; k < VW; ++k) y[k] = pre[k] * (y[k] * r);
            if (there) store_row<TU, VW, EVEN>(A.z, base, group, A.D, at, y);
        }
        if (!ALL && tpr > 64 && !(A.u && A.z)) __syncthreads();        // with one exchange a row its buffer is written again at once; with two, the other's barrier lies between
    }
}

template <class TX, class TU, int VW, int THREADS, bool ALL, bool EVEN>
__global__ __launch_bounds__(THREADS) void k_norm_backward(NormArgs A) {
    __shared__ float lds[2][16][1], lds2[16][2], fold[kCols * 256];
    const int tpr = A.tpr, group = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const int64_t step = (int64_t)gridDim.x * groups;
    const float inv = 1.0f / (float)A.D;
    const Columns<VW, EVEN> at(A.D, tpr);
    float scale[VW], post[VW], pre[VW], sums[3][VW];
    load_weight<VW, ALL, EVEN>(A.scale, A.wt, at, scale);
    load_weight<VW, ALL, EVEN>(A.post, A.wt, at, post);
    load_weight<VW, ALL, EVEN>(A.pre, A.wt, at, pre);
#pragma unroll
    for (int k = 0; k < VW; ++k) sums[0][k] = sums[1][k] = sums[2][k] = 0.0f;
    Row<TX, VW, ALL, EVEN> rx, rdy;
    Row<TU, VW, ALL, EVEN> ru, rg, rdz;
    const auto fetch = [&](int64_t base) {
        const int mine = EVEN || base + group < A.rows ? group : (int)(A.rows - 1 - base);
        rx.load(A.x, base, mine, A.sx, at);
        ru.load(A.u, base, mine, A.su, at);
        rg.load(A.gate, base, mine, A.sg, at);
        rdy.load(A.dy, base, mine, A.sdy, at);
        rdz.load(A.dz, base, mine, A.sdz, at);
    };
    for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows; base += step) {
        const bool there = EVEN || base + group < A.rows;
        float y[VW], dy[VW], r = 0.0f;
        fetch(base);
        rx.get(y);
        if (ALL || A.u) {
            float u[VW], g[VW];
            ru.get(u);
            float s[1] = {at.sum([&](int k, float p) { return fmaf(u[k], u[k], p); })};
            row_sums<1>(s, tpr, lds[0]);
            r = __builtin_amdgcn_rsqf(fmaf(s[0], inv, A.eps));
            ru.get(u);
            rg.get(g);
            if (ALL || A.gate) gates_of(A.fn, g);
            else open_gates(g);
#pragma unroll
            for (int k = 0; k < VW; ++k) y[k] = fmaf(scale[k] * g[k], post[k] * (u[k] * r), y[k]);
        }
        rdy.get(dy);
        if (ALL || A.dz) {
            float dz[VW];
            rdz.get(dz);
            float s[2] = {at.sum([&](int k, float p) { return fmaf(y[k], y[k], p); }),
                          at.sum([&](int k, float p) { return fmaf(dz[k] * pre[k], y[k], p); })};
            row_sums<2>(s, tpr, lds2);
            const float ry = __builtin_amdgcn_rsqf(fmaf(s[0], inv, A.eps)), mean = s[1] * inv * ry;
            rdz.get(dz);
            rdy.get(dy);
#pragma unroll
            for (int k = 0; k < VW; ++k) {
                const float yh = y[k] * ry;
                if (there) sums[2][k] = fmaf(dz[k], yh, sums[2][k]);
                dy[k] = fmaf(ry, fmaf(-yh, mean, dz[k] * pre[k]), dy[k]);
            }
        }
        if (there) store_row<TX, VW, EVEN>(A.dx, base, group, A.D, at, dy);
        if (ALL || A.u) {
            float u[VW], g[VW], df[VW];
            ru.get(u);
            rg.get(g);
            if (ALL || A.gate) gates_of(A.fn, g, df);
            else open_gates(g);
#pragma unroll
            for (int k = 0; k < VW; ++k) {
                const float uh = u[k] * r, t = dy[k] * scale[k], w = t * g[k], vh = post[k] * uh;
                if (there) {
                    sums[0][k] = fmaf(dy[k] * g[k], vh, sums[0][k]);
                    sums[1][k] = fmaf(w, uh, sums[1][k]);
                }
                if (ALL || A.gate) g[k] = t * vh * df[k];
                dy[k] = w * post[k];
            }
            float s[1] = {at.sum([&](int k, float p) { return fmaf(dy[k], u[k] * r, p); })};
            if ((ALL || A.gate) && there) store_row<TU, VW, EVEN>(A.dgate, base, group, A.D, at, g);
            row_sums<1>(s, tpr, lds[1]);
            const float mean = s[0] * inv;
            ru.get(u);
#pragma unroll
            for (int k = 0; k < VW; ++k) u[k] = r * fmaf(-(u[k] * r), mean, dy[k]);
            if (there) store_row<TU, VW, EVEN>(A.du, base, group, A.D, at, u);
        } else if (tpr > 64) __syncthreads();                  // (without u a row has one exchange: its buffer is free again behind this)
    }
    // a workgroup's column sums: rows side by side in it are folded through LDS first
    for (int n = 0; n < 3; ++n) {
        if (groups > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < VW; ++k) fold[k * 256 + threadIdx.x] = sums[n][k];
            __syncthreads();
            if (group == 0)
#pragma unroll
                for (int k = 0; k < VW; ++k)
                    for (int o = 1; o < groups; ++o) sums[n][k] += fold[k * 256 + o * tpr + threadIdx.x];
        }
        if (group == 0) {
            float* to = A.part + ((int64_t)blockIdx.x * 3 + n) * A.D + at.first;
#pragma unroll
            for (int k = 0; k < VW; ++k)
                if (EVEN || k >= at.skip) to[k] = sums[n][k];
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
#pragma unroll 8
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
    int tpr = width < kCols ? 8 : 4;       // (less than eight columns: a thread each)
    while (tpr * kCols < width) tpr *= 2;
    return tpr;
}
int block_of(int tpr) { return tpr > 256 ? tpr : 256; }
int blocks_of(const plmpm_norm* n, bool backward) {
    const int groups = block_of(row_threads(n->width)) / row_threads(n->width);
    const int64_t need = (n->rows + groups - 1) / groups;
    // backward: as many as run at once (each leaves a partial row of column sums), one a CU of 512 threads or more, two of 256: 8192 x 4096 157 us
    // with 256 workgroups, 165 with 512; 2999 x 1214 29 us with 512, 41 with 256 (27 with 768, whose sums then take 2 us more)
    const int most = !backward ? kForwardBlocks : groups == 1 && row_threads(n->width) >= 512 ? 256 : 512;
    return (int)std::min<int64_t>(need, most);
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
    const int groups = block_of(row_threads(n->width)) / row_threads(n->width);
    for (int64_t stride : {n->stride_x, n->stride_u, n->stride_gate, n->stride_dy, n->stride_dz})
        NN_REQUIRE(stride >= 0 && (groups == 1 || stride < ((int64_t)1 << 29) / groups), "norm: a row stride of %lld is negative, or too large for rows of %lld", (long long)stride, (long long)n->width);
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

// whether everything keeps to accesses of 16 bytes
bool keeps_to_16(const plmpm_norm* n, bool backward) {
    const int zx = dtype_size(n->x_dtype), zu = dtype_size(n->u_dtype), zw = dtype_size(n->w_dtype);
    bool ok = true;
    const auto keeps = [&](const void* p, int64_t stride, int size) { if (p) ok = ok && aligned_to(p, stride, size) >= 16; };
    keeps(n->x, n->stride_x, zx);
    keeps(n->u, n->stride_u, zu);
    keeps(n->gate, n->stride_gate, zu);
    for (const void* p : {n->scale, n->post, n->pre}) keeps(p, 0, zw);
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
    return ok;
}

template <class TX, class TU, int VW, bool ALL, bool EVEN> void launch(const NormArgs& A, bool backward, int blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks), block((unsigned)block_of(A.tpr));
    if (!backward) hipLaunchKernelGGL((k_norm_forward<TX, TU, VW, ALL, EVEN>), grid, block, 0, st, A);
    else if (A.tpr == 1024) hipLaunchKernelGGL((k_norm_backward<TX, TU, VW, 1024, ALL, EVEN>), grid, block, 0, st, A);
    else hipLaunchKernelGGL((k_norm_backward<TX, TU, VW, 512, ALL, EVEN>), grid, block, 0, st, A);
}
template <class TX, class TU> void launch(const NormArgs& A, bool even, bool backward, int blocks, hipStream_t st) {
    const bool all = A.u && A.gate && A.scale && A.post && A.pre && (backward ? A.dy && A.dz : A.y && A.z);
    even = even && A.D == A.tpr * kCols && A.rows % (block_of(A.tpr) / A.tpr) == 0;
    if (A.D < kCols) launch<TX, TU, 1, false, false>(A, backward, blocks, st);
    else if (all && even) launch<TX, TU, kCols, true, true>(A, backward, blocks, st);
    else if (all) launch<TX, TU, kCols, true, false>(A, backward, blocks, st);
    else launch<TX, TU, kCols, false, false>(A, backward, blocks, st);
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
    const bool even = keeps_to_16(n, backward);
    const int blocks = blocks_of(n, backward);
    if (blocks) {
        if (n->x_dtype == PLMPM_NN_BF16) launch<bf16, bf16>(A, even, backward, blocks, st);
        else if (n->x_dtype == PLMPM_NN_F16) launch<f16, f16>(A, even, backward, blocks, st);
        else if (n->u_dtype == PLMPM_NN_F32) launch<float, float>(A, even, backward, blocks, st);
        else if (n->u_dtype == PLMPM_NN_BF16) launch<float, bf16>(A, even, backward, blocks, st);
        else launch<float, f16>(A, even, backward, blocks, st);
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
    *bytes = n->width ? (size_t)blocks_of(n, true) * 3 * n->width * sizeof(float) : 0;
    return 0;
}
int plmpm_norm_forward(const plmpm_norm* n, void* hip_stream) { return run(n, false, (hipStream_t)hip_stream); }
int plmpm_norm_backward(const plmpm_norm* n, void* hip_stream) { return run(n, true, (hipStream_t)hip_stream); }

}  // extern "C"
