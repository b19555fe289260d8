// Gated linear recurrence (include/plmpm_policy.h: plmpm_scan) and its backward pass.
//
//   a_t = exp(la_t), la_t = -c softplus(decay) sigmoid(r_t);   h_t = a_t h_{t-1} + m_t sigmoid(i_t) x_t,  m_t = sqrt(1 - a_t^2)
//
// A run of steps acts on the state as h -> A h + H (A the product of its a, H what it ends with from zero), and runs compose, so a
// tile of 64 steps is cut into sub-runs of S steps, one a wave: every wave reduces its sub-run from registers to (A, H), the
// channels' owners chain the sub-runs through LDS from the tile's state, and every wave replays its sub-run from the state it
// starts with.  Inputs are read once and stay in registers between the two walks.
// A reset makes the run forget what came before, also a NaN: its A is then -0 (every genuine A is +0 or above), and whoever
// composes runs takes H alone where the sign is set.
#include "plmpm_nn.h"

using namespace plbnn;

namespace {

constexpr int kTile = 64;               // steps of a tile, forward and backward: the checkpoints' spacing
constexpr int kMaxWaves = 8;

struct ScanArgs {
    const void* in[3];
    int64_t sb[3], st[3];
    const float *decay, *h0;
    const uint8_t* reset;
    void* h;
    float *h_last, *ckpt;
    const void* dh;
    const float* dlast;
    void* out[3];                       // dx, dr, di
    float *part, *dh0;                  // part: [tiles][batch][width] sums of dla sigmoid(r)
    int64_t B, T;
    int D, cblks, tiles;
    float c;
};

__device__ __forceinline__ bool forgets(float A) { return (as_u(A) >> 31) != 0; }
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }

// sigmoid(r), sigmoid(i), log2 a, a and 1 - a^2.  1 - a^2 = -expm1(2 ln2 l2) cancels for a near 1: above l2 = -0.18 (a^2 > 0.78) it
// comes from a cubic for -expm1(2 ln2 l) / l, the polynomial through its values at the Chebyshev points (relative error 2.7e-7, half
// of that in the root); below, 1 - a a is off by at most 2^-24 / 0.22.
struct Gates { float sr, si, l2, a, m2; };
__device__ __forceinline__ Gates gates(float r, float i, float k2) {
    Gates g;
    g.sr = sigmoid_fast(r);
    g.si = sigmoid_fast(i);
    g.l2 = k2 * g.sr;
    g.a = exp2_fast(g.l2);
    const float q = fmaf(fmaf(fmaf(-0.13934674859046936f, g.l2, -0.4424225986003876f), g.l2, -0.960848331451416f), g.l2, -1.3862940073013306f);
    g.m2 = g.l2 >= -0.18033688f ? g.l2 * q : fmaf(-g.a, g.a, 1.0f);
    return g;
}

// which of the S steps from t on are resets: a bit each (uniform over the wave)
template <int S> __device__ __forceinline__ unsigned reset_bits(const ScanArgs& A, int64_t b, int64_t t) {
    const int lane = threadIdx.x & 63;
    const int hit = lane < S && t + lane < A.T ? A.reset[b * A.T + t + lane] != 0 : 0;
    return (unsigned)__ballot(hit);
}

template <class T, int VEC, int S, bool RESET>
__global__ __launch_bounds__(kTile / S * 64) void k_scan_forward(ScanArgs A) {
    constexpr int NCH = 64 * VEC;
    __shared__ float sA[kTile / S][NCH], sH[kTile / S][NCH], carry[NCH];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t b = blockIdx.x / A.cblks;
    const int first = (int)(blockIdx.x % A.cblks) * NCH, d0 = first + lane * VEC;
    const bool live = d0 < A.D;                          // VEC divides the width: a lane's channels are all there or none is
    const int dl = live ? d0 : 0;
    float k2[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) k2[v] = -A.c * kLog2e * softplus(A.decay[dl + v]);
    for (int ch = threadIdx.x; ch < NCH; ch += blockDim.x)
        carry[ch] = A.h0 && first + ch < A.D ? A.h0[b * A.D + first + ch] : 0.0f;
    __syncthreads();
    for (int tile = 0; tile < A.tiles; ++tile) {
        const int64_t t0 = (int64_t)tile * kTile + wave * S;
        Vec<T, VEC> raw[3][S];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const T* p = (const T*)A.in[k] + b * A.sb[k];
#pragma unroll
            for (int s = 0; s < S; ++s) raw[k][s].load(p + (t0 + s < A.T ? t0 + s : A.T - 1) * A.st[k] + dl);
        }
        const unsigned cut = RESET ? reset_bits<S>(A, b, t0) : 0u;
        float a[S][VEC], u[S][VEC], PA[VEC], PH[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) { PA[v] = 1.0f; PH[v] = 0.0f; }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[VEC], r[VEC], i[VEC];
            raw[0][s].get(x);
            raw[1][s].get(r);
            raw[2][s].get(i);
            const bool there = t0 + s < A.T;             // a step behind the end leaves the state as it is
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Gates g = gates(r[v], i[v], k2[v]);
                a[s][v] = there ? g.a : 1.0f;
                u[s][v] = there ? __builtin_amdgcn_sqrtf(g.m2) * g.si * x[v] : 0.0f;
                if (RESET && (cut >> s & 1)) {
                    u[s][v] = g.si * x[v];
                    PA[v] = -0.0f;
                    PH[v] = u[s][v];
                } else {
                    PA[v] *= a[s][v];
                    PH[v] = fmaf(a[s][v], PH[v], u[s][v]);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) { sA[wave][lane * VEC + v] = PA[v]; sH[wave][lane * VEC + v] = PH[v]; }
        __syncthreads();
        for (int ch = threadIdx.x; ch < NCH; ch += blockDim.x) {
            float c = carry[ch];
            if (A.ckpt && first + ch < A.D) A.ckpt[((int64_t)tile * A.B + b) * A.D + first + ch] = c;
            for (int w = 0; w < waves; ++w) {
                const float pa = sA[w][ch], ph = sH[w][ch];
                sA[w][ch] = c;
                c = forgets(pa) ? ph : fmaf(pa, c, ph);
            }
            carry[ch] = c;
            if (A.h_last && tile == A.tiles - 1 && first + ch < A.D) A.h_last[b * A.D + first + ch] = c;
        }
        __syncthreads();
        float now[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) now[v] = sA[wave][lane * VEC + v];
        T* out = (T*)A.h + (b * A.T + t0) * A.D + d0;
#pragma unroll
        for (int s = 0; s < S; ++s) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) now[v] = RESET && (cut >> s & 1) ? u[s][v] : fmaf(a[s][v], now[v], u[s][v]);
            if (live && t0 + s < A.T) {
                Vec<T, VEC> o;
                o.set(now);
                o.store(out + (int64_t)s * A.D);
            }
        }
    }
}

// Backward: g_t = dh_t + a_{t+1} g_{t+1}, walked from the end.  With e_t = a_t g_t as what a step hands to the one before it, a run acts
// on what comes in from behind as e -> A e + E with the same A, so both walks (forward again from the tile's checkpoint, which gives
// h_{t-1} in 32 bits, and backward) go through one exchange.
//   dx = g m s_i   di = g m x s_i (1 - s_i)   dla = g (a h_{t-1} - s_i x a^2 / m)   dr = dla la (1 - s_r)
// For la -> 0 the product la a^2 / m goes to 0 (m ~ sqrt(-2 la)): where m is 0 that term is left out.
template <class T, int VEC, int S, bool RESET>
__global__ __launch_bounds__(kTile / S * 64) void k_scan_backward(ScanArgs A) {
    constexpr int NCH = 64 * VEC;
    __shared__ float sA[kTile / S][NCH], sH[kTile / S][NCH], sE[kTile / S][NCH], carry[NCH];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t b = blockIdx.x / A.cblks;
    const int first = (int)(blockIdx.x % A.cblks) * NCH, d0 = first + lane * VEC;
    const bool live = d0 < A.D;
    const int dl = live ? d0 : 0;
    float k2[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) k2[v] = -A.c * kLog2e * softplus(A.decay[dl + v]);
    for (int ch = threadIdx.x; ch < NCH; ch += blockDim.x)
        carry[ch] = A.dlast && first + ch < A.D ? A.dlast[b * A.D + first + ch] : 0.0f;
    __syncthreads();
    for (int tile = A.tiles - 1; tile >= 0; --tile) {
        const int64_t t0 = (int64_t)tile * kTile + wave * S;
        Vec<T, VEC> raw[3][S], rawg[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int64_t t = t0 + s < A.T ? t0 + s : A.T - 1;
#pragma unroll
            for (int k = 0; k < 3; ++k) raw[k][s].load((const T*)A.in[k] + b * A.sb[k] + t * A.st[k] + dl);
            if (A.dh) rawg[s].load((const T*)A.dh + (b * A.T + t) * A.D + dl);
            else rawg[s].zero();
        }
        const unsigned cut = RESET ? reset_bits<S>(A, b, t0) : 0u;
        float a[S][VEC], m2[S][VEC], sr[S][VEC], si[S][VEC], PA[VEC], PH[VEC], PE[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) { PA[v] = 1.0f; PH[v] = PE[v] = 0.0f; }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[VEC], r[VEC], i[VEC];
            raw[0][s].get(x);
            raw[1][s].get(r);
            raw[2][s].get(i);
            const bool there = t0 + s < A.T;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Gates g = gates(r[v], i[v], k2[v]);
                a[s][v] = there ? g.a : 1.0f;
                m2[s][v] = there ? g.m2 : 0.0f;
                sr[s][v] = g.sr;
                si[s][v] = g.si;
                const float u = there ? __builtin_amdgcn_sqrtf(g.m2) * g.si * x[v] : 0.0f;
                if (RESET && (cut >> s & 1)) {
                    a[s][v] = 0.0f;
                    m2[s][v] = 1.0f;
                    PA[v] = -0.0f;
                    PH[v] = g.si * x[v];
                } else {
                    PA[v] *= a[s][v];
                    PH[v] = fmaf(a[s][v], PH[v], u);
                }
            }
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            float g[VEC];
            rawg[s].get(g);
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                PE[v] = RESET && (cut >> s & 1) ? 0.0f : t0 + s < A.T ? a[s][v] * (g[v] + PE[v]) : PE[v];
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            sA[wave][lane * VEC + v] = PA[v];
            sH[wave][lane * VEC + v] = PH[v];
            sE[wave][lane * VEC + v] = PE[v];
        }
        __syncthreads();
        for (int ch = threadIdx.x; ch < NCH; ch += blockDim.x) {
            float e = carry[ch], c = first + ch < A.D ? A.ckpt[((int64_t)tile * A.B + b) * A.D + first + ch] : 0.0f;
            for (int w = waves - 1; w >= 0; --w) {
                const float pa = sA[w][ch], pe = sE[w][ch];
                sE[w][ch] = e;
                e = forgets(pa) ? pe : fmaf(pa, e, pe);
            }
            for (int w = 0; w < waves; ++w) {
                const float pa = sA[w][ch], ph = sH[w][ch];
                sA[w][ch] = c;
                c = forgets(pa) ? ph : fmaf(pa, c, ph);
            }
            carry[ch] = e;
            if (A.dh0 && tile == 0 && first + ch < A.D) A.dh0[b * A.D + first + ch] = e;
        }
        __syncthreads();
        float now[VEC], e[VEC], hp[S][VEC], sum[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            now[v] = sA[wave][lane * VEC + v];
            e[v] = sE[wave][lane * VEC + v];
            sum[v] = 0.0f;
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[VEC];
            raw[0][s].get(x);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                hp[s][v] = now[v];
                const float u = __builtin_amdgcn_sqrtf(m2[s][v]) * si[s][v] * x[v];
                now[v] = RESET && (cut >> s & 1) ? u : fmaf(a[s][v], now[v], u);
            }
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            float x[VEC], g[VEC], dx[VEC], dr[VEC], di[VEC];
            raw[0][s].get(x);
            rawg[s].get(g);
            const bool there = t0 + s < A.T;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                g[v] = (there ? g[v] : 0.0f) + e[v];
                const bool reset = RESET && (cut >> s & 1);
                e[v] = reset ? 0.0f : a[s][v] * g[v];
                const float inv = m2[s][v] > 0.0f ? __builtin_amdgcn_rsqf(m2[s][v]) : 0.0f;
                const float sx = si[s][v] * x[v], m = m2[s][v] * inv, gm = g[v] * m;
                dx[v] = gm * si[s][v];
                di[v] = gm * sx * (1.0f - si[s][v]);
                const float dla = reset || !there ? 0.0f : g[v] * (a[s][v] * hp[s][v] - sx * (a[s][v] * a[s][v] * inv));
                dr[v] = dla * (k2[v] * kLn2 * sr[s][v]) * (1.0f - sr[s][v]);
                sum[v] += dla * sr[s][v];
            }
            if (live && there) {
                const int64_t at = (b * A.T + t0 + s) * A.D + d0;
                Vec<T, VEC> o;
                o.set(dx); o.store((T*)A.out[0] + at);
                o.set(dr); o.store((T*)A.out[1] + at);
                o.set(di); o.store((T*)A.out[2] + at);
            }
        }
        // the tile's share of d decay: one row of `part`, summed over the waves (sH is free: its last reader is behind the barrier)
#pragma unroll
        for (int v = 0; v < VEC; ++v) sH[wave][lane * VEC + v] = sum[v];
        __syncthreads();
        for (int ch = threadIdx.x; ch < NCH; ch += blockDim.x)
            if (first + ch < A.D) {
                float p = 0.0f;
                for (int w = 0; w < waves; ++w) p += sH[w][ch];
                A.part[((int64_t)tile * A.B + b) * A.D + first + ch] = p;
            }
        __syncthreads();
    }
}

// d decay[d] = -c sigmoid(decay[d]) * (sum of column d of part[rows][D]): 64 columns and 16 strips of rows a workgroup, strips joined in a
// fixed order
__global__ __launch_bounds__(1024) void k_decay_grad(const float* part, const float* decay, float* out, int64_t rows, int D, float c) {
    __shared__ float strip[16][64];
    const int col = threadIdx.x & 63, s = threadIdx.x >> 6, d = blockIdx.x * 64 + col;
    float sum = 0.0f;
    if (d < D)
        for (int64_t r = s; r < rows; r += 16) sum += part[r * D + d];
    strip[s][col] = sum;
    __syncthreads();
    if (s == 0 && d < D) {
        for (int k = 1; k < 16; ++k) sum += strip[k][col];
        out[d] = -c * sigmoid_fast(decay[d]) * sum;
    }
}

template <class T, int VEC, int S, bool RESET> void launch(const ScanArgs& A, bool backward, hipStream_t st) {
    const int64_t need = (A.T + S - 1) / S;
    const int waves = (int)(need < kTile / S ? need : kTile / S);
    const dim3 grid((unsigned)(A.B * A.cblks)), block((unsigned)(waves * 64));
    if (backward) hipLaunchKernelGGL((k_scan_backward<T, VEC, S, RESET>), grid, block, 0, st, A);
    else hipLaunchKernelGGL((k_scan_forward<T, VEC, S, RESET>), grid, block, 0, st, A);
}
template <class T, int VEC> void launch(const ScanArgs& A, bool backward, hipStream_t st) {
    if (A.reset) launch<T, VEC, 8, true>(A, backward, st);
    else launch<T, VEC, 8, false>(A, backward, st);
}
template <class T> void launch(const ScanArgs& A, int vec, bool backward, hipStream_t st) {
    if (vec == 2) launch<T, 2>(A, backward, st);
    else launch<T, 1>(A, backward, st);
}

// channels a lane: 2 where rows and pointers keep to it and a wave's 128 channels are not mostly behind the width
int vector_of(const plmpm_scan* s, bool backward) {
    const int size = dtype_size(s->dtype);
    int bytes = 16;
    const void* in[3] = {s->x, s->r, s->i};
    for (int k = 0; k < 3; ++k) bytes = std::min(bytes, std::min(aligned_to(in[k], s->stride_b[k], size), aligned_to(in[k], s->stride_t[k], size)));
    if (backward) for (const void* p : {(const void*)s->dh, (const void*)s->dx, (const void*)s->dr, (const void*)s->di}) bytes = std::min(bytes, aligned_to(p, s->width, size));
    else bytes = std::min(bytes, aligned_to(s->h, s->width, size));
    return s->width % 2 == 0 && s->width >= 128 && bytes >= 2 * size ? 2 : 1;
}

int check(const plmpm_scan* s, bool backward, bool pointers) {
    NN_REQUIRE(s, "scan: null argument");
    NN_REQUIRE(s->dtype >= PLMPM_NN_F32 && s->dtype <= PLMPM_NN_F16, "scan: unknown dtype %d", s->dtype);
    NN_REQUIRE(s->batch >= 0 && s->steps >= 0 && s->width >= 0, "scan: negative size");
    NN_REQUIRE(s->width < (1 << 30), "scan: width %lld is too large", (long long)s->width);
    NN_REQUIRE(s->steps < ((int64_t)1 << 36), "scan: %lld steps are too many", (long long)s->steps);
    NN_REQUIRE(s->batch < (1 << 30) && s->batch * ((s->width + 63) / 64) < ((int64_t)1 << 31), "scan: batch x width is too large for one launch");
    NN_REQUIRE(s->c > 0 && s->c < 1e30, "scan: c has to be positive and finite, got %g", s->c);
    if (!pointers || !s->batch || !s->steps || !s->width) return 0;
    NN_REQUIRE(s->x && s->r && s->i && s->decay, "scan: x, r, i and decay are needed");
    if (backward) NN_REQUIRE(s->checkpoint && s->dx && s->dr && s->di && s->ddecay, "scan backward: checkpoint, dx, dr, di and ddecay are needed");
    else NN_REQUIRE(s->h, "scan forward: h is needed");
    const int size = dtype_size(s->dtype);
    for (const void* p : {s->x, s->r, s->i, (const void*)s->h, s->dh, (const void*)s->dx, (const void*)s->dr, (const void*)s->di})
        NN_REQUIRE((uintptr_t)p % size == 0, "scan: a pointer is not aligned to its type");
    return 0;
}

int run(const plmpm_scan* s, bool backward, hipStream_t st) {
    if (check(s, backward, true)) return -1;
    if (!s->batch || !s->steps || !s->width) return 0;
    size_t need = 0;
    if (plmpm_scan_workspace(s, backward, &need)) return -1;
    NN_REQUIRE(s->workspace_bytes >= need && (s->workspace || !need), "scan: the workspace has %zu bytes, %zu are needed", s->workspace_bytes, need);
    ScanArgs A{};
    A.in[0] = s->x; A.in[1] = s->r; A.in[2] = s->i;
    for (int k = 0; k < 3; ++k) { A.sb[k] = s->stride_b[k]; A.st[k] = s->stride_t[k]; }
    A.decay = s->decay; A.h0 = s->h0; A.reset = s->reset;
    A.h = s->h; A.h_last = s->h_last; A.ckpt = s->checkpoint;
    A.dh = s->dh; A.dlast = s->dlast; A.out[0] = s->dx; A.out[1] = s->dr; A.out[2] = s->di;
    A.dh0 = s->dh0; A.part = (float*)s->workspace;
    A.B = s->batch; A.T = s->steps; A.D = (int)s->width; A.c = (float)s->c;
    const int vec = vector_of(s, backward);
    A.cblks = (A.D + 64 * vec - 1) / (64 * vec);
    A.tiles = (int)((s->steps + kTile - 1) / kTile);
    if (s->dtype == PLMPM_NN_F32) launch<float>(A, vec, backward, st);
    else if (s->dtype == PLMPM_NN_BF16) launch<bf16>(A, vec, backward, st);
    else launch<f16>(A, vec, backward, st);
    if (backward)
        hipLaunchKernelGGL(k_decay_grad, dim3((unsigned)((A.D + 63) / 64)), dim3(1024), 0, st, (const float*)A.part, A.decay, s->ddecay, (int64_t)A.tiles * A.B, A.D, A.c);
    NN_LAUNCHED(backward ? "scan backward" : "scan forward");
    return 0;
}

}  // namespace

extern "C" {

int plmpm_scan_workspace(const plmpm_scan* s, int backward, size_t* bytes) {
    NN_REQUIRE(bytes, "scan: null argument");
    if (check(s, backward != 0, false)) return -1;
    *bytes = backward ? (size_t)((s->steps + kTile - 1) / kTile) * s->batch * s->width * sizeof(float) : 0;
    return 0;
}
int plmpm_scan_forward(const plmpm_scan* s, void* hip_stream) { return run(s, false, (hipStream_t)hip_stream); }
int plmpm_scan_backward(const plmpm_scan* s, void* hip_stream) { return run(s, true, (hipStream_t)hip_stream); }

}  // extern "C"
