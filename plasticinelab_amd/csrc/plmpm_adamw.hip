// AdamW over many tensors at once (include/plmpm_policy.h: plmpm_adamw), moments in 32 or in 8 bits, gradients clipped by their global norm.
//
// One launch walks all tensors: they are cut into chunks of 2048 elements (8 us for the 20 tensors of a small policy, 11 with 4096), workgroups take equal runs of consecutive chunks, and the table of
// tensors travels in the kernel arguments (no copy to the device, nothing that a graph could find stale).  More tensors than the arguments
// hold: several launches.  Clipping adds one launch before: partial sums of squares in 64 bits, which every workgroup of the update
// adds up again in the same order -- the factor is the same for all, and the same each time.
//
// Every elementwise operation is rounded by itself, in the order written (no contraction), so an update has one bit pattern; the 8-bit codes
// depend on that where a value lies next to the border of two.
//
// 8 bits: a wave takes a block of 256 elements, four neighbours a lane; the block's largest magnitude is a wave maximum (on the bits: a
// NaN is larger than everything and stays visible in the scale).  Codes are of the root (first moment) and the fourth root (second) of the
// value over the scale: steps near zero are fine enough for sqrt(v), which a linear code would flush to 0 and blow the update up.
#include <algorithm>
#include <vector>

#include "plmpm_nn.h"

using namespace plbnn;

namespace {

constexpr int kChunk = 2048, kBlock = 256, kThreads = 256;
constexpr int kMaxTensors = 48;         // 72 bytes each + their first chunks: the kernel arguments stay below 4 KB
constexpr int kMaxGroups = 2048;        // workgroups of a launch (8 a CU)
constexpr int kNormGroups = 2048;

struct Table {
    plmpm_adamw_tensor t[kMaxTensors];
    int32_t first[kMaxTensors + 1];     // first chunk of each tensor; behind the last: their number
    int32_t count, per;                 // tensors; chunks a workgroup
};
struct Step {
    float decay, b1, b2, c1, c2, eps, lo, hi;      // decay = lr * weight_decay; c = 1 - b
    double beta_1, beta_2, lr, max_norm;
    int64_t* step;
    float* grad_norm;
    const double* partial;              // sums of squares, or null
    int partials, last;                 // last: this launch ends the step
};

__device__ __forceinline__ double power(double b, int64_t n) {
    double r = 1.0;
    for (; n; n >>= 1, b *= b) if (n & 1) r *= b;
    return r;
}

// sum over the workgroup, the same for every thread
__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kThreads / 64; ++w) v += lds[w];
    return v;
}

// the tensor that a chunk belongs to
__device__ __forceinline__ int tensor_of(const Table& tab, int chunk) {
    int lo = 0, hi = tab.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

// sum of the squares of g[at, stop): four vectors in flight a thread, then element by element
template <class T> __device__ __forceinline__ double run_squares(const T* g, int64_t at, int64_t stop) {
    constexpr int V = 16 / (int)sizeof(T), R = 4, whole = kThreads * V * R;
    double sum[2] = {0.0, 0.0};
    if (((uintptr_t)g & 15) == 0)
        for (; at + whole <= stop; at += whole) {
            Vec<T, V> v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) v[r].load(g + at + (r * kThreads + threadIdx.x) * V);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float f[V];
                v[r].get(f);
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e & 1] = fma((double)f[e], (double)f[e], sum[e & 1]);
            }
        }
    for (at += threadIdx.x; at < stop; at += kThreads) {
        const double f = (double)to_f(g[at]);
        sum[0] = fma(f, f, sum[0]);
    }
    return sum[0] + sum[1];
}

// The update's count: the launch before an update writes done + 1 into the word of those begun, which every workgroup of the update reads, and the
// update's first workgroup copies it to the word of those done, which none of them reads.  (Counting with an atomic in the update itself, the last
// workgroup to arrive, costs some 20 us for 1024 of them: they queue at the one address.)
__device__ __forceinline__ void begin_update(int64_t* step) { step[1] = step[0] + 1; }
__global__ void k_begin(int64_t* step) { begin_update(step); }

__global__ __launch_bounds__(kThreads) void k_square_sums(Table tab, double* partial, int64_t* step) {
    if (step && blockIdx.x == 0 && threadIdx.x == 0) begin_update(step);
    __shared__ double lds[kThreads / 64];
    const int begin = blockIdx.x * tab.per, end = min(begin + tab.per, tab.first[tab.count]);
    double sum = 0.0;
    int k = begin < end ? tensor_of(tab, begin) : 0;
    for (int chunk = begin; chunk < end;) {
        while (chunk >= tab.first[k + 1]) ++k;
        const plmpm_adamw_tensor& t = tab.t[k];
        const int to = min(end, tab.first[k + 1]);             // this workgroup's run of chunks in the tensor
        const int64_t at = (int64_t)(chunk - tab.first[k]) * kChunk, stop = min(t.n, (int64_t)(to - tab.first[k]) * kChunk);
        sum += t.dtype == PLMPM_NN_F32 ? run_squares((const float*)t.g, at, stop) : t.dtype == PLMPM_NN_BF16 ? run_squares((const bf16*)t.g, at, stop) : run_squares((const f16*)t.g, at, stop);
        chunk = to;
    }
    sum = block_sum(sum, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

struct Now { float k, lr1, den; };      // clip factor, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)

// one element: the moments and the weight.  Each operation rounds by itself.
__device__ __forceinline__ void update(const Step& S, const Now& N, float g, float& m, float& v, float& w) {
#pragma clang fp contract(off)
    g = g * N.k;
    const float m0 = S.b1 * m, m1 = S.c1 * g;
    m = m0 + m1;
    const float gg = g * g, v0 = S.b2 * v, v1 = S.c2 * gg;
    v = v0 + v1;
    const float root = sqrtf(v) * N.den, den = root + S.eps;
    const float pull = S.decay * w, kept = w - pull, lm = N.lr1 * m, move = lm / den;
    const float moved = kept - move;
    w = moved < S.lo ? S.lo : moved > S.hi ? S.hi : moved;      // (a NaN stays)
}

__device__ __forceinline__ float value_first(int code, float scale) {
#pragma clang fp contract(off)
    const float q = (float)code * (1.0f / 127.0f), a = q * fabsf(q);
    return a * scale;
}
__device__ __forceinline__ float value_second(int code, float scale) {
#pragma clang fp contract(off)
    const float q = (float)code * (1.0f / 255.0f), r = q * q, a = r * r;
    return a * scale;
}
// The codes are those of correctly rounded division and roots, which is some seventy instructions for the two of an element.  So first with
// the hardware's approximations (each within one unit in the last place: at most 4 units, 5e-7 relative, from the rounded ones): they give the
// same code unless they come that near to the border of two, and only then is it computed in full -- for 4 % of the waves where the codes
// lie evenly.  (With one distance for all codes, that of the largest, it was 40 %: 55 M elements 221 us, so 210.)
// ordinary: the scale is a number and lies where its reciprocal and the quotient are ordinary numbers.
__device__ __forceinline__ bool ordinary(float scale) { return scale > 1e-30f && scale < 1e30f; }
__device__ __forceinline__ bool near_border(float q) { return fmaf(q, 6e-7f, fabsf(q - rintf(q))) > 0.5f; }
__device__ __forceinline__ float exact_first(float m, float safe) { return sqrtf(fabsf(m) / safe) * 127.0f; }
__device__ __forceinline__ float exact_second(float v, float safe) { return sqrtf(sqrtf(fabsf(v) / safe)) * 255.0f; }
__device__ __forceinline__ void codes_of(const float (&m)[4], const float (&v)[4], float safe_m, float safe_v, int8_t (&cm)[4], uint8_t (&cv)[4]) {
    float qm[4], qv[4];
    const float im = __builtin_amdgcn_rcpf(safe_m), iv = __builtin_amdgcn_rcpf(safe_v);
    bool again = !ordinary(safe_m) | !ordinary(safe_v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        qm[e] = __builtin_amdgcn_sqrtf(fabsf(m[e]) * im) * 127.0f;
        qv[e] = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(fabsf(v[e]) * iv)) * 255.0f;
        again |= near_border(qm[e]) | near_border(qv[e]);
    }
    if (again)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            qm[e] = fminf(exact_first(m[e], safe_m), 127.0f);      // (a block whose scale is infinite or no number comes here: a NaN has no integer)
            qv[e] = fminf(exact_second(v[e], safe_v), 255.0f);
        }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int a = (int)rintf(qm[e]), b = (int)rintf(qv[e]);
        cm[e] = (int8_t)(m[e] < 0.0f ? -a : a);
        cv[e] = (uint8_t)(v[e] > 0.0f ? max(b, 1) : b);
    }
}

// four neighbouring elements: loaded, updated and written back, whole or up to `n`
template <class T, bool VECTOR> struct Quad {
    float g[4], w[4];
    __device__ __forceinline__ void load(const plmpm_adamw_tensor& t, int64_t at, int n) {
        if (VECTOR) {
            Vec<T, 4> v;
            v.load((const T*)t.g + at);
            v.get(g);
            if (t.master) { Vec<float, 4> m; m.load_past(t.master + at); m.get(w); }
            else { Vec<T, 4> p; p.load_past((const T*)t.p + at); p.get(w); }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                g[e] = e < n ? to_f(((const T*)t.g)[at + e]) : 0.0f;
                w[e] = e < n ? (t.master ? t.master[at + e] : to_f(((const T*)t.p)[at + e])) : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void store(const plmpm_adamw_tensor& t, int64_t at, int n) const {
        if (VECTOR) {
            Vec<T, 4> p;
            p.set(w);
            p.store_past((T*)t.p + at);
            if (t.master) { Vec<float, 4> m; m.set(w); m.store_past(t.master + at); }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) {
                    from_f(w[e], ((T*)t.p)[at + e]);
                    if (t.master) t.master[at + e] = w[e];
                }
        }
    }
};
// Moments, masters and parameters go past the caches: they are next touched a training step later, while the gradients that the norm has just read
// (plain loads) are still there for the update, and what a read-back needs stays for it.  8 bits, 55 M elements with masters: the three
// launches 384 us with ordinary accesses, 349 so; 32 bits, 18 M: 98 and 95; gradients past them too: 357 and 79 with the same gradients at each call,
// but an update behind a backward pass of 42 M elements then takes 295 us, not 287 (ordinary 298).
template <class U, bool VECTOR> __device__ __forceinline__ void load4(const U* p, int64_t at, int n, U* out) {
    if (VECTOR) { Vec<U, 4> v; v.load_past(p + at); memcpy(out, v.w, sizeof v.w); }
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = e < n ? p[at + e] : U(0);
}
template <class U, bool VECTOR> __device__ __forceinline__ void store4(U* p, int64_t at, int n, const U* in) {
    if (VECTOR) { Vec<U, 4> v; memcpy(v.w, in, sizeof v.w); v.store_past(p + at); }
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < n) p[at + e] = in[e];
}

// a chunk, `n` elements from `at`: rounds of 4 elements a thread.  Two rounds are loaded before the first is stored (the compiler cannot move a
// load over another round's stores: they might be the same memory); four rounds need twice the registers and gain nothing.
template <class T, int BITS, bool VECTOR> __device__ __forceinline__ void chunk_step(const Step& S, const Now& N, const plmpm_adamw_tensor& t, int64_t at, int n) {
    constexpr int R = VECTOR ? 2 : 1;
    for (int first = 0; first < n; first += R * kThreads * 4) {
        const int64_t from = at + first;
        const int tid4 = (int)threadIdx.x * 4, lane4 = (int)(threadIdx.x & 63) * 4;
        Quad<T, VECTOR> q[R];
        if (BITS == 32) {
            float m[R][4], v[R][4];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int e0 = r * kThreads * 4 + tid4, left = n - first - e0;
                q[r].load(t, from + e0, left);
                load4<float, VECTOR>((const float*)t.m, from + e0, left, m[r]);
                load4<float, VECTOR>((const float*)t.v, from + e0, left, v[r]);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int e0 = r * kThreads * 4 + tid4, left = n - first - e0;
#pragma unroll
                for (int e = 0; e < 4; ++e) update(S, N, q[r].g[e], m[r][e], v[r][e], q[r].w[e]);
                store4<float, VECTOR>((float*)t.m, from + e0, left, m[r]);
                store4<float, VECTOR>((float*)t.v, from + e0, left, v[r]);
                q[r].store(t, from + e0, left);
            }
        } else {
            int8_t cm[R][4];
            uint8_t cv[R][4];
            float sm[R], sv[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int e0 = r * kThreads * 4 + tid4, left = n - first - e0;
                q[r].load(t, from + e0, left);
                load4<int8_t, VECTOR>((const int8_t*)t.m, from + e0, left, cm[r]);
                load4<uint8_t, VECTOR>((const uint8_t*)t.v, from + e0, left, cv[r]);
                const int64_t blk = (from + e0) / kBlock;      // the wave's block: 64 lanes x 4
                const bool any = VECTOR || left + lane4 > 0;   // it has an element at all
                sm[r] = any ? t.m_scale[blk] : 0.0f;
                sv[r] = any ? t.v_scale[blk] : 0.0f;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int e0 = r * kThreads * 4 + tid4, left = n - first - e0;
                float m[4], v[4];
                uint32_t tm = 0, tv = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    m[e] = value_first(cm[r][e], sm[r]);
                    v[e] = value_second(cv[r][e], sv[r]);
                    update(S, N, q[r].g[e], m[e], v[e], q[r].w[e]);
                    if (!VECTOR && e >= left) continue;
                    tm = max(tm, as_u(m[e]) & 0x7fffffffu);
                    tv = max(tv, as_u(v[e]) & 0x7fffffffu);
                }
                const float top_m = as_f(wave_max(tm)), top_v = as_f(wave_max(tv));
                codes_of(m, v, top_m == 0.0f ? 1.0f : top_m, top_v == 0.0f ? 1.0f : top_v, cm[r], cv[r]);
                store4<int8_t, VECTOR>((int8_t*)t.m, from + e0, left, cm[r]);
                store4<uint8_t, VECTOR>((uint8_t*)t.v, from + e0, left, cv[r]);
                if ((VECTOR || left + lane4 > 0) && lane4 == 0) {
                    const int64_t blk = (from + e0) / kBlock;
                    t.m_scale[blk] = top_m;
                    t.v_scale[blk] = top_v;
                }
                q[r].store(t, from + e0, left);
            }
        }
    }
}

template <class T, int BITS> __device__ __forceinline__ void chunk_step(const Step& S, const Now& N, const plmpm_adamw_tensor& x, int64_t at, int n) {
    const uintptr_t low = ((uintptr_t)x.p | (uintptr_t)x.g) % (4 * sizeof(T)) | ((uintptr_t)x.master & 15) | ((uintptr_t)x.m | (uintptr_t)x.v) % (BITS == 32 ? 16 : 4);
    if (n == kChunk && low == 0) chunk_step<T, BITS, true>(S, N, x, at, n);
    else chunk_step<T, BITS, false>(S, N, x, at, n);
}

template <int BITS> __global__ __launch_bounds__(kThreads) void k_adamw(Table tab, Step S) {
    __shared__ double lds[kThreads / 64];
    const int64_t t = S.step[1];
    Now N{1.0f, (float)(S.lr / (1.0 - power(S.beta_1, t))), (float)(1.0 / sqrt(1.0 - power(S.beta_2, t)))};
    if (S.partial) {
        double sum = 0.0;
        for (int k = threadIdx.x; k < S.partials; k += kThreads) sum += S.partial[k];
        const double norm = sqrt(block_sum(sum, lds)), ratio = S.max_norm / norm;
        N.k = (float)(ratio > 1.0 ? 1.0 : ratio);              // (norm 0: ratio inf -> 1; a NaN norm stays one)
        if (S.grad_norm && S.last && blockIdx.x == 0 && threadIdx.x == 0) *S.grad_norm = (float)norm;
    }
    const int begin = blockIdx.x * tab.per, end = min(begin + tab.per, tab.first[tab.count]);
    int k = begin < end ? tensor_of(tab, begin) : 0;
    for (int chunk = begin; chunk < end; ++chunk) {
        while (chunk >= tab.first[k + 1]) ++k;
        const plmpm_adamw_tensor& x = tab.t[k];
        const int64_t at = (int64_t)(chunk - tab.first[k]) * kChunk;
        const int n = (int)min((int64_t)kChunk, x.n - at);
        if (x.dtype == PLMPM_NN_F32) chunk_step<float, BITS>(S, N, x, at, n);
        else if (x.dtype == PLMPM_NN_BF16) chunk_step<bf16, BITS>(S, N, x, at, n);
        else chunk_step<f16, BITS>(S, N, x, at, n);
    }
    if (S.last && blockIdx.x == 0 && threadIdx.x == 0) S.step[0] = t;
}

struct Values {
    const void* codes[kMaxTensors];
    const float* scales[kMaxTensors];
    float* out[kMaxTensors];
    int64_t n[kMaxTensors];
    int32_t which[kMaxTensors], first[kMaxTensors + 1], count, per;
};
__global__ __launch_bounds__(kThreads) void k_values(Values V) {
    const int begin = blockIdx.x * V.per, end = min(begin + V.per, V.first[V.count]);
    int k = 0;
    for (int chunk = begin; chunk < end; ++chunk) {
        while (chunk >= V.first[k + 1]) ++k;
        const int64_t at = (int64_t)(chunk - V.first[k]) * kChunk;
        const int n = (int)min((int64_t)kChunk, V.n[k] - at);
        const bool whole = n == kChunk && ((uintptr_t)V.codes[k] & 3) == 0 && ((uintptr_t)V.out[k] & 15) == 0;
        for (int e0 = (int)threadIdx.x * 4; e0 < n; e0 += kThreads * 4) {
            const float s = V.scales[k][(at + e0) / kBlock];
            uint8_t c[4];
            if (whole) load4<uint8_t, true>((const uint8_t*)V.codes[k], at + e0, 4, c);
            else load4<uint8_t, false>((const uint8_t*)V.codes[k], at + e0, n - e0, c);
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = V.which[k] ? value_second(c[e], s) : value_first((int8_t)c[e], s);
            if (whole) store4<float, true>(V.out[k], at + e0, 4, o);
            else store4<float, false>(V.out[k], at + e0, n - e0, o);
        }
    }
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

int check(const plmpm_adamw* a, const plmpm_adamw_tensor* tensors, int count) {
    NN_REQUIRE(a && (tensors || !count), "adamw: null argument");
    NN_REQUIRE(a->state_bits == 32 || a->state_bits == 8, "adamw: states have 32 or 8 bits, got %d", a->state_bits);
    NN_REQUIRE(count >= 0, "adamw: negative count");
    const int state = a->state_bits == 32 ? 4 : 1;
    int64_t total = 0;
    for (int k = 0; k < count; ++k) {
        const plmpm_adamw_tensor& t = tensors[k];
        NN_REQUIRE(t.n >= 0, "adamw: tensor %d has a negative size", k);
        if (!t.n) continue;
        NN_REQUIRE(t.dtype >= PLMPM_NN_F32 && t.dtype <= PLMPM_NN_F16, "adamw: tensor %d: unknown dtype %d", k, t.dtype);
        const int size = dtype_size(t.dtype);
        NN_REQUIRE(t.p && t.g && t.m && t.v && (state == 4 || (t.m_scale && t.v_scale)), "adamw: tensor %d has a null pointer", k);
        NN_REQUIRE(!t.master || t.dtype != PLMPM_NN_F32, "adamw: tensor %d: a master copy goes with 16-bit parameters", k);
        NN_REQUIRE(((uintptr_t)t.p | (uintptr_t)t.g) % size == 0 && ((uintptr_t)t.m | (uintptr_t)t.v) % state == 0 && ((uintptr_t)t.master | (uintptr_t)t.m_scale | (uintptr_t)t.v_scale) % 4 == 0,
                   "adamw: tensor %d: a pointer is not aligned to its type", k);
        total += chunks_of(t.n);
        NN_REQUIRE(total < (1 << 30), "adamw: too many elements for one call");
    }
    return 0;
}

// fills the table with tensors from `from` on; -> the next one.  Empty tensors are left out.
int fill(Table& tab, const plmpm_adamw_tensor* tensors, int count, int from) {
    tab.count = 0;
    tab.first[0] = 0;
    for (; from < count && tab.count < kMaxTensors; ++from) {
        if (!tensors[from].n) continue;
        tab.t[tab.count] = tensors[from];
        tab.first[tab.count + 1] = tab.first[tab.count] + (int32_t)chunks_of(tensors[from].n);
        ++tab.count;
    }
    return from;
}
int groups_of(int chunks, int most, int32_t& per) {
    per = (chunks + most - 1) / most;
    return per ? (chunks + per - 1) / per : 0;
}

int launches_of(const plmpm_adamw_tensor* tensors, int count) {
    int live = 0;
    for (int k = 0; k < count; ++k) live += tensors[k].n > 0;
    return (live + kMaxTensors - 1) / kMaxTensors;
}

}  // namespace

extern "C" {

int plmpm_adamw_workspace(const plmpm_adamw* a, const plmpm_adamw_tensor* tensors, int count, size_t* bytes) {
    NN_REQUIRE(a && bytes && (tensors || !count) && count >= 0, "adamw: null argument");
    *bytes = a->max_norm > 0 ? (size_t)launches_of(tensors, count) * kNormGroups * sizeof(double) : 0;
    return 0;
}

int plmpm_adamw_step(const plmpm_adamw* a, const plmpm_adamw_tensor* tensors, int count, void* hip_stream) {
    if (check(a, tensors, count)) return -1;
    NN_REQUIRE(a->step, "adamw: step is needed");
    NN_REQUIRE(a->beta_1 >= 0 && a->beta_1 < 1 && a->beta_2 >= 0 && a->beta_2 < 1, "adamw: betas lie in [0, 1)");
    NN_REQUIRE(a->epsilon >= 0, "adamw: epsilon is zero or above");
    NN_REQUIRE(a->max_norm >= 0, "adamw: max_norm is zero (no clipping) or above");
    NN_REQUIRE(a->lo <= a->hi, "adamw: bounds are (lower, upper)");
    size_t need = 0;
    if (plmpm_adamw_workspace(a, tensors, count, &need)) return -1;
    NN_REQUIRE(a->workspace_bytes >= need && (a->workspace || !need), "adamw: the workspace has %zu bytes, %zu are needed", a->workspace_bytes, need);
    NN_REQUIRE((uintptr_t)a->workspace % 8 == 0, "adamw: the workspace is not aligned to 8 bytes");
    const int launches = launches_of(tensors, count);
    if (!launches) return 0;
    hipStream_t st = (hipStream_t)hip_stream;
    Table tab;
    double* partial = (double*)a->workspace;
    int partials = 0;
    if (a->max_norm > 0)
        for (int from = 0, n = 0; n < launches; ++n) {
            from = fill(tab, tensors, count, from);
            const int groups = groups_of(tab.first[tab.count], kNormGroups, tab.per);
            hipLaunchKernelGGL(k_square_sums, dim3((unsigned)groups), dim3(kThreads), 0, st, tab, partial + partials, n ? nullptr : a->step);
            partials += groups;
        }
    else
        hipLaunchKernelGGL(k_begin, dim3(1), dim3(1), 0, st, a->step);
    Step S{};
    S.decay = (float)(a->lr * a->weight_decay);
    S.b1 = (float)a->beta_1; S.b2 = (float)a->beta_2; S.c1 = (float)(1.0 - a->beta_1); S.c2 = (float)(1.0 - a->beta_2);
    S.eps = (float)a->epsilon; S.lo = (float)a->lo; S.hi = (float)a->hi;
    S.beta_1 = a->beta_1; S.beta_2 = a->beta_2; S.lr = a->lr; S.max_norm = a->max_norm;
    S.step = a->step; S.grad_norm = a->grad_norm;
    S.partial = a->max_norm > 0 ? partial : nullptr;
    S.partials = partials;
    for (int from = 0, n = 0; n < launches; ++n) {
        from = fill(tab, tensors, count, from);
        const int groups = groups_of(tab.first[tab.count], kMaxGroups, tab.per);
        S.last = n == launches - 1;
        if (a->state_bits == 32) hipLaunchKernelGGL(k_adamw<32>, dim3((unsigned)groups), dim3(kThreads), 0, st, tab, S);
        else hipLaunchKernelGGL(k_adamw<8>, dim3((unsigned)groups), dim3(kThreads), 0, st, tab, S);
    }
    NN_LAUNCHED("adamw");
    return 0;
}

int plmpm_adamw_values(const void* const* codes, const float* const* scales, float* const* out, const int64_t* n, const int32_t* which, int count,
                       void* hip_stream) {
    NN_REQUIRE(count >= 0 && (!count || (codes && scales && out && n && which)), "adamw values: null argument");
    for (int k = 0; k < count; ++k)
        NN_REQUIRE(n[k] >= 0 && n[k] < ((int64_t)1 << 41) && (!n[k] || (codes[k] && scales[k] && out[k])) && (uintptr_t)out[k] % 4 == 0, "adamw values: tensor %d: bad pointer or size", k);
    for (int from = 0; from < count;) {
        Values V;
        int64_t chunks = 0;
        V.count = 0;
        V.first[0] = 0;
        for (; from < count && V.count < kMaxTensors && chunks + chunks_of(n[from]) < (1 << 30); ++from) {
            if (!n[from]) continue;
            V.codes[V.count] = codes[from]; V.scales[V.count] = scales[from]; V.out[V.count] = out[from];
            V.n[V.count] = n[from]; V.which[V.count] = which[from];
            chunks += chunks_of(n[from]);
            V.first[++V.count] = (int32_t)chunks;
        }
        if (!V.count) break;
        const int groups = groups_of((int)chunks, kMaxGroups, V.per);
        hipLaunchKernelGGL(k_values, dim3((unsigned)groups), dim3(kThreads), 0, (hipStream_t)hip_stream, V);
    }
    NN_LAUNCHED("adamw values");
    return 0;
}

}  // extern "C"
