// Gated linear recurrence (include/plmpm_policy.h: plmpm_scan) and its backward pass.
//
//   a_t = exp(la_t), la_t = -c softplus(decay) sigmoid(r_t);   h_t = a_t h_{t-1} + m_t sigmoid(i_t) x_t,  m_t = sqrt(1 - a_t^2)
//
// A run of steps acts on the state as h -> A h + H (A the product of its a, H what it ends with from zero), and runs compose.  A workgroup
// takes a tile (S steps a wave, W waves) of 64 VEC channels: every wave reduces its sub-run from registers to (A, H), the channels'
// owners chain the sub-runs through LDS from the state the tile starts with, and every wave replays its sub-run from the state it starts with.
// Inputs are read once and stay in registers between the two walks.
//
// The state a tile starts with comes from the tiles before it while all of them are under way: a tile first publishes its own (A, H) for each
// channel, then walks back over its predecessors' until it meets one that already knows the state it ends with, and publishes
// its own end.  A word of 64 bits holds what is published and says what it is, so one relaxed store and load (agent scope: past the caches of the
// compute units and of the eight dies) carry both, and nothing else has to be ordered.  Tiles are handed out by a ticket in the order of time, all
// channels of a tile before the next tile: whoever waits, waits for tickets below its own, which are held by workgroups that run already
// and publish before they wait -- the lowest unfinished ticket waits for nobody, so every wait ends.
// The words and the ticket are cleared by a small kernel before each launch (not a memset node: calls may be captured).
//
// A reset makes the run forget what came before, also a NaN (and, backward, what comes behind it): its A is then -0, whatever its other steps
// are (every genuine A is +0 or above), and whoever composes runs takes H alone where the sign is set.
#include <algorithm>
#include <type_traits>

#include "plmpm_nn.h"

using namespace plbnn;

namespace {

constexpr int kCheckpoint = 64;         // steps between the states kept for the backward pass
typedef unsigned long long Word;

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
    unsigned* ticket;
    Word* words;                        // [tiles][batch][width], in the order the tiles are handed out
    float* k2;                          // [width]: -c log2(e) softplus(decay), where there is more than one tile
    int64_t B, T;
    int D, cblks, tiles;
    bool past;                          // the gradients go past the caches
    float c;
};

__device__ __forceinline__ bool forgets(float A) { return (as_u(A) >> 31) != 0; }
// max(x, 0) + log(1 + e), e = exp(-|x|): e as a power of two with the product's rounding put right behind it, and log(1 + e) = e P(e) with the polynomial
// through its values at the Chebyshev points of [0, 1] (relative error 5e-9).  In all within 5.3 x 2^-24, like log1pf(expf(-|x|)), which takes
// three times as long: 500 x 2048, one step, 7.9 us with those, 5.7 so.
__device__ __forceinline__ float softplus(float x) {
    const float far = fabsf(x), to = far > 200.0f ? 200.0f : far;                          // (a NaN stays)
    const float p = -kLog2e * to, off = fmaf(-1.9259629911266175e-8f, to, fmaf(-kLog2e, to, -p));
    float e = exp2f(p);
    e = fmaf(e * off, kLn2, e);
    constexpr float c[10] = {-0.0031760570127516985f, 0.019542526453733444f, -0.056373611092567444f, 0.10543623566627502f, -0.1526966691017151f,
                             0.1966327428817749f, -0.24951615929603577f, 0.33329710364341736f, -0.49999892711639404f, 1.0f};
    float q = c[0];
#pragma unroll
    for (int k = 1; k < 10; ++k) q = fmaf(q, e, c[k]);
    return fmaf(e, q, fmaxf(x, 0.0f));
}

// sigmoid(r), sigmoid(i), log2 a, a and 1 - a^2.  1 - a^2 = -expm1(2 ln2 l2) cancels for a near 1: above l2 = -0.18 (a^2 > 0.78) it
// comes from a cubic for -expm1(2 ln2 l) / l, the polynomial through its values at the Chebyshev points (relative error 2.7e-7, half
// of that in the root); below, 1 - a a is off by at most 2^-24 / 0.22.
// BOTH (backward): the sigmoids also as both_sides has them, and taken from there, so that the walks that come back to them see the same numbers.
struct Gates { float sr, si, l2, a, m2, both_r, both_i; };
template <bool BOTH = false> __device__ __forceinline__ Gates gates(float r, float i, float k2) {
    Gates g;
    if (BOTH) {
        g.both_r = both_sides(r);
        g.both_i = both_sides(i);
        g.sr = side_of(g.both_r);
        g.si = side_of(g.both_i);
    } else {
        g.sr = sigmoid_fast(r);
        g.si = sigmoid_fast(i);
    }
    g.l2 = k2 * g.sr;
    g.a = exp2_fast(g.l2);
    const float q = fmaf(fmaf(fmaf(-0.13934674859046936f, g.l2, -0.4424225986003876f), g.l2, -0.960848331451416f), g.l2, -1.3862940073013306f);
    g.m2 = g.l2 >= -0.18033688f ? g.l2 * q : fmaf(-g.a, g.a, 1.0f);
    return g;
}

// which of the S steps from t on are resets: a bit each (uniform over the wave)
template <int S> __device__ __forceinline__ unsigned reset_bits(const ScanArgs& A, int64_t b, int64_t t, int left) {
    const int lane = threadIdx.x & 63;
    const int hit = A.reset && lane < S && lane < left ? A.reset[b * A.T + t + lane] != 0 : 0;
    return (unsigned)__ballot(hit);
}

// S steps from t on, `stride` elements apart: whole, or the first `left` of them (those behind load the last one again)
template <bool WHOLE, class T, int VEC, bool LOOSE, int S>
__device__ __forceinline__ void load_steps(const void* base, int64_t stride, int left, unsigned offset, Vec<T, VEC, LOOSE> (&raw)[S]) {
    T* row = (T*)base;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        raw[s].load(at_offset(row, offset));
        if (WHOLE || s + 1 < left) row += stride;
    }
}
template <int VEC> __device__ __forceinline__ void load_k2(const ScanArgs& A, int d, float (&k2)[VEC]) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        const int at = VEC == 1 || d + v < A.D ? d + v : d;
        k2[v] = A.k2 ? A.k2[at] : -A.c * kLog2e * softplus(A.decay[at]);
    }
}
// a lane's channels of a row.  LOOSE: rows at any element's address, and the last lane may have one channel only (`tail`): it loads the two that the
// row ends with and drops the first, and stores one.
template <class T, int VEC, bool LOOSE> struct Channels {
    int d0;
    bool live, tail;
    unsigned in, out;                   // byte offsets
    __device__ __forceinline__ Channels(int first, int D) {
        d0 = first + (int)(threadIdx.x & 63) * VEC;
        live = d0 < D;
        tail = LOOSE && live && d0 + VEC > D;
        out = (unsigned)(live ? d0 : 0) * (unsigned)sizeof(T);
        in = out - (tail ? (unsigned)sizeof(T) : 0u);
    }
    __device__ __forceinline__ void loaded(Vec<T, VEC, LOOSE>& v) const {
        if constexpr (LOOSE) v.drop(tail ? 1 : 0);
    }
    // `past`: past the caches (the empty asm keeps the compiler from making one ordinary store of the two)
    __device__ __forceinline__ void store(const Vec<T, VEC, LOOSE>& v, T* row, bool past) const {
        if (LOOSE && tail) {
            Vec<T, 1> one;
            memcpy(one.w, v.w, sizeof(T));
            one.store(at_offset(row, out));
        } else if (past) {
            v.store_past(at_offset(row, out));
            asm volatile("");
        } else v.store(at_offset(row, out));
    }
};
__device__ __forceinline__ int steps_left(int64_t T, int64_t t, int most) {
    const int64_t n = T - t;
    return n < most ? (n < 0 ? 0 : (int)n) : most;
}

// What a tile publishes for a channel: the state behind it in the high half; in the low half 0 (nothing yet), the bits of its A plus one (A and
// H of the tile alone), or all ones (the high half is the state itself).
constexpr unsigned kState = 0xffffffffu;
__device__ __forceinline__ Word word_of(float A, float H) {
    const unsigned a = A != A ? 0x7fc00000u : as_u(A);
    return ((Word)as_u(H) << 32) | (a + 1u);
}
__device__ __forceinline__ Word state_word(float h) { return ((Word)as_u(h) << 32) | kState; }
__device__ __forceinline__ void publish(Word* p, Word w) { __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ Word look(const Word* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The state that position `pos` starts with (`p`: this channel's word at position 0, `stride` words apart): back over the positions before it to one
// whose state is known, then forward again over what those in between published.  The state behind a position is always its H + A times the
// state before it, so every route gives the same bits, however far a walk happens to go.  What it meets on the way is kept in `path` (this
// channel's column of [kPath][NCH]); a walk that has filled it waits for the state of the position it has reached.  Position 0 publishes its
// state, so no walk goes further.  Two words a poll, each past the caches: 65537 x 1024 forward / 8 x 2047 x 2048 backward 134 / 131 us, with four
// 133 / 143; without any handing over, wrong, 118 / 129.
constexpr int kPath = 16;
struct Run { float A, H; };
template <int NCH> __device__ __forceinline__ float state_before(const Word* p, int64_t stride, int pos, Run* path) {
    int n = 0;
    float h = 0.0f;
    for (bool found = false; !found;) {
        Word w[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) w[q] = look(p + (pos - 1 - n > q ? pos - 1 - n - q : 0) * stride);
        bool waits = false;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (found || waits) continue;
            const unsigned low = (unsigned)w[q];
            const float A = as_f(low - 1u);
            h = as_f((unsigned)(w[q] >> 32));
            if (low == kState || (low && forgets(A))) found = true;
            else if (low == 0 || n == kPath) waits = true;
            else path[n++ * NCH] = {A, h};
        }
        if (waits) sleep_a_little();
    }
    while (n) {
        const Run r = path[--n * NCH];
        h = fmaf(r.A, h, r.H);
    }
    return h;
}

// Which tile and which channels this workgroup takes: in the order of a ticket where there is more than one tile.  (Workgroups that stay and draw their
// next ticket while they work on one hold tiles back that others wait for: 174 us instead of 133 at 65537 x 1024.)
struct Place { int64_t b; int pos, first; };
template <int NCH> __device__ __forceinline__ Place place(const ScanArgs& A, unsigned* shared) {
    unsigned id = blockIdx.x;
    if (A.tiles > 1) {
        if (threadIdx.x == 0) *shared = atomicAdd(A.ticket, 1u);
        __syncthreads();
        id = (unsigned)__builtin_amdgcn_readfirstlane((int)*shared);
    }
    // (divisions run in vector registers: back to scalar ones, or every row's address would be built a lane)
    const unsigned blocks = (unsigned)(A.B * A.cblks), pos = (unsigned)__builtin_amdgcn_readfirstlane((int)(id / blocks)), rest = id - pos * blocks;
    const unsigned b = (unsigned)__builtin_amdgcn_readfirstlane((int)(rest / (unsigned)A.cblks));
    return {(int64_t)b, (int)pos, (int)(rest - b * (unsigned)A.cblks) * NCH};
}

template <class T, int VEC, int S, int W, bool RESET, bool LOOSE>
__global__ __launch_bounds__(W * 64) void k_scan_forward(ScanArgs A) {
    constexpr int NCH = 64 * VEC;
    __shared__ float sA[W][NCH], sH[W][NCH];
    __shared__ Run path[kPath][NCH];
    __shared__ unsigned ticket;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const Place at = place<NCH>(A, &ticket);
    const int64_t b = at.b;
    const int first = at.first;
    const Channels<T, VEC, LOOSE> mine(first, A.D);
    const int64_t t0 = (int64_t)at.pos * (S * W) + wave * S;
    const int left = __builtin_amdgcn_readfirstlane(steps_left(A.T, t0, S));
    const int64_t from = left ? t0 : A.T - 1;            // (a wave whole behind the end loads the last step)
    const unsigned cut = RESET ? reset_bits<S>(A, b, t0, left) : 0u;
    float k2[VEC], a[S][VEC], u[S][VEC], PA[VEC], PH[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        PA[v] = 1.0f;
        PH[v] = 0.0f;
    }
    const auto walk = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        Vec<T, VEC, LOOSE> raw[3][S];
#pragma unroll
        for (int k = 0; k < 3; ++k) load_steps<WHOLE>((const T*)A.in[k] + b * A.sb[k] + from * A.st[k], A.st[k], left, mine.in, raw[k]);
        load_k2<VEC>(A, mine.live ? mine.d0 : 0, k2);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[VEC], r[VEC], i[VEC];
#pragma unroll
            for (int k = 0; k < 3; ++k) mine.loaded(raw[k][s]);
            raw[0][s].get(x);
            raw[1][s].get(r);
            raw[2][s].get(i);
            const bool there = WHOLE || s < left;        // a step behind the end leaves the state as it is
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Gates g = gates(r[v], i[v], k2[v]);
                a[s][v] = there ? g.a : 1.0f;
                u[s][v] = g.si * x[v];
                if (RESET && (cut >> s & 1)) PH[v] = u[s][v];
                else {
                    u[s][v] = there ? u[s][v] * __builtin_amdgcn_sqrtf(g.m2) : 0.0f;
                    PA[v] *= a[s][v];
                    PH[v] = fmaf(a[s][v], PH[v], u[s][v]);
                }
            }
        }
    };
    if (left == S) walk(std::true_type());
    else walk(std::false_type());
#pragma unroll
    for (int v = 0; v < VEC; ++v) { sA[wave][lane * VEC + v] = RESET && cut ? -0.0f : PA[v]; sH[wave][lane * VEC + v] = PH[v]; }
    __syncthreads();
    for (int ch = threadIdx.x; ch < NCH; ch += blockDim.x) {
        if (first + ch >= A.D) continue;
        const int64_t col = b * A.D + first + ch, stride = A.B * A.D;
        float c = at.pos == 0 && A.h0 ? A.h0[col] : 0.0f;
        if (A.tiles > 1) {
            float ta = 1.0f, th = 0.0f;
            for (int w = 0; w < waves; ++w) {
                const float pa = sA[w][ch], ph = sH[w][ch];
                th = forgets(pa) ? ph : fmaf(pa, th, ph);
                ta = forgets(pa) ? -0.0f : ta * pa;
            }
            Word* own = A.words + (int64_t)at.pos * stride + col;
            if (at.pos > 0) {
                if (at.pos < A.tiles - 1) publish(own, word_of(ta, th));
                c = state_before<NCH>(A.words + col, stride, at.pos, &path[0][ch]);
            }
            if (at.pos < A.tiles - 1) publish(own, state_word(forgets(ta) ? th : fmaf(ta, c, th)));
        }
        for (int w = 0; w < waves; ++w) {
            const float pa = sA[w][ch], ph = sH[w][ch];
            const int64_t t = (int64_t)at.pos * (S * W) + w * S;
            if (A.ckpt && t % kCheckpoint == 0 && t < A.T) A.ckpt[(t / kCheckpoint) * stride + col] = c;
            sA[w][ch] = c;
            c = forgets(pa) ? ph : fmaf(pa, c, ph);
        }
        if (A.h_last && at.pos == A.tiles - 1) A.h_last[col] = c;
    }
    __syncthreads();
    float now[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) now[v] = sA[wave][lane * VEC + v];
    // (without it the compiler waits before every store below, in case one of the loads above is still out, and so for the store before it:
    // 8 x 2047 x 2048 77 us instead of 70)
    wait_for_memory();
    if (!mine.live) return;
    T* out = (T*)A.h + (b * A.T + t0) * A.D;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (s >= left) continue;
#pragma unroll
        for (int v = 0; v < VEC; ++v) now[v] = RESET && (cut >> s & 1) ? u[s][v] : fmaf(a[s][v], now[v], u[s][v]);
        Vec<T, VEC, LOOSE> o;
        o.set(now);
        mine.store(o, out + (int64_t)s * A.D, false);
    }
}

// One step (a rollout's): nothing to chain, so a wave takes 64 VEC channels of a row and the rows below it, 4 waves a workgroup.  The state may move
// on in place (h0 = h_last): a thread reads and writes its own channels only.  500 x 2048, bf16: 5 us; as a tile of the kernel above, whose
// waves then walk 15 steps behind the end, 23 (both with a slower softplus).
template <class T, int VEC>
__global__ __launch_bounds__(256) void k_scan_step(ScanArgs A) {
    const int d = (blockIdx.x * 64 + (threadIdx.x & 63)) * VEC;
    if (d >= A.D) return;
    float k2[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) k2[v] = -A.c * kLog2e * softplus(A.decay[d + v]);
    for (int64_t b = blockIdx.y * 4 + (threadIdx.x >> 6); b < A.B; b += gridDim.y * 4) {
        Vec<T, VEC> in[3], out;
        Vec<float, VEC> state;
#pragma unroll
        for (int k = 0; k < 3; ++k) in[k].load((const T*)A.in[k] + b * A.sb[k] + d);
        const int64_t at = b * A.D + d;
        if (A.h0) state.load(A.h0 + at);
        else state.zero();
        if (A.ckpt) state.store(A.ckpt + at);
        const bool cut = A.reset && A.reset[b];
        float x[VEC], r[VEC], i[VEC], h[VEC];
        in[0].get(x);
        in[1].get(r);
        in[2].get(i);
        state.get(h);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Gates g = gates(r[v], i[v], k2[v]);
            const float u = g.si * x[v];
            h[v] = cut ? u : fmaf(g.a, h[v], u * __builtin_amdgcn_sqrtf(g.m2));
        }
        out.set(h);
        out.store((T*)A.h + at);
        state.set(h);
        if (A.h_last) state.store(A.h_last + at);
    }
}

// Backward: g_t = dh_t + a_{t+1} g_{t+1}, walked from the end.  With e_t = a_t g_t as what a step hands to the one before it, a run acts
// on what comes in from behind as e -> A e + E with the same A, so both walks (forward again from the tile's checkpoint, which gives
// h_{t-1} in 32 bits, and backward) go through one exchange; tiles are handed out from the last to the first.
//   dx = g m s_i   di = g m x s_i (1 - s_i)   dla = g (a h_{t-1} - s_i x a^2 / m)   dr = dla la (1 - s_r)
// For la -> 0 the product la a^2 / m goes to 0 (m ~ sqrt(-2 la)): where m is 0 that term is left out.
// s (1 - s) comes from the smaller side (both_sides): 3 % more time at 8 x 2047 x 2048 than with 1 - s from s, whose gradients are wrong far out.
template <class T, int VEC, int S, int W, bool LOOSE>
__global__ __launch_bounds__(W * 64, 4) void k_scan_backward(ScanArgs A) {
    static_assert(S * W % kCheckpoint == 0, "a tile starts at a checkpoint");
    constexpr int NCH = 64 * VEC;
    __shared__ float sA[W][NCH], sH[W][NCH], sE[W][NCH];
    __shared__ Run path[kPath][NCH];
    __shared__ unsigned ticket;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const Place at = place<NCH>(A, &ticket);
    const int tile = A.tiles - 1 - at.pos;
    const int64_t b = at.b;
    const int first = at.first;
    const Channels<T, VEC, LOOSE> mine(first, A.D);
    const int64_t t0 = (int64_t)tile * (S * W) + wave * S;
    const int left = __builtin_amdgcn_readfirstlane(steps_left(A.T, t0, S));
    const int64_t from = left ? t0 : A.T - 1;
    const unsigned cut = reset_bits<S>(A, b, t0, left);
    // Kept for the second walk: x and dh as they came, a, m and both sides of the gates (sr, si).  What can be had from those in a few operations is
    // not: a register more here is one spilled to memory.  (8 x 2047 x 2048: with m s_i and s_i x a^2 / m held in m's place, 29 of them, 154 us instead of 131.  The
    // compiler would do the same by itself, hence forget and anew: calls in bf16 and fp16 without resets 165 and 171 us, with the 16 and 32
    // registers that it keeps otherwise 185 and 196.  A kernel without the resets' selects kept more of them and was the slower one.  These were taken with the
    // gates themselves held; both sides of them cost 3 %, 14 to 26 spilled registers until they were taken back from one number, here and at the last walk.)
    Vec<T, VEC, LOOSE> rawx[S], rawg[S];
    float k2[VEC], a[S][VEC], sr[S][VEC], si[S][VEC], m[S][VEC], PA[VEC], PH[VEC], PE[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        PA[v] = 1.0f;
        PH[v] = PE[v] = 0.0f;
    }
    const auto walk = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        Vec<T, VEC, LOOSE> rawr[S], rawi[S];
        load_steps<WHOLE>((const T*)A.in[1] + b * A.sb[1] + from * A.st[1], A.st[1], left, mine.in, rawr);
        load_steps<WHOLE>((const T*)A.in[2] + b * A.sb[2] + from * A.st[2], A.st[2], left, mine.in, rawi);
        load_steps<WHOLE>((const T*)A.in[0] + b * A.sb[0] + from * A.st[0], A.st[0], left, mine.in, rawx);
        if (A.dh) load_steps<WHOLE>((const T*)A.dh + (b * A.T + from) * A.D, (int64_t)A.D, left, mine.in, rawg);
#pragma unroll
        for (int s = 0; s < S; ++s) if (!A.dh || !(WHOLE || s < left)) rawg[s].zero();
        load_k2<VEC>(A, mine.live ? mine.d0 : 0, k2);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float x[VEC], r[VEC], i[VEC];
            mine.loaded(rawx[s]);
            mine.loaded(rawr[s]);
            mine.loaded(rawi[s]);
            mine.loaded(rawg[s]);
            rawx[s].forget();
            rawg[s].forget();
            rawx[s].get(x);
            rawr[s].get(r);
            rawi[s].get(i);
            const bool there = WHOLE || s < left;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Gates g = gates<true>(r[v], i[v], k2[v]);
                sr[s][v] = there ? g.both_r : 0.0f;
                si[s][v] = g.both_i;
                if ((cut >> s & 1)) {
                    a[s][v] = sr[s][v] = 0.0f;          // (r has no part in a step that begins anew, whatever it is)
                    m[s][v] = 1.0f;
                    PH[v] = g.si * x[v];
                } else {
                    a[s][v] = there ? g.a : 1.0f;
                    m[s][v] = there ? __builtin_amdgcn_sqrtf(g.m2) : 0.0f;
                    PA[v] *= a[s][v];
                    PH[v] = fmaf(a[s][v], PH[v], m[s][v] * g.si * x[v]);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < S; ++s) { rawx[s].forget(); rawg[s].forget(); }
    };
    if (left == S) walk(std::true_type());
    else walk(std::false_type());
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
        float g[VEC];
        rawg[s].get(g);
#pragma unroll
        for (int v = 0; v < VEC; ++v) PE[v] = (cut >> s & 1) ? 0.0f : a[s][v] * (g[v] + PE[v]);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        sA[wave][lane * VEC + v] = cut ? -0.0f : PA[v];
        sH[wave][lane * VEC + v] = PH[v];
        sE[wave][lane * VEC + v] = PE[v];
    }
    __syncthreads();
    for (int ch = threadIdx.x; ch < NCH; ch += blockDim.x) {
        if (first + ch >= A.D) continue;
        const int64_t col = b * A.D + first + ch, stride = A.B * A.D;
        float c = A.ckpt[(int64_t)tile * (S * W / kCheckpoint) * stride + col], e = at.pos == 0 && A.dlast ? A.dlast[col] : 0.0f;
        if (A.tiles > 1) {
            float ta = 1.0f, te = 0.0f;
            for (int w = waves - 1; w >= 0; --w) {
                const float pa = sA[w][ch], pe = sE[w][ch];
                te = forgets(pa) ? pe : fmaf(pa, te, pe);
                ta = forgets(pa) ? -0.0f : ta * pa;
            }
            Word* own = A.words + (int64_t)at.pos * stride + col;
            if (at.pos > 0) {
                if (at.pos < A.tiles - 1) publish(own, word_of(ta, te));
                e = state_before<NCH>(A.words + col, stride, at.pos, &path[0][ch]);
            }
            if (at.pos < A.tiles - 1) publish(own, state_word(forgets(ta) ? te : fmaf(ta, e, te)));
        }
        for (int w = waves - 1; w >= 0; --w) {
            const float pa = sA[w][ch], pe = sE[w][ch];
            sE[w][ch] = e;
            e = forgets(pa) ? pe : fmaf(pa, e, pe);
        }
        if (A.dh0 && at.pos == A.tiles - 1) A.dh0[col] = e;
        for (int w = 0; w < waves; ++w) {
            const float pa = sA[w][ch], ph = sH[w][ch];
            sA[w][ch] = c;
            c = forgets(pa) ? ph : fmaf(pa, c, ph);
        }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s) {
        rawx[s].forget();
        rawg[s].forget();
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            anew(m[s][v]);
            anew(si[s][v]);
            anew(a[s][v]);
            anew(sr[s][v]);
        }
    }
    float now[VEC], e[VEC], sum[VEC], pull[S][VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        now[v] = sA[wave][lane * VEC + v];
        e[v] = sE[wave][lane * VEC + v];
        sum[v] = 0.0f;
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
        float x[VEC];
        rawx[s].get(x);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const bool reset = (cut >> s & 1);
            const float sx = side_of(si[s][v]) * x[v], u = m[s][v] * sx, inv = m[s][v] == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(m[s][v]);
            pull[s][v] = reset ? 0.0f : a[s][v] * fmaf(-sx * inv, a[s][v], now[v]);        // dla / g
            now[v] = reset ? u : fmaf(a[s][v], now[v], u);
        }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
        float x[VEC], g[VEC], dx[VEC], dr[VEC], di[VEC];
        rawx[s].get(x);
        rawg[s].get(g);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const bool reset = (cut >> s & 1);
            anew(si[s][v]);
            g[v] += e[v];
            e[v] = reset ? 0.0f : a[s][v] * g[v];
            dx[v] = g[v] * m[s][v] * side_of(si[s][v]);
            di[v] = g[v] * m[s][v] * x[v] * product_of(si[s][v]);
            const float q = reset || s >= left ? 0.0f : g[v] * pull[s][v];         // (behind the end: 0 times a state that may be infinite)
            dr[v] = q * (k2[v] * kLn2) * product_of(sr[s][v]);
            sum[v] = fmaf(q, side_of(sr[s][v]), sum[v]);
        }
        if (mine.live && s < left) {
            const int64_t to = (b * A.T + t0 + s) * A.D;
            const auto put = [&](int k, const float* d) {
                Vec<T, VEC, LOOSE> o;
                o.set(d);
                mine.store(o, (T*)A.out[k] + to, A.past);
            };
            put(0, dx);
            put(1, dr);
            put(2, di);
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
}

// before a launch of more than one tile: the ticket and the words cleared, and the channels' k2 (softplus is more work than a step)
__global__ __launch_bounds__(256) void k_prepare(Word* p, int64_t n, float* k2, const float* decay, int D, float c) {
    const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)gridDim.x * 256;
    for (int64_t k = first; k < n; k += all) publish(p + k, 0);        // (4.4 us; with ordinary stores, to be written back at the end, 4.8)
    for (int64_t d = first; d < D; d += all) k2[d] = -c * kLog2e * softplus(decay[d]);
}

// d decay[d] = -c sigmoid(decay[d]) * (sum of column d of part[rows][D]): 64 columns and 16 strips of rows a workgroup, strips joined in a
// fixed order, all in 64 bits: a row is a tile of one sequence, and there can be hundreds of thousands of them
__global__ __launch_bounds__(1024) void k_decay_grad(const float* part, const float* decay, float* out, int64_t rows, int D, float c) {
    __shared__ double strip[16][64];
    const int col = threadIdx.x & 63, s = threadIdx.x >> 6, d = blockIdx.x * 64 + col;
    double sum = 0.0;
    if (d < D)
#pragma unroll 8
        for (int64_t r = s; r < rows; r += 16) sum += part[r * D + d];
    strip[s][col] = sum;
    __syncthreads();
    if (s == 0 && d < D) {
        for (int k = 1; k < 16; ++k) sum += strip[k][col];
        out[d] = (float)(-c * sigmoid_fast(decay[d]) * sum);
    }
}

// Steps a wave and waves a workgroup of the two kernels.  Measured at 65537 steps x 1024 channels (forward) and 8 x 2047 x 2048 (both), bf16, us:
// forward 16 x 8 135 / 75, 8 x 8 155 / 73, 8 x 16 162 / 83, 16 x 4 149 / 81; backward 8 x 8 at 136 registers 171, held to 128 (two workgroups a
// CU, for some twenty spilled registers) 142, without those 128; 4 x 16 167, 8 x 16 180, 16 x 4 202.  (8 x 8 with both sides of the gates: 131 to 136.)  32 bits have
// one channel a lane and 98 registers; 8 x 2047 x 1024 101 us of a floor of 90, so its tiles were not looked for apart.
constexpr int kForwardSteps = 16, kForwardWaves = 8, kBackwardSteps = 8, kBackwardWaves = 8;
// Gradients of more bytes than this go past the caches: the first of them would be gone from the 256 MB cache when the last is written, and x, r, i and
// dh stay in it.  The backward kernel and a copy that reads its gradients, us: 25 MB 25.5 + 19.9 (past the caches 23.0 + 25.4), 75 MB 55.0 + 58.6
// (54.9 + 72.6), 101 MB 70.8 + 89.9 (70.9 + 104.2), 138 MB 91.8 + 142.7 (90.1 + 139.9), 201 MB 133.4 + 215.1 (131.8 + 208.6).
constexpr double kPastCaches = 128 << 20;
int tile_of(bool backward) { return backward ? kBackwardSteps * kBackwardWaves : kForwardSteps * kForwardWaves; }
int64_t tiles_of(const plmpm_scan* s, bool backward) { return (s->steps + tile_of(backward) - 1) / tile_of(backward); }
// workspace: one word for the ticket, the words, k2 (an even number of floats), and (backward) the rows of d decay's sums
size_t word_bytes(const plmpm_scan* s, bool backward) {
    const int64_t tiles = tiles_of(s, backward);
    return tiles > 1 ? sizeof(Word) * (1 + (size_t)tiles * s->batch * s->width) : 0;
}
size_t k2_bytes(const plmpm_scan* s, bool backward) { return tiles_of(s, backward) > 1 ? round_up(s->width * sizeof(float), 8) : 0; }

// a workgroup: the waves of a tile, fewer where the steps end before
unsigned threads_of(int64_t steps, bool backward) {
    const int S = backward ? kBackwardSteps : kForwardSteps, W = backward ? kBackwardWaves : kForwardWaves;
    return 64u * (unsigned)std::min<int64_t>((steps + S - 1) / S, W);
}
template <class T, int VEC, bool LOOSE> void launch(const ScanArgs& A, bool backward, hipStream_t st) {
    const dim3 grid((unsigned)(A.B * A.cblks * A.tiles)), block(threads_of(A.T, backward));
    if (backward) hipLaunchKernelGGL((k_scan_backward<T, VEC, kBackwardSteps, kBackwardWaves, LOOSE>), grid, block, 0, st, A);
    else if (A.reset) hipLaunchKernelGGL((k_scan_forward<T, VEC, kForwardSteps, kForwardWaves, true, LOOSE>), grid, block, 0, st, A);
    else hipLaunchKernelGGL((k_scan_forward<T, VEC, kForwardSteps, kForwardWaves, false, LOOSE>), grid, block, 0, st, A);
}
template <class T> void launch(const ScanArgs& A, int vec, bool loose, bool backward, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (vec == 2) return loose ? launch<T, 2, true>(A, backward, st) : launch<T, 2, false>(A, backward, st);
    launch<T, 1, false>(A, backward, st);
}

// one step: four channels a lane where everything keeps to them
template <class T> void launch_step(const ScanArgs& A, hipStream_t st) {
    bool four = A.D % 4 == 0 && aligned_to(A.h, 0, 1) >= 4 * (int)sizeof(T);
    for (int k = 0; k < 3; ++k) four = four && aligned_to(A.in[k], A.sb[k], (int)sizeof(T)) >= 4 * (int)sizeof(T);
    for (const void* p : {(const void*)A.h0, (const void*)A.h_last, (const void*)A.ckpt}) four = four && aligned_to(p, 0, 1) >= 16;
    const int vec = four ? 4 : 1;
    const int64_t across = (A.D + 64 * vec - 1) / (64 * vec), down = std::min<int64_t>((A.B + 3) / 4, std::max<int64_t>(1, 4096 / across));
    const dim3 grid((unsigned)across, (unsigned)down);
    if (four) hipLaunchKernelGGL((k_scan_step<T, 4>), grid, dim3(256), 0, st, A);
    else hipLaunchKernelGGL((k_scan_step<T, 1>), grid, dim3(256), 0, st, A);
}

// Channels a lane: 4 bytes' worth, so that a wave's rows are 256 bytes -- 2 channels of 16 bits where at least half of a wave's 128 channels are
// there, else 1.  (16 bits, 8 x 2047 x 2048, forward and backward: 2 channels 70 + 141 us, 1 channel 80 + 158, 4 channels 72 + 202; 32 bits,
// 16 x 50 x 256: 1 channel 7.2 + 9.0 us, 2 channels 8.1 + 11.9.)
int vector_of(const plmpm_scan* s) { return dtype_size(s->dtype) == 2 && s->width >= 64 ? 2 : 1; }
// Whether such a row may begin between two words: an odd width, odd strides or pointers.  (16 bits, calls at
// 8 x 2047 x 2047, forward and backward: 77 + 185 us; with 1 channel a lane 98 + 215.  The kernels alone: 84 + 150.)
bool loose(const plmpm_scan* s, bool backward) {
    const int size = dtype_size(s->dtype);
    int bytes = 16;
    const void* in[3] = {s->x, s->r, s->i};
    for (int k = 0; k < 3; ++k) bytes = std::min(bytes, std::min(aligned_to(in[k], s->stride_b[k], size), aligned_to(in[k], s->stride_t[k], size)));
    if (backward) for (const void* p : {(const void*)s->dh, (const void*)s->dx, (const void*)s->dr, (const void*)s->di}) bytes = std::min(bytes, aligned_to(p, s->width, size));
    else bytes = std::min(bytes, aligned_to(s->h, s->width, size));
    return bytes < 4;
}

// a launch takes less than 2^32 threads
int blocks_across(const plmpm_scan* s) { return (int)((s->width + 64 * vector_of(s) - 1) / (64 * vector_of(s))); }
bool fits_a_launch(const plmpm_scan* s, bool backward) {
    return (uint64_t)s->batch * blocks_across(s) * tiles_of(s, backward) * threads_of(s->steps, backward) < ((uint64_t)1 << 32);
}

int check(const plmpm_scan* s, bool backward, bool pointers) {
    NN_REQUIRE(s, "scan: null argument");
    NN_REQUIRE(s->dtype >= PLMPM_NN_F32 && s->dtype <= PLMPM_NN_F16, "scan: unknown dtype %d", s->dtype);
    NN_REQUIRE(s->batch >= 0 && s->steps >= 0 && s->width >= 0, "scan: negative size");
    NN_REQUIRE(s->width < (1 << 27), "scan: width %lld is too large", (long long)s->width);
    NN_REQUIRE(s->steps < ((int64_t)1 << 36), "scan: %lld steps are too many", (long long)s->steps);
    NN_REQUIRE(s->batch < (1 << 30) && s->batch * ((s->width + 63) / 64) < ((int64_t)1 << 31) &&
               s->batch * ((s->width + 63) / 64) * ((s->steps + kCheckpoint - 1) / kCheckpoint) < ((int64_t)1 << 31), "scan: batch x width x steps is too large for one launch");
    NN_REQUIRE(s->c > 0 && s->c < 1e30, "scan: c has to be positive and finite, got %g", s->c);
    if (!pointers || !s->batch || !s->steps || !s->width) return 0;
    NN_REQUIRE(s->x && s->r && s->i && s->decay, "scan: x, r, i and decay are needed");
    if (backward) NN_REQUIRE(s->checkpoint && s->dx && s->dr && s->di && s->ddecay, "scan backward: checkpoint, dx, dr, di and ddecay are needed");
    else NN_REQUIRE(s->h, "scan forward: h is needed");
    const int size = dtype_size(s->dtype);
    for (const void* p : {s->x, s->r, s->i, (const void*)s->h, s->dh, (const void*)s->dx, (const void*)s->dr, (const void*)s->di})
        NN_REQUIRE((uintptr_t)p % size == 0, "scan: a pointer is not aligned to its type");
    for (const float* p : {s->decay, s->h0, (const float*)s->h_last, (const float*)s->checkpoint, s->dlast, (const float*)s->ddecay, (const float*)s->dh0})
        NN_REQUIRE((uintptr_t)p % sizeof(float) == 0, "scan: a pointer is not aligned to its type");
    return 0;
}

int run(const plmpm_scan* s, bool backward, hipStream_t st) {
    if (check(s, backward, true)) return -1;
    if (!s->batch || !s->steps || !s->width) return 0;
    size_t need = 0;
    if (plmpm_scan_workspace(s, backward, &need)) return -1;
    NN_REQUIRE(s->workspace_bytes >= need && (s->workspace || !need), "scan: the workspace has %zu bytes, %zu are needed", s->workspace_bytes, need);
    NN_REQUIRE((uintptr_t)s->workspace % 8 == 0, "scan: the workspace is not aligned to 8 bytes");
    ScanArgs A{};
    A.in[0] = s->x; A.in[1] = s->r; A.in[2] = s->i;
    for (int k = 0; k < 3; ++k) { A.sb[k] = s->stride_b[k]; A.st[k] = s->stride_t[k]; }
    A.decay = s->decay; A.h0 = s->h0; A.reset = s->reset;
    A.h = s->h; A.h_last = s->h_last; A.ckpt = s->checkpoint;
    A.dh = s->dh; A.dlast = s->dlast; A.out[0] = s->dx; A.out[1] = s->dr; A.out[2] = s->di;
    A.dh0 = s->dh0;
    A.B = s->batch; A.T = s->steps; A.D = (int)s->width; A.c = (float)s->c;
    // (a forward call that keeps checkpoints is refused where its backward call would be)
    NN_REQUIRE(((!backward && s->steps == 1) || fits_a_launch(s, backward)) && (backward || !s->checkpoint || fits_a_launch(s, true)), "scan: batch x width x steps is too large for one launch");
    if (!backward && s->steps == 1) {
        if (s->dtype == PLMPM_NN_F32) launch_step<float>(A, st);
        else if (s->dtype == PLMPM_NN_BF16) launch_step<bf16>(A, st);
        else launch_step<f16>(A, st);
        NN_LAUNCHED("scan forward");
        return 0;
    }
    const int vec = vector_of(s);
    const bool between = vec == 2 && loose(s, backward);
    A.cblks = blocks_across(s);
    A.tiles = (int)tiles_of(s, backward);
    A.past = 3.0 * dtype_size(s->dtype) * s->batch * s->steps * s->width > kPastCaches;
    const size_t words = word_bytes(s, backward);
    A.part = (float*)((char*)s->workspace + words + k2_bytes(s, backward));
    if (words) {
        A.ticket = (unsigned*)s->workspace;
        A.words = (Word*)s->workspace + 1;
        A.k2 = (float*)((char*)s->workspace + words);
        const int64_t n = (int64_t)(words / sizeof(Word)), groups = (n + 1023) / 1024;
        hipLaunchKernelGGL(k_prepare, dim3((unsigned)(groups < 2048 ? groups : 2048)), dim3(256), 0, st, (Word*)s->workspace, n, A.k2, A.decay, A.D, A.c);
    }
    if (s->dtype == PLMPM_NN_F32) launch<float>(A, vec, between, backward, st);
    else if (s->dtype == PLMPM_NN_BF16) launch<bf16>(A, vec, between, backward, st);
    else launch<f16>(A, vec, between, backward, st);
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
    *bytes = word_bytes(s, backward != 0) + k2_bytes(s, backward != 0) + (backward ? (size_t)tiles_of(s, true) * s->batch * s->width * sizeof(float) : 0);
    return 0;
}
int plmpm_scan_forward(const plmpm_scan* s, void* hip_stream) { return run(s, false, (hipStream_t)hip_stream); }
int plmpm_scan_backward(const plmpm_scan* s, void* hip_stream) { return run(s, true, (hipStream_t)hip_stream); }

}  // extern "C"
