// gsx_gated.hip -- the gated linear recurrence h_t = a_t h_(t-1) + b_t along one axis, and its gradients: the compositing formula
// ("over", front index 0, last layer first) without the splats, for layers, traces and sequences of any length.
//   linear  a = z,     b = x         blend  a = 1 - z, b = z x         over  a = 1 - z, b = x
// Backward, from the last step to the first with c = dL/dh flowing back:  g_t = d_t + c,  dx = g (z g for blend),
// dz = g h_(t-1) (linear), g (x - h_(t-1)) (blend), -g h_(t-1) (over),  c = a_t g_t;  dL/dinitial is the c that leaves the first step.
// Three to eight flops per element against 6 to 16 bytes: HBM bounds it.  A lane owns a channel (NV neighbouring ones, or R planes that
// share a gate) and walks the steps in batches of K whose loads are all in flight together; the state stays in a 32-bit register.
// The backward needs h_(t-1) in 32 bits, not as `states` rounds it: the forward leaves the state in front of every K-th step ("marks",
// 4 / K bytes per element) and the backward runs each batch forward again from its mark, in registers.  It then reads gate, x and
// the states' gradient, once each -- as much as a backward that reads `states` instead of x, and `states` need not exist.
// Few channels and many steps: the steps are split into spans, one per wave.  A first kernel folds every span to the (A, H) of
// h -> A h + H, and every workgroup's spans to one; the second begins each span from what the spans in front of it come to.  One pass that hands
// the state from workgroup to workgroup would read once, but its waves would wait for one another in a chain of hundreds.
// Measured, with other inputs and outputs in turn, against a copy's 5.15 TB/s: 60 steps x 1 M channels in 32 bits 134 us (5.4 TB/s); 32 layers of 800 x 800 (3 planes in
// 32 bits) 66 us forward (5.5) and 120 backward (5.7); split, 2 x 32768 x 512 in bf16, mean of the folds 33 us (4.1), walks 35 forward (5.7) and 62 backward (5.4).
#include <type_traits>
#include "gsx_common.h"

namespace gsx {

constexpr int kGatedWaves = 4;
constexpr int kGatedSpans = 8;                      // spans (waves) of a workgroup where the steps are split

template <int R>
struct GatedBatch { static constexpr int value = R == 1 ? 16 : 8; };        // K: steps in flight; planes multiply the registers

struct GatedArgs {
    const void* gate; const void* x; const float* initial; const int32_t* lengths;
    void* states; float* last; float* marks;
    const void* d_states; const float* d_last; void* d_gate; void* d_x; float* d_initial;
    long long T, groups, row;                  // steps, lanes' groups of NV channels in all, groups of one sequence
    long long D;
    long long gate_b, gate_t, x_b, x_t, x_r, ds_b, ds_t, ds_r;
    int form, reverse;
    // split steps: `span` steps each (a multiple of K), kGatedSpans of them to a workgroup, `blocks` workgroups per 64 groups
    long long span, blocks, columns;
    double* span_a; double* span_h;            // [span][B D], [span][planes][B D]
    double* block_a; double* block_h;           // the same of whole workgroups
};

template <typename T, int NV>
struct alignas(sizeof(T) * NV) Pack { T v[NV]; };

// What a walk reads for the last time and writes goes past the caches, which hold less than it: 1 M channels x 60 steps 146 us through them, 136 past them; 32 layers of
// 800 x 800, both ways, 208 and 188.  What the fold of a split walk reads is read again by the walk, and stays: 96 channels x 100001 steps 42.5 us past the caches, 35.7
// through them; so do the inputs of a split backward (8 x 2048 x 2048: 145, 141).
template <bool PAST, typename P>
__device__ __forceinline__ P pack_load(const void* at)
{
    using W = std::conditional_t<sizeof(P) == 2, uint16_t, std::conditional_t<sizeof(P) == 4, uint32_t, unsigned long long>>;
    return __builtin_bit_cast(P, PAST ? __builtin_nontemporal_load((const W*)at) : *(const W*)at);
}
template <typename P>
__device__ __forceinline__ void pack_store(void* at, const P& p)
{
    using W = std::conditional_t<sizeof(P) == 2, uint16_t, std::conditional_t<sizeof(P) == 4, uint32_t, unsigned long long>>;
    __builtin_nontemporal_store(__builtin_bit_cast(W, p), (W*)at);
}

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }         // round to nearest even

// coefficients of one step: a, and m of b = m x
template <int FORM>
__device__ __forceinline__ void gated_am(float z, float& a, float& m)
{
    a = FORM == GSX_GATED_LINEAR ? z : 1.0f - z;
    m = FORM == GSX_GATED_BLEND ? z : 1.0f;
}

// f(form) with the form known to the compiler: decided once per kernel, where a choice per element costs as much as the element
template <typename F>
__device__ __forceinline__ void gated_formed(int form, F f)
{
    if (form == GSX_GATED_LINEAR) f(std::integral_constant<int, GSX_GATED_LINEAR>{});
    else if (form == GSX_GATED_BLEND) f(std::integral_constant<int, GSX_GATED_BLEND>{});
    else f(std::integral_constant<int, GSX_GATED_OVER>{});
}

// A lane's place: which sequence and channels, and where its steps lie.  Scan position s is memory step s, or T - 1 - s in reverse;
// the sequence's own steps are scan positions [lo, hi) (a padded sequence in reverse starts behind its padding).
struct Lane {
    long long b, d, lo, hi;
    bool on;
};

template <int NV>
__device__ __forceinline__ Lane lane_of(const GatedArgs& p, long long group)
{
    Lane l;
    l.on = group < p.groups;
    const long long g = l.on ? group : p.groups - 1;
    if (p.groups < (1ll << 31)) {                                            // 32-bit division where it is enough
        const uint32_t q = (uint32_t)g / (uint32_t)p.row;
        l.b = q; l.d = (long long)((uint32_t)g - q * (uint32_t)p.row) * NV;
    } else {
        l.b = g / p.row; l.d = (g - l.b * p.row) * NV;
    }
    long long len = p.T;
    if (p.lengths) { const int n = p.lengths[l.b]; len = n < 0 ? 0 : n < p.T ? n : p.T; }
    l.lo = p.reverse ? p.T - len : 0;
    l.hi = p.reverse ? p.T : len;
    return l;
}

template <typename T, int FORM, int NV, int R, int K, bool WHOLE>
__device__ __forceinline__ void gated_fwd_batch(const GatedArgs& p, const Lane& l, long long group, long long s0, float (&h)[R][NV])
{
    using P = Pack<T, NV>;
    P z[K], x[K][R];
    const long long dir = p.reverse ? -1 : 1, m0 = p.reverse ? p.T - 1 - s0 : s0;
    const T* gp = (const T*)p.gate + l.b * p.gate_b + m0 * p.gate_t + l.d;
    const T* xp = (const T*)p.x + l.b * p.x_b + m0 * p.x_t + l.d;
#pragma unroll
    for (int k = 0; k < K; k++)
    {
        if (WHOLE || (s0 + k >= l.lo && s0 + k < l.hi)) {
            z[k] = pack_load<true, P>(gp);
#pragma unroll
            for (int r = 0; r < R; r++) x[k][r] = pack_load<true, P>(xp + r * p.x_r);
        }
        gp += dir * p.gate_t; xp += dir * p.x_t;                             // one step on: the multiples of a step would fill the scalar registers
    }
    if (p.marks) {                                                           // behind the loads: a wait for these is none for the stores
        float* mk = p.marks + (s0 / K) * R * p.groups * NV + group * NV;
#pragma unroll
        for (int r = 0; r < R; r++) {
            Pack<float, NV> o;
#pragma unroll
            for (int i = 0; i < NV; i++) o.v[i] = h[r][i];
            *(Pack<float, NV>*)(mk + r * p.groups * NV) = o;
        }
    }
    T* sp = (T*)p.states + ((l.b * p.T + m0) * R) * p.D + l.d;              // no states: not written
#pragma unroll
    for (int k = 0; k < K; k++) {
        const bool in = WHOLE || (s0 + k >= l.lo && s0 + k < l.hi);
        if (in) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                float a, m;
                gated_am<FORM>(to_f(z[k].v[i]), a, m);
#pragma unroll
                for (int r = 0; r < R; r++) h[r][i] = __builtin_fmaf(a, h[r][i], m * to_f(x[k][r].v[i]));
            }
        }
        if (p.states && (WHOLE || s0 + k < p.T)) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                P o;
#pragma unroll
                for (int i = 0; i < NV; i++) o.v[i] = in ? from_f<T>(h[r][i]) : from_f<T>(0.0f);
                pack_store(sp + r * p.D, o);
            }
        }
        sp += dir * R * p.D;
    }
}

// A product of gates in 64 bits that stays finite: times a zero state it is a zero, times any other one it leaves 32 bits, as the walk would.  Four more gates of up to 2^128
// reach 2^1012 at most, two products 2^1000.  And that stays off zero, unless a gate is one: an infinite state stays infinite, as in the walk, and any other one falls
// below 32 bits all the same (2^128 2^-400).  Four more gates of 2^-149 at least leave 2^-996, two products 2^-800.  (2 x 32768 x 512 in bf16: 2 us of 164.  On the exponent's word, or once a batch where a
// product has become small, it costs 4, in registers.)
__device__ __forceinline__ double gated_bound(double A)
{
    const double m = fmin(fabs(A), 0x1p500);
    return copysign(A != 0.0 ? fmax(m, 0x1p-400) : 0.0, A);
}

// Folds steps [s0, s0 + K) to h -> A h + H, in 64 bits: H and A h may be far larger than the state that they add up to, and a 32-bit H would
// then be less exact than the walk itself (its 64-bit FMA is as fast on this card as the 32-bit one).  Backward: c -> A c + H of c_t = a_t (d_t + c_(t+1)), from the last step to the first.
template <typename T, int FORM, int NV, int R, int K, bool BACK, bool HASV, bool WHOLE>
__device__ __forceinline__ void gated_fold_batch(const GatedArgs& p, const Lane& l, long long s0, double (&A)[NV], double (&H)[R][NV])
{
    using P = Pack<T, NV>;
    P z[K], v[K][R];
    const long long dir = p.reverse ? -1 : 1, m0 = p.reverse ? p.T - 1 - s0 : s0;
    const T* gp = (const T*)p.gate + l.b * p.gate_b + m0 * p.gate_t + l.d;
    const T* vp = BACK ? (const T*)p.d_states + l.b * p.ds_b + m0 * p.ds_t + l.d : (const T*)p.x + l.b * p.x_b + m0 * p.x_t + l.d;       // !HASV: not read
    const long long v_t = BACK ? p.ds_t : p.x_t, v_r = BACK ? p.ds_r : p.x_r;
#pragma unroll
    for (int k = 0; k < K; k++)
    {
        if (WHOLE || (s0 + k >= l.lo && s0 + k < l.hi)) {
            z[k] = *(const P*)gp;
            if (HASV)
#pragma unroll
                for (int r = 0; r < R; r++) v[k][r] = *(const P*)(vp + r * v_r);
        }
        gp += dir * p.gate_t; vp += dir * v_t;
    }
#pragma unroll
    for (int q = 0; q < K; q++) {
        const int k = BACK ? K - 1 - q : q;
        if (WHOLE || (s0 + k >= l.lo && s0 + k < l.hi))
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const double zd = (double)to_f(z[k].v[i]), a = FORM == GSX_GATED_LINEAR ? zd : 1.0 - zd;
                A[i] = !WHOLE || (q & 3) == 3 ? gated_bound(A[i] * a) : A[i] * a;       // a sequence may begin and end anywhere in a batch
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const double vd = HASV ? (double)to_f(v[k][r].v[i]) : 0.0;
                    H[r][i] = BACK ? a * (H[r][i] + vd) : fma(a, H[r][i], FORM == GSX_GATED_BLEND ? zd * vd : vd);
                }
            }
    }
}

// where the spans of a split walk lie: the workgroup's and wave's place in the order of the walk (backward: from the end), and its steps
struct Span { long long group, block, index, s0, s1; };

template <bool BACK>
__device__ __forceinline__ Span span_of(const GatedArgs& p)
{
    Span s;
    const long long column = blockIdx.x % p.columns;
    s.block = blockIdx.x / p.columns;
    s.group = column * 64 + (threadIdx.x & 63);
    s.index = s.block * kGatedSpans + (threadIdx.x >> 6);
    const long long at = BACK ? p.blocks * kGatedSpans - 1 - s.index : s.index;
    s.s0 = at * p.span < p.T ? at * p.span : p.T;
    s.s1 = s.s0 + p.span < p.T ? s.s0 + p.span : p.T;
    return s;
}

// (A, H) behind (A0, H0): h -> A (A0 h + H0) + H
__device__ __forceinline__ double gated_apply(double A, double h, double H) { return h == 0.0 ? H : fma(A, h, H); }

template <typename T, int NV, int R, bool BACK, bool HASV>
__global__ __launch_bounds__(64 * kGatedSpans) void gated_fold_kernel(GatedArgs p)
{
    constexpr int K = GatedBatch<R>::value;
    __shared__ double s_a[kGatedSpans][64 * NV];
    __shared__ double s_h[kGatedSpans][R][64 * NV];
    const Span sp = span_of<BACK>(p);
    const Lane l = lane_of<NV>(p, sp.group);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double A[NV], H[R][NV];
#pragma unroll
    for (int i = 0; i < NV; i++) { A[i] = 1.0; for (int r = 0; r < R; r++) H[r][i] = 0.0; }
    if (l.on)
        gated_formed(p.form, [&](auto form) {
            for (long long n = 0; n < p.span; n += K) {
                const long long s0 = sp.s0 + (BACK ? p.span - K - n : n);
                if (s0 >= sp.s1) continue;
                if (__all(s0 >= l.lo && s0 + K <= l.hi)) gated_fold_batch<T, form.value, NV, R, K, BACK, HASV, true>(p, l, s0, A, H);
                else gated_fold_batch<T, form.value, NV, R, K, BACK, HASV, false>(p, l, s0, A, H);
            }
        });
    const long long BD = p.groups * NV, at = sp.group * NV;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        s_a[wave][lane * NV + i] = A[i];
        if (l.on) p.span_a[sp.index * BD + at + i] = A[i];
#pragma unroll
        for (int r = 0; r < R; r++) {
            s_h[wave][r][lane * NV + i] = H[r][i];
            if (l.on) p.span_h[(sp.index * R + r) * BD + at + i] = H[r][i];
        }
    }
    __syncthreads();
    if (wave == 0 && l.on)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            double a = 1.0, h[R];
#pragma unroll
            for (int r = 0; r < R; r++) h[r] = 0.0;
            for (int w = 0; w < kGatedSpans; w++) {
                const double aw = s_a[w][lane * NV + i];
                a = gated_bound(a * aw);
#pragma unroll
                for (int r = 0; r < R; r++) h[r] = gated_apply(aw, h[r], s_h[w][r][lane * NV + i]);
            }
            p.block_a[sp.block * BD + at + i] = a;
#pragma unroll
            for (int r = 0; r < R; r++) p.block_h[(sp.block * R + r) * BD + at + i] = h[r];
        }
}

// The state in front of this wave's span: the workgroups in front of its own, folded by all waves together, then the spans in front of it in its own.
template <int NV, int R>
__device__ __forceinline__ void gated_carry(const GatedArgs& p, const Span& sp, bool on, float (&h)[R][NV])
{
    __shared__ double s_a[kGatedSpans][64 * NV];
    __shared__ double s_h[kGatedSpans][R][64 * NV];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long BD = p.groups * NV, at = sp.group * NV;
    const long long each = (sp.block + kGatedSpans - 1) / kGatedSpans;
    const long long b0 = wave * each, b1 = b0 + each < sp.block ? b0 + each : sp.block;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        double a = 1.0, c[R];
#pragma unroll
        for (int r = 0; r < R; r++) c[r] = 0.0;
        if (on) {
#pragma unroll 4
            for (long long b = b0; b < b1; b++) {
                const double ab = p.block_a[b * BD + at + i];
                a = gated_bound(a * ab);
#pragma unroll
                for (int r = 0; r < R; r++) c[r] = gated_apply(ab, c[r], p.block_h[(b * R + r) * BD + at + i]);
            }
        }
        s_a[wave][lane * NV + i] = a;
#pragma unroll
        for (int r = 0; r < R; r++) s_h[wave][r][lane * NV + i] = c[r];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; i++) {
        double c[R];
#pragma unroll
        for (int r = 0; r < R; r++) c[r] = h[r][i];
        for (int w = 0; w < kGatedSpans; w++)
#pragma unroll
            for (int r = 0; r < R; r++) c[r] = gated_apply(s_a[w][lane * NV + i], c[r], s_h[w][r][lane * NV + i]);
        if (on)
            for (int w = 0; w < wave; w++) {
                const long long q = sp.block * kGatedSpans + w;
                const double aq = p.span_a[q * BD + at + i];
#pragma unroll
                for (int r = 0; r < R; r++) c[r] = gated_apply(aq, c[r], p.span_h[(q * R + r) * BD + at + i]);
            }
#pragma unroll
        for (int r = 0; r < R; r++) h[r][i] = (float)c[r];
    }
}

template <typename T, int NV, int R, bool SPLIT>
__global__ __launch_bounds__(64 * (SPLIT ? kGatedSpans : kGatedWaves)) void gated_fwd_kernel(GatedArgs p)
{
    constexpr int K = GatedBatch<R>::value;
    Span sp;
    if (SPLIT) sp = span_of<false>(p);
    else { sp.group = block_of() * (64 * kGatedWaves) + threadIdx.x; sp.s0 = 0; sp.s1 = p.T; }
    const long long group = sp.group;
    const Lane l = lane_of<NV>(p, group);
    const long long out = (l.b * R) * p.D + l.d;                             // in B x R x D
    float h[R][NV];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < NV; i++) h[r][i] = p.initial ? p.initial[out + r * p.D + i] : 0.0f;
    if (SPLIT) gated_carry<NV, R>(p, sp, l.on, h);
    if (!l.on) return;
    gated_formed(p.form, [&](auto form) {
        for (long long s0 = sp.s0; s0 < sp.s1; s0 += K) {
            if (__all(s0 >= l.lo && s0 + K <= l.hi)) gated_fwd_batch<T, form.value, NV, R, K, true>(p, l, group, s0, h);
            else gated_fwd_batch<T, form.value, NV, R, K, false>(p, l, group, s0, h);
        }
    });
    if (!SPLIT || sp.index == p.blocks * kGatedSpans - 1)
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < NV; i++) p.last[out + r * p.D + i] = h[r][i];
}

template <typename T, int FORM, int NV, int R, int K, bool SPLIT, bool HASD, bool WHOLE>
__device__ __forceinline__ void gated_bwd_batch(const GatedArgs& p, const Lane& l, long long group, long long s0, float (&c)[R][NV])
{
    using P = Pack<T, NV>;
    P z[K], x[K][R], d[K][R];
    const long long dir = p.reverse ? -1 : 1, m0 = p.reverse ? p.T - 1 - s0 : s0;
    const T* gp = (const T*)p.gate + l.b * p.gate_b + m0 * p.gate_t + l.d;
    const T* xp = (const T*)p.x + l.b * p.x_b + m0 * p.x_t + l.d;
    const T* dp = (const T*)p.d_states + l.b * p.ds_b + m0 * p.ds_t + l.d;           // !HASD: not read
    float h[R][NV];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const Pack<float, NV> o = *(const Pack<float, NV>*)(p.marks + ((s0 / K) * R + r) * p.groups * NV + group * NV);
#pragma unroll
        for (int i = 0; i < NV; i++) h[r][i] = o.v[i];
    }
#pragma unroll
    for (int k = 0; k < K; k++)
    {
        if (WHOLE || (s0 + k >= l.lo && s0 + k < l.hi)) {
            z[k] = pack_load<!SPLIT, P>(gp);
#pragma unroll
            for (int r = 0; r < R; r++) {
                x[k][r] = pack_load<!SPLIT, P>(xp + r * p.x_r);
                if (HASD) d[k][r] = pack_load<!SPLIT, P>(dp + r * p.ds_r);
            }
        }
        gp += dir * p.gate_t; xp += dir * p.x_t; dp += dir * p.ds_t;
    }
    float before[K][R][NV];
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < NV; i++) before[k][r][i] = h[r][i];
        if (WHOLE || (s0 + k >= l.lo && s0 + k < l.hi)) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                float a, m;
                gated_am<FORM>(to_f(z[k].v[i]), a, m);
#pragma unroll
                for (int r = 0; r < R; r++) h[r][i] = __builtin_fmaf(a, h[r][i], m * to_f(x[k][r].v[i]));
            }
        }
    }
    const long long m1 = m0 + dir * (K - 1);
    T* ogp = (T*)p.d_gate + (l.b * p.T + m1) * p.D + l.d;                    // no d_gate, no d_x: not written
    T* oxp = (T*)p.d_x + ((l.b * p.T + m1) * R) * p.D + l.d;
#pragma unroll
    for (int k = K - 1; k >= 0; k--) {
        const bool in = WHOLE || (s0 + k >= l.lo && s0 + k < l.hi);
        P oz, ox[R];
#pragma unroll
        for (int i = 0; i < NV; i++) { oz.v[i] = from_f<T>(0.0f); for (int r = 0; r < R; r++) ox[r].v[i] = from_f<T>(0.0f); }
        if (in) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                float a, m, dz = 0.0f;
                gated_am<FORM>(to_f(z[k].v[i]), a, m);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float g = c[r][i] + (HASD ? to_f(d[k][r].v[i]) : 0.0f);
                    const float h0 = before[k][r][i];
                    dz = __builtin_fmaf(g, FORM == GSX_GATED_LINEAR ? h0 : FORM == GSX_GATED_BLEND ? to_f(x[k][r].v[i]) - h0 : -h0, dz);
                    ox[r].v[i] = from_f<T>(m * g);
                    c[r][i] = a * g;
                }
                oz.v[i] = from_f<T>(dz);
            }
        }
        if (WHOLE || s0 + k < p.T) {
            if (p.d_gate) pack_store(ogp, oz);
            if (p.d_x)
#pragma unroll
                for (int r = 0; r < R; r++) pack_store(oxp + r * p.D, ox[r]);
        }
        ogp -= dir * p.D; oxp -= dir * R * p.D;
    }
}

template <typename T, int NV, int R, bool SPLIT, bool HASD>
__global__ __launch_bounds__(64 * (SPLIT ? kGatedSpans : kGatedWaves)) void gated_bwd_kernel(GatedArgs p)
{
    constexpr int K = GatedBatch<R>::value;
    Span sp;
    if (SPLIT) sp = span_of<true>(p);
    else { sp.group = block_of() * (64 * kGatedWaves) + threadIdx.x; sp.s0 = 0; sp.s1 = p.T; }
    const long long group = sp.group;
    const Lane l = lane_of<NV>(p, group);
    const long long out = (l.b * R) * p.D + l.d;
    float c[R][NV];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < NV; i++) c[r][i] = p.d_last ? p.d_last[out + r * p.D + i] : 0.0f;
    if (SPLIT) gated_carry<NV, R>(p, sp, l.on, c);
    if (!l.on) return;
    gated_formed(p.form, [&](auto form) {
        for (long long n = (sp.s1 - sp.s0 + K - 1) / K; n > 0; n--) {
            const long long s0 = sp.s0 + (n - 1) * K;
            if (__all(s0 >= l.lo && s0 + K <= l.hi)) gated_bwd_batch<T, form.value, NV, R, K, SPLIT, HASD, true>(p, l, group, s0, c);
            else gated_bwd_batch<T, form.value, NV, R, K, SPLIT, HASD, false>(p, l, group, s0, c);
        }
    });
    if (p.d_initial && (!SPLIT || sp.index == p.blocks * kGatedSpans - 1))
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < NV; i++) p.d_initial[out + r * p.D + i] = c[r][i];
}

// One step in place, for a state that lives between calls: 12 bytes and more per element, and at a serving batch's size (64 x 2048)
// nothing but the launch.  The state may itself be the gate or the input: a lane reads its elements of all three before it writes.
template <typename T, int NV>
__global__ __launch_bounds__(kBlock) void gated_step_kernel(float* state, const T* gate, const T* x, long long n, int form)
{
    const long long i = (block_of() * kBlock + threadIdx.x) * NV;
    if (i >= n) return;                                                      // NV divides n
    Pack<float, NV> h = *(const Pack<float, NV>*)(state + i);
    const Pack<T, NV> z = *(const Pack<T, NV>*)(gate + i), v = *(const Pack<T, NV>*)(x + i);
    gated_formed(form, [&](auto known) {
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float a, m;
            gated_am<known.value>(to_f(z.v[k]), a, m);
            h.v[k] = __builtin_fmaf(a, h.v[k], m * to_f(v.v[k]));
        }
    });
    *(Pack<float, NV>*)(state + i) = h;
}

static int gated_check(const gsx_gated* s)
{
    if (!s || s->B < 0 || s->T < 0 || s->D < 0 || s->planes < 1 || s->planes > GSX_GATED_MAX_PLANES) return GSX_E_INVALID;
    if (s->dtype != GSX_F32 && s->dtype != GSX_BF16 && s->dtype != GSX_F16) return GSX_E_INVALID;
    if (s->form != GSX_GATED_LINEAR && s->form != GSX_GATED_BLEND && s->form != GSX_GATED_OVER) return GSX_E_INVALID;
    if (s->T >= (1ll << 40) || s->B >= (1ll << 31) || s->D >= (1ll << 31) || (s->B && s->D > (1ll << 40) / s->B)) return GSX_E_RANGE;
    return GSX_OK;
}

static size_t size_of(int dtype) { return dtype == GSX_F32 ? 4 : 2; }

// NV channels per lane want every row of every array on a boundary of NV elements
static bool aligned_for(const gsx_gated* s, int nv, bool backward)
{
    const int64_t e = (int64_t)size_of(s->dtype);
    auto at = [&](const void* p, int64_t size) { return ((uintptr_t)p & (uintptr_t)(size * nv - 1)) == 0; };
    auto by = [&](int64_t stride) { return stride % nv == 0; };
    if (s->D % nv || !at(s->gate, e) || !at(s->x, e)) return false;
    if (!by(s->gate_stride[0]) || !by(s->gate_stride[1]) || !by(s->x_stride[0]) || !by(s->x_stride[1]) || !by(s->x_stride[2])) return false;
    if (!at(s->marks, 4)) return false;
    if (!backward) return at(s->states, e);
    if (!at(s->d_gate, e) || !at(s->d_x, e)) return false;
    return !s->d_states || (at(s->d_states, e) && by(s->d_states_stride[0]) && by(s->d_states_stride[1]) && by(s->d_states_stride[2]));
}

static GatedArgs gated_args(const gsx_gated* s, int nv)
{
    GatedArgs p;
    p.gate = s->gate; p.x = s->x; p.initial = s->initial; p.lengths = s->lengths;
    p.states = s->states; p.last = s->last; p.marks = s->marks;
    p.d_states = s->d_states; p.d_last = s->d_last; p.d_gate = s->d_gate; p.d_x = s->d_x; p.d_initial = s->d_initial;
    p.T = s->T; p.D = s->D; p.row = s->D / nv; p.groups = s->B * p.row;
    p.gate_b = s->gate_stride[0]; p.gate_t = s->gate_stride[1];
    p.x_b = s->x_stride[0]; p.x_t = s->x_stride[1]; p.x_r = s->x_stride[2];
    p.ds_b = s->d_states_stride[0]; p.ds_t = s->d_states_stride[1]; p.ds_r = s->d_states_stride[2];
    p.form = s->form; p.reverse = s->reverse != 0;
    return p;
}

struct GatedPlan { int nv; int64_t span, blocks, columns; size_t span_a, span_h, block_a, block_h, bytes; };

// How a call is laid out.  A lane moves 4 bytes where the rows allow it: two channels of a 16-bit type, one in 32 bits (two there: 1 M channels x 60 steps 142 us both ways,
// 96 channels x 100001 steps 43 us against 38, whose waves are twice as many).  The steps are split when whole columns alone would leave the card short of kGatedWant waves
// (8 per CU), down to spans of two batches: a split walk reads its inputs twice.
constexpr int64_t kGatedWant = 2048;

static GatedPlan gated_plan(const gsx_gated* s, bool backward)
{
    GatedPlan g;
    const int64_t K = s->planes == 1 ? GatedBatch<1>::value : GatedBatch<2>::value, BD = s->B * s->D;
    g.nv = s->dtype != GSX_F32 && s->planes == 1 && aligned_for(s, 2, backward) ? 2 : 1;
    g.columns = ceil_div(BD / g.nv, 64);
    g.blocks = 1; g.span = s->T;
    g.span_a = g.span_h = g.block_a = g.block_h = g.bytes = 0;
    const int64_t spans = g.columns < kGatedWant ? ceil_div(kGatedWant, g.columns) : 1;
    int64_t span = ceil_div(ceil_div(s->T, spans), K) * K;
    if (span < 2 * K) span = 2 * K;
    if (spans == 1 || span * 2 > s->T) return g;
    g.span = span;
    g.blocks = ceil_div(ceil_div(s->T, span), kGatedSpans);
    const size_t n = (size_t)g.blocks * kGatedSpans;
    g.span_a = 0; g.bytes = align_up(n * BD * 8);
    g.span_h = g.bytes; g.bytes += align_up(n * s->planes * BD * 8);
    g.block_a = g.bytes; g.bytes += align_up((size_t)g.blocks * BD * 8);
    g.block_h = g.bytes; g.bytes += align_up((size_t)g.blocks * s->planes * BD * 8);
    return g;
}

template <typename T, int NV, int R>
static int gated_launch(const gsx_gated* s, const GatedPlan& g, bool backward, hipStream_t stream)
{
    GatedArgs p = gated_args(s, NV);
    if (g.bytes) {
        char* ws = (char*)s->ws;
        p.span = g.span; p.blocks = g.blocks; p.columns = g.columns;
        p.span_a = (double*)(ws + g.span_a); p.span_h = (double*)(ws + g.span_h);
        p.block_a = (double*)(ws + g.block_a); p.block_h = (double*)(ws + g.block_h);
        const dim3 dg((unsigned)(g.columns * g.blocks)), db(64 * kGatedSpans);           // some kGatedWant waves
        if (backward) {
            if (p.d_states) gated_fold_kernel<T, NV, R, true, true><<<dg, db, 0, stream>>>(p);
            else gated_fold_kernel<T, NV, R, true, false><<<dg, db, 0, stream>>>(p);
            GSX_LAUNCH_CHECK();
            if (p.d_states) gated_bwd_kernel<T, NV, R, true, true><<<dg, db, 0, stream>>>(p);
            else gated_bwd_kernel<T, NV, R, true, false><<<dg, db, 0, stream>>>(p);
        } else {
            gated_fold_kernel<T, NV, R, false, true><<<dg, db, 0, stream>>>(p);
            GSX_LAUNCH_CHECK();
            gated_fwd_kernel<T, NV, R, true><<<dg, db, 0, stream>>>(p);
        }
    } else {
        const int64_t blocks = ceil_div(p.groups, 64 * kGatedWaves);
        if (blocks > kMostBlocks) return GSX_E_RANGE;
        const dim3 dg = grid_of(blocks), db(64 * kGatedWaves);
        if (backward && p.d_states) gated_bwd_kernel<T, NV, R, false, true><<<dg, db, 0, stream>>>(p);
        else if (backward) gated_bwd_kernel<T, NV, R, false, false><<<dg, db, 0, stream>>>(p);
        else gated_fwd_kernel<T, NV, R, false><<<dg, db, 0, stream>>>(p);
    }
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

template <typename T>
static int gated_by_planes(const gsx_gated* s, const GatedPlan& g, bool backward, hipStream_t stream)
{
    switch (s->planes) {
    case 1:
        if constexpr (sizeof(T) == 2)
            if (g.nv == 2) return gated_launch<T, 2, 1>(s, g, backward, stream);
        return gated_launch<T, 1, 1>(s, g, backward, stream);
    case 2: return gated_launch<T, 1, 2>(s, g, backward, stream);
    case 3: return gated_launch<T, 1, 3>(s, g, backward, stream);
    default: return gated_launch<T, 1, 4>(s, g, backward, stream);
    }
}

static int gated_run(const gsx_gated* s, bool backward, void* stream)
{
    const GatedPlan g = gated_plan(s, backward);
    if (g.bytes && (!s->ws || ((uintptr_t)s->ws & 255))) return GSX_E_INVALID;
    if (s->ws_bytes < g.bytes) return GSX_E_CAPACITY;
    switch (s->dtype) {
    case GSX_F32: return gated_by_planes<float>(s, g, backward, (hipStream_t)stream);
    case GSX_BF16: return gated_by_planes<__bf16>(s, g, backward, (hipStream_t)stream);
    default: return gated_by_planes<_Float16>(s, g, backward, (hipStream_t)stream);
    }
}

}  // namespace gsx

using namespace gsx;

GSX_API int64_t gsx_gated_marks_floats(int64_t B, int64_t T, int32_t planes, int64_t D)
{
    if (B < 0 || T < 0 || D < 0 || planes < 1 || planes > GSX_GATED_MAX_PLANES) return GSX_E_INVALID;
    if (T >= (1ll << 40) || B >= (1ll << 31) || D >= (1ll << 31) || (B && D > (1ll << 40) / B)) return GSX_E_RANGE;        // as gated_check
    const int64_t batches = ceil_div(T, planes == 1 ? GatedBatch<1>::value : GatedBatch<2>::value), each = planes * B * D;
    return each && batches > (1ll << 60) / each ? (int64_t)GSX_E_RANGE : batches * each;
}

GSX_API size_t gsx_gated_workspace_bytes(const gsx_gated* s, int32_t backward)
{
    if (gated_check(s) != GSX_OK || s->B == 0 || s->D == 0) return 0;
    return gated_plan(s, backward != 0).bytes;
}

GSX_API int gsx_gated_scan_fwd(const gsx_gated* s, void* stream)
{
    const int st = gated_check(s);
    if (st != GSX_OK) return st;
    if (s->B == 0 || s->D == 0) return GSX_OK;
    if (!s->last || (s->T && (!s->gate || !s->x))) return GSX_E_INVALID;
    return gated_run(s, false, stream);
}

GSX_API int gsx_gated_scan_bwd(const gsx_gated* s, void* stream)
{
    const int st = gated_check(s);
    if (st != GSX_OK) return st;
    if (s->B == 0 || s->D == 0) return GSX_OK;
    if (s->T && (!s->gate || !s->x || !s->marks)) return GSX_E_INVALID;
    return gated_run(s, true, stream);
}

GSX_API int gsx_gated_step(int32_t dtype, int32_t form, int64_t n, float* state, const void* gate, const void* x, void* stream)
{
    if (n < 0 || (dtype != GSX_F32 && dtype != GSX_BF16 && dtype != GSX_F16)) return GSX_E_INVALID;
    if (form != GSX_GATED_LINEAR && form != GSX_GATED_BLEND && form != GSX_GATED_OVER) return GSX_E_INVALID;
    if (n == 0) return GSX_OK;
    if (!state || !gate || !x) return GSX_E_INVALID;
    const uintptr_t e = size_of(dtype);
    // an input that shares memory with the state at another place would be read by one lane and written by another
    auto meets = [&](const void* p) { return (uintptr_t)p < (uintptr_t)state + (uintptr_t)n * 4 && (uintptr_t)state < (uintptr_t)p + (uintptr_t)n * e && !(p == state && e == 4); };
    if (meets(gate) || meets(x)) return GSX_E_INVALID;
    const bool four = n % 4 == 0 && ((uintptr_t)state & 15) == 0 && ((uintptr_t)gate & (4 * e - 1)) == 0 && ((uintptr_t)x & (4 * e - 1)) == 0;
    const int64_t blocks = ceil_div(n, four ? 4 * kBlock : kBlock);
    if (blocks > kMostBlocks) return GSX_E_RANGE;
    const dim3 grid = grid_of(blocks), block(kBlock);
    hipStream_t st = (hipStream_t)stream;
#define GSX_STEP(T) do { if (four) gated_step_kernel<T, 4><<<grid, block, 0, st>>>(state, (const T*)gate, (const T*)x, n, form); \
                         else gated_step_kernel<T, 1><<<grid, block, 0, st>>>(state, (const T*)gate, (const T*)x, n, form); } while (0)
    if (dtype == GSX_F32) GSX_STEP(float);
    else if (dtype == GSX_BF16) GSX_STEP(__bf16);
    else GSX_STEP(_Float16);
#undef GSX_STEP
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}
