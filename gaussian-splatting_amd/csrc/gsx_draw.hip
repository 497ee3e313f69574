// gsx_draw.hip -- draws from softmax(logits / temperature), cut to the top k, the top p and the min p, by given random numbers.
// A row's weights are w_i = exp((l_i - top) / T) as shares of the largest.  The tokens ranked by (logit descending, index ascending),
// the cuts keep a prefix of the ranking: the first k; of these the fewest whose mass reaches p of their mass; of these the ones with
// w >= min_p.  A draw u is the lowest index whose inclusive mass over the kept tokens, in index order, exceeds u M.
// Which index a u falls on is a comparison of sums of up to millions of terms: weights and sums are held in 64 bits (the card's
// 64-bit vector FMA rate equals its 32-bit one, so a 64-bit exp per logit costs little beside reading the logits), and the masses of
// the histogram that ranks are whole numbers in two 64-bit limbs, so that the order of its atomics cannot change a result.
#include "gsx_common.h"

namespace gsx {

constexpr int kDrawBlock = 1024;
constexpr int kDrawBins = 256;
constexpr int kDrawEach = 4;                        // consecutive tokens per thread and tile
constexpr double kLimb = (double)(1ull << 36);      // a weight is hi 2^-36 + lo 2^-72; 2^27 weights fit a 64-bit sum of either

struct DrawArgs {
    const void* logits; long long row_stride, V, S;
    const void* uniforms;
    float temperature, top_p, min_p; int top_k, uniforms_f64;
    const float* temperatures; const float* top_ps; const float* min_ps; const int32_t* top_ks;
    long long* indices; float* logprobs;
    double* mass; double* total;                    // R x V inclusive masses, R totals (-1: the row has no valid settings)
    float* tops;
    uint32_t* keys; long long* bounds;              // per row: kept are the keys above, and of this key the indices below the bound
};

// logits as floats: NaN counts as -inf (a masked token), -0 as 0
template <typename T>
__device__ __forceinline__ float draw_logit(T v)
{
    const float f = (float)v;
    return f != f ? -__builtin_inff() : f + 0.0f;
}

// ascending unsigned order of the logits; never 0
__device__ __forceinline__ uint32_t draw_key(float l)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, l);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ double draw_weight(float l, float top, double inv_t)
{
    if (l == top) return 1.0;
    if (l == -__builtin_inff() || top == __builtin_inff()) return 0.0;
    return exp(((double)l - (double)top) * inv_t);
}

struct DrawRow { double inv_t, p, min_p; long long k; bool valid; };

__device__ __forceinline__ DrawRow draw_row(const DrawArgs& a, long long r)
{
    DrawRow s;
    const float t = a.temperatures ? a.temperatures[r] : a.temperature;
    const float p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float m = a.min_ps ? a.min_ps[r] : a.min_p;
    const int k = a.top_ks ? a.top_ks[r] : a.top_k;
    s.valid = t >= 0.0f && p > 0.0f && m >= 0.0f && m <= 1.0f;
    s.inv_t = t > 0.0f ? 1.0 / (double)t : 1.0;
    s.p = (double)p; s.min_p = (double)m;
    s.k = k > 0 && k < a.V ? k : a.V;
    if (t == 0.0f) { s.k = 1; s.p = 1.0; }           // the limit: the largest logit, its lowest index
    return s;
}

__device__ __forceinline__ double kept_weight(float l, long long i, uint32_t key, long long bound, float top, const DrawRow& set)
{
    const uint32_t q = draw_key(l);
    if (q < key || (q == key && i >= bound)) return 0.0;
    const double w = draw_weight(l, top, set.inv_t);
    return w < set.min_p ? 0.0 : w;
}

template <typename T>
__device__ __forceinline__ T block_reduce(T v, T* s_wave, T (*op)(T, T))
{
#pragma unroll
    for (int d = 32; d; d >>= 1) v = op(v, __shfl_xor(v, d, 64));
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) s_wave[wave] = v;
    __syncthreads();
    T r = s_wave[0];
    for (int w = 1; w < kDrawBlock / 64; w++) r = op(r, s_wave[w]);
    __syncthreads();
    return r;
}
__device__ __forceinline__ float op_maxf(float a, float b) { return fmaxf(a, b); }

// exclusive sums over the block's threads; *sum = the block's
template <typename T>
__device__ __forceinline__ T block_before(T v, T* s_wave, T* sum)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(incl, d, 64);
        if (lane >= d) incl += o;
    }
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    T base = 0, all = 0;
    for (int w = 0; w < kDrawBlock / 64; w++) {
        if (w == wave) base = all;
        all += s_wave[w];
    }
    *sum = all;
    __syncthreads();
    T before = __shfl_up(incl, 1, 64);
    return base + (lane ? before : (T)0);
}

struct DrawSel {                                    // LDS of the ranking
    uint32_t count[kDrawBins];
    unsigned long long hi[kDrawBins], lo[kDrawBins];
    uint32_t prefix;                                // key bits settled so far
    long long above_n; unsigned long long above_hi, above_lo;      // tokens in front of the settled bin, and their mass
    double total;
    uint32_t key; long long ties;                   // the last kept key, and how many of its tokens are kept
    long long bound;                                // ... as an index: ties at an index below it are kept
};

__device__ __forceinline__ double limbs(unsigned long long hi, unsigned long long lo) { return (double)hi * (1.0 / kLimb) + (double)lo * (1.0 / (kLimb * kLimb)); }

// One level, 8 key bits, of the ranking by count (the first k) or by mass (the fewest that reach p of what the count cut left: keys above
// floor_key, and of floor_key the indices below floor_bound).
template <typename T>
__device__ void draw_level(const T* row, long long V, float top, double inv_t, DrawSel& s, int shift, bool by_mass, uint32_t floor_key, long long floor_bound, long long k, double p)
{
    for (int b = threadIdx.x; b < kDrawBins; b += kDrawBlock) { s.count[b] = 0; s.hi[b] = 0; s.lo[b] = 0; }
    __syncthreads();
    const uint32_t prefix = s.prefix;
    for (long long i = threadIdx.x; i < V; i += kDrawBlock) {
        const float l = draw_logit(row[i]);
        const uint32_t key = draw_key(l);
        if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
        if (by_mass && (key < floor_key || (key == floor_key && i >= floor_bound))) continue;
        const int b = 255 - (int)((key >> shift) & 255);             // bin 0 holds the largest
        atomicAdd(&s.count[b], 1u);
        if (by_mass) {
            const double w = draw_weight(l, top, inv_t) * kLimb;
            const unsigned long long hi = (unsigned long long)w, lo = (unsigned long long)((w - (double)hi) * kLimb);
            atomicAdd(&s.hi[b], hi);
            atomicAdd(&s.lo[b], lo);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        if (by_mass && shift == 24) {                                // the mass that p is a share of: all that the count cut left
            unsigned long long hi = 0, lo = 0;
            for (int b = 0; b < kDrawBins; b++) { hi += s.hi[b]; lo += s.lo[b]; }
            s.total = limbs(hi, lo);
        }
        int b = 0;
        for (; b < kDrawBins - 1; b++) {
            if (by_mass ? limbs(s.above_hi + s.hi[b], s.above_lo + s.lo[b]) >= p * s.total : s.above_n + (long long)s.count[b] >= k) break;
            s.above_n += s.count[b]; s.above_hi += s.hi[b]; s.above_lo += s.lo[b];
        }
        s.prefix = prefix | (uint32_t)(255 - b) << shift;
        if (shift == 0) {
            s.key = s.prefix;
            const long long n = s.count[b];
            if (!by_mass) s.ties = k - s.above_n < n ? k - s.above_n : n;
            else {
                const double left = p * s.total - limbs(s.above_hi, s.above_lo);
                const double w = draw_weight(__builtin_bit_cast(float, s.key & 0x80000000u ? s.key & 0x7fffffffu : ~s.key), top, inv_t);
                long long m = w > 0.0 ? (long long)ceil(left / w) : n;
                s.ties = m < 1 ? 1 : m < n ? m : n;
            }
        }
    }
    __syncthreads();
}

template <typename T>
__device__ void draw_bound(const T* row, long long V, DrawSel& s, uint32_t* s_wave)
{
    const uint32_t key = s.key; const long long ties = s.ties;
    if (threadIdx.x == 0) s.bound = V;
    long long seen = 0;
    for (long long base = 0; base < V; base += kDrawBlock) {
        const long long i = base + threadIdx.x;
        const uint32_t is = i < V && draw_key(draw_logit(row[i])) == key;
        uint32_t sum;
        const uint32_t before = block_before<uint32_t>(is, s_wave, &sum);
        if (is && seen + before == ties - 1) s.bound = i + 1;
        seen += sum;
        if (seen >= ties) break;                                     // the same for every thread
    }
    __syncthreads();
}

// one workgroup per row: top, cuts, inclusive masses
template <typename T>
__global__ __launch_bounds__(kDrawBlock) void draw_mass_kernel(DrawArgs a)
{
    __shared__ DrawSel s;
    __shared__ double s_d[kDrawBlock / 64];
    __shared__ float s_f[kDrawBlock / 64];
    __shared__ uint32_t s_u[kDrawBlock / 64];
    const long long r = blockIdx.x, V = a.V;
    const T* row = (const T*)a.logits + r * a.row_stride;
    const DrawRow set = draw_row(a, r);
    float top = -__builtin_inff();
    for (long long i = threadIdx.x; i < V; i += kDrawBlock) top = fmaxf(top, draw_logit(row[i]));
    top = block_reduce<float>(top, s_f, op_maxf);
    if (!set.valid || top == -__builtin_inff()) {
        if (threadIdx.x == 0) { a.total[r] = -1.0; a.tops[r] = top; }
        return;
    }
    uint32_t key = 0; long long bound = V;                           // keep keys above `key`, and of `key` the indices below `bound`
    for (int cut = 0; cut < 2; cut++) {
        if (cut == 0 ? set.k >= V : !(set.p < 1.0)) continue;
        if (threadIdx.x == 0) { s.prefix = 0; s.above_n = 0; s.above_hi = 0; s.above_lo = 0; }
        __syncthreads();
        for (int shift = 24; shift >= 0; shift -= 8) draw_level(row, V, top, set.inv_t, s, shift, cut == 1, key, bound, set.k, set.p);
        draw_bound(row, V, s, s_u);
        key = s.key; bound = s.bound;
        __syncthreads();
    }
    if (threadIdx.x == 0) { a.keys[r] = key; a.bounds[r] = bound; }
    double carry = 0.0;
    double* mass = a.mass + r * V;
    for (long long base = 0; base < V; base += kDrawBlock * kDrawEach) {
        const long long i0 = base + threadIdx.x * kDrawEach;
        double w[kDrawEach], sum = 0.0, all;
#pragma unroll
        for (int j = 0; j < kDrawEach; j++) {
            w[j] = 0.0;
            if (i0 + j < V) {
                w[j] = kept_weight(draw_logit(row[i0 + j]), i0 + j, key, bound, top, set);
            }
            sum += w[j];
        }
        double at = carry + block_before<double>(sum, s_d, &all);
#pragma unroll
        for (int j = 0; j < kDrawEach; j++) { at += w[j]; if (i0 + j < V) mass[i0 + j] = at; }
        carry += all;
    }
    if (threadIdx.x == 0) { a.total[r] = carry; a.tops[r] = top; }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void draw_pick_kernel(DrawArgs a, long long n)
{
    const long long t = (long long)blockIdx.x * kBlock + threadIdx.x;
    if (t >= n) return;
    const long long r = t / a.S;
    const double total = a.total[r];
    if (!(total > 0.0)) { a.indices[t] = -1; if (a.logprobs) a.logprobs[t] = -__builtin_inff(); return; }
    const double* mass = a.mass + r * a.V;
    double u = a.uniforms_f64 ? ((const double*)a.uniforms)[t] : (double)((const float*)a.uniforms)[t];
    u = u >= 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;                        // NaN: 0
    const double want = u * mass[a.V - 1];
    long long lo = 0, hi = a.V - 1;                                  // the lowest index with mass above `want`, or the last one
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (mass[mid] > want) hi = mid; else lo = mid + 1;
    }
    // sums of neighbouring threads' spans may differ by a rounding from each other: never a token without weight, the last one with weight for u = 1
    const DrawRow set = draw_row(a, r);
    const float top = a.tops[r];
    const T* row = (const T*)a.logits + r * a.row_stride;
    while (lo > 0 && !(kept_weight(draw_logit(row[lo]), lo, a.keys[r], a.bounds[r], top, set) > 0.0)) lo--;
    a.indices[t] = lo;
    if (a.logprobs) {
        const float l = draw_logit(row[lo]);
        a.logprobs[t] = (float)((l == top ? 0.0 : ((double)l - (double)top) * set.inv_t) - log(total));
    }
}

static int draw_check(const gsx_draw* s)
{
    if (!s || s->R < 0 || s->V < 0 || s->S < 0) return GSX_E_INVALID;
    if (s->dtype != GSX_F32 && s->dtype != GSX_BF16 && s->dtype != GSX_F16) return GSX_E_INVALID;
    if (!s->temperatures && !(s->temperature >= 0.0f)) return GSX_E_INVALID;
    if (!s->top_ps && !(s->top_p > 0.0f)) return GSX_E_INVALID;
    if (!s->min_ps && !(s->min_p >= 0.0f && s->min_p <= 1.0f)) return GSX_E_INVALID;
    if (!s->top_ks && s->top_k < 0) return GSX_E_INVALID;
    if (s->V > GSX_DRAW_MAX_V || s->R > 0x7fffffffll || s->S > (1ll << 38) || (s->R && s->S > (1ll << 38) / s->R)) return GSX_E_RANGE;
    return GSX_OK;
}

struct DrawLayout { size_t mass, total, bounds, tops, keys, bytes; };

static DrawLayout draw_layout(const gsx_draw* s)
{
    DrawLayout l;
    size_t at = 0;
    l.mass = at; at += align_up((size_t)s->R * (size_t)s->V * 8);
    l.total = at; at += align_up((size_t)s->R * 8);
    l.bounds = at; at += align_up((size_t)s->R * 8);
    l.tops = at; at += align_up((size_t)s->R * 4);
    l.keys = at; at += align_up((size_t)s->R * 4);
    l.bytes = at;
    return l;
}

template <typename T>
static int draw_run(const DrawArgs& a, int64_t R, hipStream_t stream)
{
    draw_mass_kernel<T><<<dim3((unsigned)R), dim3(kDrawBlock), 0, stream>>>(a);
    GSX_LAUNCH_CHECK();
    const int64_t n = R * a.S;
    draw_pick_kernel<T><<<dim3((unsigned)ceil_div(n, kBlock)), dim3(kBlock), 0, stream>>>(a, n);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

}  // namespace gsx

using namespace gsx;

GSX_API size_t gsx_draw_workspace_bytes(const gsx_draw* s)
{
    return draw_check(s) == GSX_OK ? draw_layout(s).bytes : 0;
}

GSX_API int gsx_draw_indices(const gsx_draw* s, void* stream)
{
    const int st = draw_check(s);
    if (st != GSX_OK) return st;
    if (s->R == 0 || s->S == 0) return GSX_OK;
    if ((s->V && !s->logits) || !s->uniforms || !s->indices || !s->ws || ((uintptr_t)s->ws & 255)) return GSX_E_INVALID;
    const DrawLayout l = draw_layout(s);
    if (s->ws_bytes < l.bytes) return GSX_E_CAPACITY;
    char* ws = (char*)s->ws;
    DrawArgs a;
    a.logits = s->logits; a.row_stride = s->row_stride; a.V = s->V; a.S = s->S;
    a.uniforms = s->uniforms; a.uniforms_f64 = s->uniforms_f64 != 0;
    a.temperature = s->temperature; a.top_p = s->top_p; a.min_p = s->min_p; a.top_k = s->top_k;
    a.temperatures = s->temperatures; a.top_ps = s->top_ps; a.min_ps = s->min_ps; a.top_ks = s->top_ks;
    a.indices = (long long*)s->indices; a.logprobs = s->logprobs;
    a.mass = (double*)(ws + l.mass); a.total = (double*)(ws + l.total); a.tops = (float*)(ws + l.tops);
    a.bounds = (long long*)(ws + l.bounds); a.keys = (uint32_t*)(ws + l.keys);
    switch (s->dtype) {
    case GSX_F32: return draw_run<float>(a, s->R, (hipStream_t)stream);
    case GSX_BF16: return draw_run<__bf16>(a, s->R, (hipStream_t)stream);
    default: return draw_run<_Float16>(a, s->R, (hipStream_t)stream);
    }
}
