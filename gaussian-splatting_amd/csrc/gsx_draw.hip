// gsx_draw.hip -- draws from softmax(logits / temperature), cut to the top k, the top p and the min p, by given random numbers.
// A row's weights are w_i = exp((l_i - top) / T) as shares of the largest.  The tokens ranked by (logit descending, index ascending),
// the cuts keep a prefix of the ranking: the first k; of these the fewest whose mass reaches p of their mass; of these the ones with
// w >= min_p.  A draw u is the lowest index whose inclusive mass over the kept tokens, in index order, exceeds u M.
//
// Which index a u falls on is a comparison of sums of up to millions of terms, and so is where the top p ends: weights and sums are held in
// 64 bits (the card's 64-bit vector FMA rate equals its 32-bit one; the exp below is 17 of them), and the masses of histograms are whole
// numbers in two limbs, so that the order of atomics cannot change a result.
//
// Three ways, by the length of a row:
//   short  (V <= 512)      a few lanes to a row, its tokens in registers; the cuts by bisection of the key with ballots and masked sums.
//   row    (one workgroup) the row read once per pass, from cache after the first: the top, a histogram, the tokens of the bin where a
//                          cut falls, the masses, the draws -- one launch.
//   parts  (a few long rows) the same passes as kernels, a row cut into parts over the card.
// A histogram's 2048 bins are 1/64 of a unit of (top - l) / T wide: the tokens spread over hundreds of bins (few collisions in LDS), and the bin where
// a cut falls holds few enough tokens to be ranked in LDS.  Where it does not (ties, extreme temperatures), narrower histograms of the 59-bit rank
// (key, index) follow until it does: every row ends, whatever its values.
// Measured with three inputs in turn, us a call and what bounds it: 640000 rows of 32, 4 draws each, 55 (short; issue, 475 instructions a wave of eight rows); one row of 5000 16 (row; a workgroup's chain
// of passes); 256 rows of 131072 in 32 bits 117 (row; the top 16, the histogram 17, the pass of 64-bit weights 50 by issue, the decision 7, against 26 for the bytes);
// 64 rows of 100003 in 16 bits 49 (parts; seven launches that wait for one another); one row of 1 M and 1 M draws 48, of 6 M with a top p 138 (parts; loads that wait).
#include <type_traits>
#include "gsx_common.h"

namespace gsx {

constexpr int kDrawBins = 2048;                     // of the first histogram
constexpr float kDrawBinsPerUnit = 64.0f;
constexpr int kDrawFine = 512;                      // bins of the narrower ones
constexpr int kDrawCand = 1024;                     // tokens that are ranked in LDS
// Which way, thread count and kernels a call takes; us a call, by length, rows and draws, of N(0, 2) logits in 32 bits cut to k = 50, p = 0.9, one input
// repeated in a graph (here and at the rules further down: a few per cent less than with inputs in turn, on both sides):
// Longest row of the short way.  100000 rows of 500: 532, with a workgroup each 2866; one row of 500: 19 against 15.
constexpr int kDrawShort = 512;
// Longest row whose workgroup is of 512 threads and decides by itself in every case; 1024 threads read a longer one sooner while it has a CU to itself, and of more rows
// than CUs two of 512 share one.  1 x 32000: 30.4 with 512 threads, 29.7 with 1024; 1000 x 32000: 90, 117; 256 x 60000: 57, 50; 300 x 60000: 68, 83; 512 x 131072: 136, 149.
constexpr int64_t kDrawSmall = 16384, kDrawSmallOfMany = 65536, kDrawCus = 256;
constexpr int kDrawWaveTiles = 2048;                // spans of 256 tokens whose masses are kept in LDS: rows of up to 512 k tokens
// Draws per row that its workgroup makes itself, a wave to a draw; of more a kernel with a thread to each.  1000 x 2000: 16 draws 41.8 in the row's workgroup, 42.9 in a
// kernel; 32: 52, 43; 64: 71, 44.  10 x 20000: 32 draws 33, 40; 64: 38, 40.
constexpr int64_t kDrawInRow = 64, kDrawInRowOfMany = 16;
// Longer rows are cut into parts, where there are at most kDrawFewRows of them.  1 x 48000: 32.4 in parts, 34.8 by a workgroup; 32 x 48000: 39, 36; 32 x 64000: 43, 41;
// 64 x 131072: 46, 61; 128 x 40000: 43, 36; 128 x 131072: 65, 67; 192 x 131072: 87, 72.
constexpr int64_t kDrawLong = 49152, kDrawFewRows = 128;
constexpr int kDrawExact = 512;                     // threads where a cut is searched for: all of the registers that it needs
constexpr int kDrawIndexBits = 27;

typedef unsigned long long u64;

struct DrawArgs {
    const void* logits; long long row_stride, R, V, S;
    const void* uniforms;
    float temperature, top_p, min_p; int top_k, uniforms_f64;
    double inv_t;                                   // of `temperature`: a 64-bit division per row would cost as much as an exp
    const float* temperatures; const float* top_ps; const float* min_ps; const int32_t* top_ks;
    long long* indices; float* logprobs;
    // workspace of rows whose draws are made by a kernel of their own
    double* spans;                                  // [row][spans_row]: inclusive mass behind every group of four tokens
    double* total; float* tops; u64* floors;        // per row: kept mass (-1: none), top, lowest kept rank
    uint32_t* left;                                 // per row: its cuts are left to the exact way
    long long spans_row;
    long long share;                                // short rows: draws that a wave makes of its rows', the next share being another workgroup's
    double* lines;                                  // every 16th of them again, side by side (rows in parts)
    // rows in parts: `part` groups of four places each, `parts` to a row; `walkers` workgroups per row where a workgroup takes several parts
    int part, parts, nodes, nodes_log, walkers, cuts;
    float* walk_top;                                // [row][walker]
    double* part_mass;                              // [row][part]
    u64* hist;                                      // [row][walker][bin]
    uint32_t* row_n; u64* row_m;                    // [row][bin]
    struct DrawNear* near;                          // [row]
    double* sums;                                   // [row][walker][2]: 64-bit mass in front of the bracket, and the total's part
    u64* list; uint32_t* list_n; long long list_most;        // [row]: ranks of the tokens where the cuts may end
};

// ---- tokens ---------------------------------------------------------------------------------------------------------------
// logits as floats: NaN counts as -inf (a masked token).  A NaN float further on is "not a token" (a place outside the row).
template <typename T>
__device__ __forceinline__ float draw_logit(T v)
{
    const float f = (float)v;
    return f != f ? -__builtin_inff() : f;
}

// ascending unsigned order of the logits, -0 as 0
__device__ __forceinline__ uint32_t draw_key(float l)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, l + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float draw_unkey(uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// ascending order of (logit, -index): a cut keeps the tokens whose rank is at least some floor
constexpr u64 kDrawIndexMask = (1ull << kDrawIndexBits) - 1;
__device__ __forceinline__ u64 draw_rank(float l, int i) { return (u64)draw_key(l) << kDrawIndexBits | (kDrawIndexMask - (u64)i); }
__device__ __forceinline__ float draw_rank_logit(u64 rank) { return draw_unkey((uint32_t)(rank >> kDrawIndexBits)); }
__device__ __forceinline__ int draw_rank_index(u64 rank) { return (int)(kDrawIndexMask - (rank & kDrawIndexMask)); }

// A floor as the token that it is: kept are larger logits, and equal ones up to its index.  Rank 0: everything is kept.
struct DrawFloor {
    float l; int i;
    __device__ __forceinline__ DrawFloor(u64 rank) : l(rank ? draw_rank_logit(rank) : -__builtin_inff()), i(rank ? draw_rank_index(rank) : 0x7fffffff) {}
    __device__ __forceinline__ bool keeps(float v, int at) const { return v > l || (v == l && at <= i); }
};

// exp(x) for x <= 0; 0 below -708, for -inf and for NaN.  x = n ln 2 + r with ln 2 in two parts (the first of 32 bits: n times it is exact),
// |r| <= ln 2 / 2, the Taylor sum to r^13 / 13! (what is left out is below 5e-18), times 2^n by the exponent's bits.  n comes from an addition
// that leaves it in the low bits: conversions and roundings of 64-bit numbers run at a quarter of the rate of the FMA.
__device__ __forceinline__ double draw_exp(double x)
{
    const double t = fma(x, 0x1.71547652b82fep+0, 0x1.8p52), n = t - 0x1.8p52;
    double r = fma(n, -0x1.62e42ff000000p-1, x);
    r = fma(n, 0x1.718432a1b0e26p-35, r);
    double s = 1.0 / 6227020800.0;
    s = fma(s, r, 1.0 / 479001600.0);
    s = fma(s, r, 1.0 / 39916800.0);
    s = fma(s, r, 1.0 / 3628800.0);
    s = fma(s, r, 1.0 / 362880.0);
    s = fma(s, r, 1.0 / 40320.0);
    s = fma(s, r, 1.0 / 5040.0);
    s = fma(s, r, 1.0 / 720.0);
    s = fma(s, r, 1.0 / 120.0);
    s = fma(s, r, 1.0 / 24.0);
    s = fma(s, r, 1.0 / 6.0);
    s = fma(s, r, 0.5);
    s = fma(s, r, 1.0);
    s = fma(s, r, 1.0);
    const u64 bits = __builtin_bit_cast(u64, s);
    const uint32_t hi = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(u64, t) << 20);
    const double v = __builtin_bit_cast(double, (u64)hi << 32 | (uint32_t)bits);
    return x >= -708.0 ? v : 0.0;
}

// 1 at the top, 0 where masked and outside the row; the top is finite (Places)
__device__ __forceinline__ double draw_weight(float l, float top, double inv_t) { return draw_exp(((double)l - (double)top) * inv_t); }

// bin of the first histogram: does not fall as l falls
__device__ __forceinline__ float draw_depth(float l, float top, float scale)
{
    return fminf((top - l) * scale, (float)(kDrawBins - 1));         // NaN (-inf at an endless temperature): the last
}
__device__ __forceinline__ int draw_bin(float l, float top, float scale)
{
    const float t = (top - l) * scale;
    return t < (float)(kDrawBins - 1) ? (int)t : kDrawBins - 1;
}

// a weight as whole numbers: w = hi 2^-31 + lo 2^-63, to the nearest; sums of 2^27 of either fit 64 bits
__device__ __forceinline__ void draw_limbs(double w, uint32_t& hi, uint32_t& lo)
{
    const double t = w * 0x1p31;
    hi = (uint32_t)t;
    lo = (uint32_t)fmin((t - (double)hi) * 0x1p32 + 0.5, 4294967295.0);
}
__device__ __forceinline__ double limbs(u64 hi, u64 lo) { return (double)hi * 0x1p-31 + (double)lo * 0x1p-63; }

// the largest power of two up to n
__device__ __forceinline__ int draw_power(int n) { return 1 << (31 - __builtin_clz(n)); }

// How many of the n ascending numbers at(0) .. at(n - 1) lie at or below `want`, n - 1 at most: the place of a draw.  Steps of falling powers of two, no branches; `top` is the
// largest power of two below 2 n.
template <typename At>
__device__ __forceinline__ int draw_place(const At& at, int n, int top, double want)
{
    int place = 0;
    for (int step = top; step; step >>= 1) {
        const int i = place + step - 1;
        place = i < n - 1 && at(i < n ? i : n - 1) <= want ? place + step : place;
    }
    return place;
}

struct DrawRow { double inv_t, p, min_p; long long k; float scale; bool valid; };

__device__ __forceinline__ DrawRow draw_row(const DrawArgs& a, long long r)
{
    DrawRow s;
    const float t = a.temperatures ? a.temperatures[r] : a.temperature;
    const float p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float m = a.min_ps ? a.min_ps[r] : a.min_p;
    const int k = a.top_ks ? a.top_ks[r] : a.top_k;
    s.valid = t >= 0.0f && p > 0.0f && m >= 0.0f && m <= 1.0f;
    s.inv_t = a.inv_t;
    if (a.temperatures) s.inv_t = t > 0.0f ? 1.0 / (double)t : 1.0;
    s.scale = (float)(s.inv_t * (double)kDrawBinsPerUnit);
    s.p = (double)p; s.min_p = (double)m;
    s.k = k > 0 && k < a.V ? k : a.V;
    if (t == 0.0f) { s.k = 1; s.p = 1.0; }           // the limit: the largest logit, its lowest index
    return s;
}

__device__ __forceinline__ double draw_uniform(const DrawArgs& a, long long t)
{
    const double u = a.uniforms_f64 ? ((const double*)a.uniforms)[t] : (double)((const float*)a.uniforms)[t];
    return u >= 0.0 ? (u < 1.0 ? u : 0x1.fffffffffffffp-1) : 0.0;    // NaN: 0; u total stays below the total, also when rounded
}

// Where rounding has led a draw to a place `q` (> 0) without weight: the place to try next, in front of it.  Sums at(i) of two orders of addition differ by some units of
// 2^-53 (less than 2^-47 of them) where no weight lies between, so the last place with weight is the first whose sum comes that near to the one in front of q.
// One by one, a thread would walk over a whole row whose kept tokens lie at its start.
template <typename At>
__device__ __forceinline__ int draw_back(const At& at, int q)
{
    const double least = at(q - 1) * (1.0 - 0x1p-47);
    int a = 0, b = q - 1;
    while (a < b) {
        const int mid = (a + b) >> 1;
        if (at(mid) >= least) b = mid; else a = mid + 1;
    }
    return a;
}

__device__ __forceinline__ double draw_kept(float l, int i, const DrawFloor& floor, float top, const DrawRow& set)
{
    if (!__any(floor.keeps(l, i))) return 0.0;                       // most waves beyond a cut keep nothing
    const double w = draw_weight(l, top, set.inv_t);
    return floor.keeps(l, i) && w >= set.min_p ? w : 0.0;
}

// log(x) for x >= 1 (a row's top weighs 1): the 32-bit one and a Newton step, y + x e^-y - 1, which squares its error of 1e-6
__device__ __forceinline__ double draw_log(double x)
{
    const double y = (double)(__builtin_amdgcn_logf((float)x) * 0.693147181f);
    return y + (x * draw_exp(-y) - 1.0);
}

__device__ __forceinline__ float draw_logprob(float l, float top, double inv_t, double log_total)
{
    return (float)(((double)l - (double)top) * inv_t - log_total);
}

// A row as groups of four tokens on a boundary of four: place 4 g + j is token 4 g + j - off.
template <typename T>
struct Four { T v[4]; } __attribute__((aligned(4 * sizeof(T))));

// Where a row's top is +inf, such tokens share all mass: they are taken as 0 and all others as -inf.
template <typename T>
struct Places {
    const T* base; int V, off; bool infinite;
    __device__ __forceinline__ Places(const DrawArgs& a, long long r) : V((int)a.V), infinite(false)
    {
        const T* row = (const T*)a.logits + r * a.row_stride;
        off = (int)(((uintptr_t)row / sizeof(T)) & 3);
        base = row - off;
    }
    __device__ __forceinline__ float finite_top(float top) { infinite = top == __builtin_inff(); return infinite ? 0.0f : top; }
    __device__ __forceinline__ int groups() const { return (V + off + 3) >> 2; }
    __device__ __forceinline__ bool whole(int g) const { return 4 * g >= off && 4 * g + 4 <= V + off; }        // all four of its places are tokens
    // A group's load and what follows on it are apart, so that several loads are in flight: any use of one waits for it.  fetch() reads the nearest
    // group that lies in the row whole (rows here have more than 512 tokens); finish() reads the two at the ends token by token.
    __device__ __forceinline__ Four<T> fetch(int g) const
    {
        const int first = off ? 1 : 0, last = ((V + off) >> 2) - 1;
        g = g < first ? first : g > last ? last : g;
        return *(const Four<T>*)(base + 4ll * g);
    }
    // places outside the row, and groups from `end` on, are NaN
    __device__ __forceinline__ void finish(int g, int end, const Four<T>& f, float (&l)[4]) const
    {
        const int i0 = 4 * g - off;
#pragma unroll
        for (int j = 0; j < 4; j++) l[j] = draw_logit(f.v[j]);
        if (i0 < 0 || i0 + 4 > V || g >= end)
#pragma unroll
            for (int j = 0; j < 4; j++) l[j] = g < end && i0 + j >= 0 && i0 + j < V ? draw_logit(base[4ll * g + j]) : __builtin_nanf("");
        if (infinite)
#pragma unroll
            for (int j = 0; j < 4; j++) l[j] = l[j] != l[j] ? l[j] : l[j] == __builtin_inff() ? 0.0f : -__builtin_inff();
    }
    __device__ __forceinline__ void load(int g, int end, float (&l)[4]) const { finish(g, end, fetch(g), l); }
    // N groups, `step` apart
    template <int N>
    __device__ __forceinline__ void load_many(int g, int step, int end, float (&l)[N][4]) const
    {
        Four<T> f[N];
#pragma unroll
        for (int q = 0; q < N; q++) f[q] = fetch(g + q * step);
#pragma unroll
        for (int q = 0; q < N; q++) finish(g + q * step, end, f[q], l[q]);
    }
};

// ---- wave and workgroup helpers --------------------------------------------------------------------------------------------------
// Values moved between lanes by DPP: register moves of a few cycles, where a shuffle is a round trip through the LDS unit that the histograms' atomics
// keep busy.  Lanes without a source get zero (with all rows enabled by the instruction's own bound control, without a move).
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T draw_dpp(T v)
{
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, ROWS == 0xf));
    } else {
        const u64 u = __builtin_bit_cast(u64, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, ROWS == 0xf);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, ROWS == 0xf);
        return __builtin_bit_cast(T, (u64)hi << 32 | lo);
    }
}
// inclusive sums over the wave: within rows of 16 lanes, then the rows' last lanes onto the rows behind them
template <typename T>
__device__ __forceinline__ T draw_wave_scan(T v)
{
    v += draw_dpp<0x111, 0xf>(v);     // row_shr:1
    v += draw_dpp<0x112, 0xf>(v);
    v += draw_dpp<0x114, 0xf>(v);
    v += draw_dpp<0x118, 0xf>(v);
    v += draw_dpp<0x142, 0xa>(v);     // row_bcast:15 onto rows 1 and 3
    v += draw_dpp<0x143, 0xc>(v);     // row_bcast:31 onto rows 2 and 3
    return v;
}
template <typename T>
__device__ __forceinline__ T draw_wave_shift(T v) { return draw_dpp<0x138, 0xf>(v); }       // from the lane before; zero into lane 0

template <int NT, typename T>
__device__ __forceinline__ T draw_before(T v, T* s_wave, T* sum)       // exclusive sums over the threads
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T incl = draw_wave_scan(v);
    __syncthreads();                                                 // s_wave may still be read from the call before
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    T base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        if (w == wave) base = all;
        all += s_wave[w];
    }
    *sum = all;
    return base + draw_wave_shift(incl);
}

template <int CTRL, int ROWS>                       // lanes without a source keep their own
__device__ __forceinline__ float draw_dpp_or(float v)
{
    const int u = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, CTRL, ROWS, 0xf, false));
}

// sums of two values over the workgroup
template <int NT>
__device__ __forceinline__ void draw_sums(double& x, double& y, double (*s_wave)[2])
{
    x = draw_wave_scan(x); y = draw_wave_scan(y);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) { s_wave[threadIdx.x >> 6][0] = x; s_wave[threadIdx.x >> 6][1] = y; }
    __syncthreads();
    x = s_wave[0][0]; y = s_wave[0][1];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) { x += s_wave[w][0]; y += s_wave[w][1]; }
}

template <int NT>
__device__ __forceinline__ float draw_max(float v, float* s_wave)
{
    v = fmaxf(v, draw_dpp_or<0x111, 0xf>(v));
    v = fmaxf(v, draw_dpp_or<0x112, 0xf>(v));
    v = fmaxf(v, draw_dpp_or<0x114, 0xf>(v));
    v = fmaxf(v, draw_dpp_or<0x118, 0xf>(v));
    v = fmaxf(v, draw_dpp_or<0x142, 0xa>(v));
    v = fmaxf(v, draw_dpp_or<0x143, 0xc>(v));
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = s_wave[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) r = fmaxf(r, s_wave[w]);
    return r;
}

struct DrawHist { uint32_t count[kDrawBins]; u64 hi[kDrawBins], lo[kDrawBins]; };
struct DrawFine { uint32_t count[kDrawFine]; u64 hi[kDrawFine], lo[kDrawFine]; };
struct DrawCand { u64 rank[kDrawCand], ranked[kDrawCand]; };

// The first try at the cuts of a row: where the histogram's bounds let them end.  Bins: k in bin bk, p in one of lo .. hi.
struct DrawNear { int bk, lo, hi; long long above_k, to_bk; int before_bk, upto_hi; bool sure; };       // above_k, to_bk: tokens in front of bin bk, and with it

// What the threads of a workgroup share while a cut is found
struct DrawCut {
    long long above_n; u64 above_hi, above_lo;      // tokens in front of the bin, and their mass: base and the limbs
    double base;
    int bin; uint32_t in_bin, slots; int last;
    u64 lo, hi;                                     // ranks of the bin
    u64 floor_rank; double mass;                    // the answer: the lowest kept rank, the mass kept
    DrawNear near;
    u64 wave_u[16]; uint32_t wave_n[16]; double wave_d[16], wave_2[16][2]; float wave_f[16];
};

// the value of the lane whose number differs in bit D
template <int D>
__device__ __forceinline__ u64 draw_lane_xor(u64 v)
{
    if constexpr (D == 1) return draw_dpp<0xB1, 0xf>(v);
    else if constexpr (D == 2) return draw_dpp<0x4E, 0xf>(v);
    else if constexpr (D == 4) return draw_dpp<0x1B, 0xf>(draw_dpp<0x141, 0xf>(v));      // the half row mirrored, then each quad
    else if constexpr (D == 8) return draw_dpp<0x141, 0xf>(draw_dpp<0x140, 0xf>(v));     // the row mirrored, then each half
    else return __shfl_xor(v, D, 64);
}
template <int SIZE, int D>
__device__ __forceinline__ u64 draw_sort_step(u64 v, int lane)
{
    const u64 o = draw_lane_xor<D>(v);
    const bool larger = ((lane & D) == 0) == ((lane & SIZE) == 0);   // this lane keeps the larger one
    v = (o > v) == larger ? o : v;
    if constexpr (D > 1) return draw_sort_step<SIZE, D / 2>(v, lane);
    else return v;
}
// descending over the wave: a bitonic network of 21 steps
__device__ __forceinline__ u64 draw_sort_wave(u64 v, int lane)
{
    v = draw_sort_step<2, 1>(v, lane);
    v = draw_sort_step<4, 2>(v, lane);
    v = draw_sort_step<8, 4>(v, lane);
    v = draw_sort_step<16, 8>(v, lane);
    v = draw_sort_step<32, 16>(v, lane);
    return draw_sort_step<64, 32>(v, lane);
}

// Ranks cand.rank[0 .. m), all different, sorted descending into cand.ranked (m at most NT): each wave sorts its 64 in registers, then every one looks its
// place up in the other waves' by bisection.  (Counting the larger ones costs m^2 / 128 LDS reads, a network over the workgroup 55
// steps with barriers: 10 and 8 us at 400; this 2.)
template <int NT>
__device__ __forceinline__ void draw_rank_cand(DrawCand& cand, int m)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, runs = (m + 63) >> 6;
    const u64 mine = wave < runs ? draw_sort_wave(t < m ? cand.rank[t] : 0, lane) : 0;
    __syncthreads();
    u64* run = cand.rank;                                            // they stay the first m, in another order
    if (wave < runs) run[t] = mine;
    __syncthreads();
    if (wave < runs) {
        int place = lane;
        for (int w0 = 0; w0 < runs; w0 += 4) {                       // four bisections at a time
            int at[4] = {0, 0, 0, 0};
#pragma unroll
            for (int step = 32; step; step >>= 1)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int w = w0 + q < runs ? w0 + q : runs - 1;
                    if (run[w * 64 + at[q] + step - 1] > mine) at[q] += step;
                }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int w = w0 + q;
                if (w < runs && w != wave) place += at[q] + (run[w * 64 + at[q]] > mine ? 1 : 0);
            }
        }
        if (mine) cand.ranked[place] = mine;                         // no rank is 0
    }
    __syncthreads();
}

// The first of bins 0 .. last where what lies in and in front of it reaches k tokens or `want` mass, or else `last`; c.above_* move up to it (masses only with_mass).
template <int NT>
__device__ __forceinline__ void draw_find(DrawCut& c, const uint32_t* count, const u64* hi, const u64* lo, int bins, int last, bool by_mass, bool with_mass, long long k, double want)
{
    const int per = bins > NT ? bins / NT : 1, b0 = threadIdx.x * per;
    uint32_t n = 0, all_n; u64 h = 0, l = 0, all;
    const double base = c.base;
    const bool mine = b0 < bins;
    if (mine)
        for (int b = b0; b < b0 + per; b++) { n += count[b]; if (with_mass) { h += hi[b]; l += lo[b]; } }
    const long long start_n = c.above_n; const u64 start_h = c.above_hi, start_l = c.above_lo;
    long long at_n = start_n + draw_before<NT, uint32_t>(n, c.wave_n, &all_n);
    u64 at_h = start_h, at_l = start_l;
    if (with_mass) { at_h += draw_before<NT, u64>(h, c.wave_u, &all); at_l += draw_before<NT, u64>(l, c.wave_u, &all); }
    __syncthreads();
    if (mine) {
        bool before = by_mass ? b0 > 0 && base + limbs(at_h, at_l) >= want : at_n >= k;
        for (int b = b0; b < b0 + per && b <= last && !before; b++) {
            const long long next_n = at_n + count[b];
            const u64 next_h = at_h + (with_mass ? hi[b] : 0), next_l = at_l + (with_mass ? lo[b] : 0);
            const bool here = by_mass ? base + limbs(next_h, next_l) >= want : next_n >= k;
            if (here || b == last) { c.bin = b; c.in_bin = count[b]; c.above_n = at_n; c.above_hi = at_h; c.above_lo = at_l; }
            before = here;
            at_n = next_n; at_h = next_h; at_l = next_l;
        }
    }
    __syncthreads();
}

// Finds where a cut ends among the tokens of bins bin0 .. bin1 (c.in_bin of them at most) whose rank is at least `floor_rank`.  each(f) calls f(l, rank)
// for every token of the source, over all threads.
template <int NT, typename Each>
__device__ __forceinline__ void draw_resolve(DrawCut& c, DrawFine& fine, DrawCand& cand, const Each& each, float top, double inv_t, float scale, int bin0, int bin1, u64 floor_rank, bool by_mass, bool with_mass, long long k, double want)
{
    u64 lo = floor_rank, hi = ~0ull;
    uint32_t n = c.in_bin;
    const int most = NT < kDrawCand ? NT : kDrawCand;
    bool narrowed = false;
    while (n > (uint32_t)most) {
        if (!narrowed) {                                             // the ranks of the bin: its keys are neighbours
            if (threadIdx.x < 2) {
                uint32_t a = draw_key(-__builtin_inff()), b = draw_key(__builtin_inff());
                // the lowest key whose bin is at most bin1; one below the lowest key whose bin is less than bin0
                const int want_bin = threadIdx.x == 0 ? bin1 : bin0 - 1;
                b += threadIdx.x;                                    // "none" for bin 0
                while (a < b) {
                    const uint32_t mid = a + (b - a) / 2;
                    if (draw_bin(draw_unkey(mid), top, scale) <= want_bin) b = mid; else a = mid + 1;
                }
                if (threadIdx.x == 0) c.lo = (u64)a << kDrawIndexBits;
                else c.hi = ((u64)a << kDrawIndexBits) - 1;
            }
            __syncthreads();
            lo = c.lo > lo ? c.lo : lo; hi = c.hi;
            narrowed = true;
        }
        int shift = 0;
        while (((hi - lo) >> shift) >= (u64)kDrawFine) shift++;
        for (int b = threadIdx.x; b < kDrawFine; b += NT) { fine.count[b] = 0; fine.hi[b] = 0; fine.lo[b] = 0; }
        __syncthreads();
        each([&](float l, u64 rank) {
            if (rank < lo || rank > hi) return;
            const int b = (int)((hi - rank) >> shift);
            atomicAdd(&fine.count[b], 1u);
            if (with_mass) {
                uint32_t wh, wl;
                draw_limbs(draw_weight(l, top, inv_t), wh, wl);
                atomicAdd(&fine.hi[b], (u64)wh);
                atomicAdd(&fine.lo[b], (u64)wl);
            }
        });
        __syncthreads();
        draw_find<NT>(c, fine.count, fine.hi, fine.lo, kDrawFine, (int)((hi - lo) >> shift), by_mass, with_mass, k, want);
        hi -= (u64)c.bin << shift;
        const u64 width = (1ull << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
        n = c.in_bin;
        __syncthreads();
    }
    if (threadIdx.x == 0) { c.slots = 0; c.last = 0; }
    __syncthreads();
    each([&](float l, u64 rank) {
        if (rank < lo || rank > hi) return;
        if (!narrowed) { const int b = draw_bin(l, top, scale); if (b < bin0 || b > bin1) return; }
        const uint32_t slot = atomicAdd(&c.slots, 1u);
        if (slot < (uint32_t)most) cand.rank[slot] = rank;
    });
    __syncthreads();
    const int m = (int)(c.slots < (uint32_t)most ? c.slots : (uint32_t)most);
    const int t = threadIdx.x;
    draw_rank_cand<NT>(cand, m);
    double all;
    const double w = t < m ? draw_weight(draw_rank_logit(cand.ranked[t]), top, inv_t) : 0.0;
    const double above = c.base + limbs(c.above_hi, c.above_lo);
    const double before = draw_before<NT, double>(w, c.wave_d, &all);
    const bool in = t < m && (t == 0 || (by_mass ? above + before < want : c.above_n + t < k));
    if (in) atomicMax(&c.last, t);
    __syncthreads();
    if (t == c.last && m) { c.floor_rank = cand.ranked[t]; c.mass = above + before + w; }
    if (t == 0 && !m) { c.floor_rank = lo; c.mass = above; }
    __syncthreads();
}

__device__ __forceinline__ void draw_hist_add(DrawHist& h, float l, float top, double inv_t, float scale, bool by_mass)
{
    const int b = draw_bin(l, top, scale);
    atomicAdd(&h.count[b], 1u);
    if (by_mass) {
        uint32_t wh, wl;
        draw_limbs(draw_weight(l, top, inv_t), wh, wl);
        if (wh) atomicAdd(&h.hi[b], (u64)wh);
        if (wl) atomicAdd(&h.lo[b], (u64)wl);
    }
}

// Both cuts from the first histogram; -> the lowest kept rank.
template <int NT, typename Each>
__device__ __forceinline__ u64 draw_cuts(DrawCut& c, const DrawHist& hist, DrawFine& fine, DrawCand& cand, const Each& each, float top, const DrawRow& set, bool by_k, bool by_p)
{
    u64 floor_rank = 0;
    int last = kDrawBins - 1;
    double total = 0.0;
    if (by_k) {
        if (threadIdx.x == 0) { c.above_n = 0; c.above_hi = 0; c.above_lo = 0; c.base = 0.0; }
        __syncthreads();
        draw_find<NT>(c, hist.count, hist.hi, hist.lo, kDrawBins, last, false, by_p, set.k, 0.0);
        last = c.bin;
        draw_resolve<NT>(c, fine, cand, each, top, set.inv_t, set.scale, c.bin, c.bin, 0, false, by_p, set.k, 0.0);
        floor_rank = c.floor_rank;
        total = c.mass;
        __syncthreads();
    }
    if (by_p) {
        if (!by_k) {
            u64 h = 0, l = 0, all_h, all_l;
            for (int b = threadIdx.x; b < kDrawBins; b += NT) { h += hist.hi[b]; l += hist.lo[b]; }
            draw_before<NT, u64>(h, c.wave_u, &all_h);
            draw_before<NT, u64>(l, c.wave_u, &all_l);
            total = limbs(all_h, all_l);
        }
        if (threadIdx.x == 0) { c.above_n = 0; c.above_hi = 0; c.above_lo = 0; c.base = 0.0; }
        __syncthreads();
        draw_find<NT>(c, hist.count, hist.hi, hist.lo, kDrawBins, last, true, true, 0, set.p * total);
        draw_resolve<NT>(c, fine, cand, each, top, set.inv_t, set.scale, c.bin, c.bin, floor_rank, true, true, 0, set.p * total);
        floor_rank = c.floor_rank > floor_rank ? c.floor_rank : floor_rank;
    }
    return floor_rank;
}

// The cuts in one pass over the row behind the histogram, where few enough tokens lie where they may end.
// The histogram counts tokens and adds up 32-bit weights: near enough to say in which bins the top p may end (a bracket, usually
// of one bin), not where.  One pass then adds up the 64-bit weights of the tokens in front of the bracket, which are kept whatever
// happens, and collects the tokens inside it and in the bin where the top k end; these few are ranked and decided exactly.  `false`: too
// many of them, or the sums do not bear the bracket out; the longer way has no such limits.
// A bin is one 64-bit word, one atomic per token: its tokens from bit 45 on, below the 32-bit weights in units of 2^-26 (2^19 tokens fit both).
constexpr int kDrawCountBit = 45;
constexpr int64_t kDrawMostInHist = 1 << 19;
__device__ __forceinline__ void draw_near_add(u64* bins, float l, float top, float scale, float units)
{
    const uint32_t m = (uint32_t)fmaf(__builtin_amdgcn_exp2f((l - top) * units), 0x1p26f, 0.5f);      // NaN: 0
    atomicAdd(&bins[draw_bin(l, top, scale)], (1ull << kDrawCountBit) + m);
}
__device__ __forceinline__ uint32_t draw_near_count(u64 v) { return (uint32_t)(v >> kDrawCountBit); }
__device__ __forceinline__ u64 draw_near_mass(u64 v) { return v & ((1ull << kDrawCountBit) - 1); }

// The 64-bit weights of a group's tokens at depths `t` (places outside the row weigh nothing): those in front of `lo` to `above`, and to the total all of them (kAll), those in
// front of `upto` (kUpto) or none; -> those in front of lo that min_p keeps.  The kinds are the compiler's: as choices per token they took a tenth of the pass.
enum DrawTotal { kNone, kAll, kUpto };
template <int TOTAL, bool LEAST>
__device__ __forceinline__ double draw_group_sums(const float (&l)[4], const float (&t)[4], float lo, float upto, float top, const DrawRow& set, double& above, double& total)
{
    double front = 0.0, kept = 0.0, all = 0.0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const double w = draw_weight(l[j], top, set.inv_t), f = t[j] < lo ? w : 0.0;
        front += f;
        if (LEAST) kept += f >= set.min_p ? f : 0.0;
        if (TOTAL != kNone) all += TOTAL == kAll || t[j] < upto ? w : 0.0;
    }
    above += front; total += all;
    return LEAST ? kept : front;
}

// where the cuts may end, from the histogram; c.near
template <int NT, typename Count, typename Mass>
__device__ __forceinline__ void draw_bracket(DrawCut& c, const Count& count, const Mass& mass, const DrawRow& set, long long V, bool by_k, bool by_p)
{
    constexpr int per = kDrawBins / NT;
    const int b0 = threadIdx.x * per;
    if (threadIdx.x == 0) { c.near.bk = kDrawBins - 1; c.near.above_k = c.near.to_bk = 0; c.near.lo = c.near.hi = kDrawBins - 1; }
    uint32_t n = 0, all_n; u64 m = 0, all_m = 0, at_m = 0;
#pragma unroll
    for (int j = 0; j < per; j++) { if (by_k) n += count(b0 + j); if (by_p) m += mass(b0 + j); }
    if (by_k) {
        long long at = draw_before<NT, uint32_t>(n, c.wave_n, &all_n);
#pragma unroll
        for (int j = 0; j < per; j++) {
            const long long next = at + count(b0 + j);
            if (at < set.k && next >= set.k) { c.near.bk = b0 + j; c.near.above_k = at; c.near.to_bk = next; }
            at = next;
        }
    }
    if (by_p) {
        at_m = draw_before<NT, u64>(m, c.wave_u, &all_m);
        __syncthreads();
        // mass in front of bin bk and with it, and what the sums of 32-bit weights may be off: 2^-15 of them and half a unit per token
        const int bk = c.near.bk;
        double low = (double)all_m, high = low;
        if (by_k) {
            if (bk / per == (int)threadIdx.x) {
                u64 a = at_m;
#pragma unroll
                for (int j = 0; j < per; j++) { if (b0 + j == bk) { c.lo = a; c.hi = a + mass(b0 + j); } a += mass(b0 + j); }
            }
            __syncthreads();
            low = (double)c.lo; high = (double)c.hi;
        }
        const double off = (double)V * 0.5;
        low = set.p * (low * (1.0 - 0x1p-15) - off); high = set.p * (high * (1.0 + 0x1p-15) + off);
        const double want_lo = low * (1.0 - 0x1p-15) - off, want_hi = high * (1.0 + 0x1p-15) + off;
        u64 at = at_m;
#pragma unroll
        for (int j = 0; j < per; j++) {
            const u64 next = at + mass(b0 + j);
            const int b = b0 + j;
            if (b <= bk) {
                if ((b == 0 || (double)at < want_lo) && ((double)next >= want_lo || b == bk)) c.near.lo = b;
                if ((b == 0 || (double)at < want_hi) && ((double)next >= want_hi || b == bk)) c.near.hi = b;
            }
            at = next;
        }
    }
    __syncthreads();
}

// The collected tokens (c.slots of them) ranked, and the cuts among them.  above: the 64-bit mass of all tokens in front of bin near.lo; total: of
// all in front of bin near.bk (of all, without a top k).
template <int NT>
__device__ __forceinline__ bool draw_decide(DrawCut& c, DrawCand& cand, const DrawRow& set, float top, bool by_k, bool by_p, double above, double total, bool all_listed = false)
{
    const int most = NT < kDrawCand ? NT : kDrawCand, t = threadIdx.x;
    if (c.slots > (uint32_t)most) return false;
    const int m = (int)c.slots;
    draw_rank_cand<NT>(cand, m);
    if (t == 0) { c.near.before_bk = 0; c.near.upto_hi = 0; c.near.sure = false; c.last = 0; }
    __syncthreads();
    const float l = draw_rank_logit(cand.ranked[t]);
    const int bin = t < m ? draw_bin(l, top, set.scale) : kDrawBins;
    const u64 front = __ballot(bin < c.near.bk), upto = __ballot(bin <= c.near.hi);
    if ((t & 63) == 0) { atomicAdd(&c.near.before_bk, (int)__popcll(front)); atomicAdd(&c.near.upto_hi, (int)__popcll(upto)); }
    __syncthreads();
    int n = m;                                                       // candidates that the top k leaves
    if (by_k) {
        const long long left = all_listed ? set.k : (long long)c.near.before_bk + set.k - c.near.above_k;
        n = left < m ? (int)left : m;
    }
    double all;
    const double w = t < n ? draw_weight(l, top, set.inv_t) : 0.0;
    const double before = draw_before<NT, double>(w, c.wave_d, &all);
    if (!by_p) {
        if (t == 0) c.floor_rank = cand.ranked[n - 1];
        __syncthreads();
        return true;
    }
    // the candidates of bin bk, where it lies behind the bracket, count for the total only
    double tail = 0.0, none = 0.0;
    if (by_k) { tail = all_listed || t >= c.near.before_bk ? w : 0.0; draw_sums<NT>(tail, none, c.wave_2); }
    const double want = set.p * (total + tail);
    const int upto_n = c.near.upto_hi < n ? c.near.upto_hi : n;
    const bool in = t < upto_n && ((t == 0 && c.near.lo == 0) || above + before < want);
    if (in) atomicMax(&c.last, t + 1);
    // borne out: the first candidate is kept, and all of them reach the share, or nothing lies behind them
    if (t == upto_n - 1) c.near.sure = above + before + w >= want || c.near.hi == c.near.bk;
    __syncthreads();
    const int last = c.last;
    if (!c.near.sure || last == 0) return false;
    if (t == 0) c.floor_rank = cand.ranked[last - 1];
    __syncthreads();
    return true;
}

// The cuts of a row exactly from the first histogram on: for rows that the quicker way cannot decide (ties, brackets of too many tokens).  The workgroups of 512 threads
// (short enough rows, the floor of rows in parts) go on with it at once; behind those of 1024, whose registers it would not leave room for, a kernel of its own does.
template <typename T, int NT>
__device__ __forceinline__ u64 draw_exact_floor(const DrawArgs& a, const Places<T>& row, const DrawRow& set, float top, DrawCut& c, DrawHist& hist, DrawFine& fine, DrawCand& cand)
{
    const int groups = row.groups();
    auto each = [&](auto f) {
        for (int g = threadIdx.x; g < groups; g += NT) {
            float l[4];
            row.load(g, groups, l);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (l[j] == l[j]) f(l[j], draw_rank(l[j], 4 * g + j - row.off));
        }
    };
    const bool by_k = set.k < a.V, by_p = set.p < 1.0;
    for (int b = threadIdx.x; b < kDrawBins; b += NT) { hist.count[b] = 0; hist.hi[b] = 0; hist.lo[b] = 0; }
    __syncthreads();
    each([&](float l, u64) { draw_hist_add(hist, l, top, set.inv_t, set.scale, by_p); });
    __syncthreads();
    const u64 floor_rank = draw_cuts<NT>(c, hist, fine, cand, each, top, set, by_k, by_p);
    __syncthreads();
    return floor_rank;
}

// ---- one workgroup per row -----------------------------------------------------------------------------------------------------
// Masses and draws of a row whose lowest kept rank is known; `tiled`: the tiles' masses lie in `tile` already.
template <typename T, int NT, bool PICK>
__device__ __forceinline__ void draw_row_draws(const DrawArgs& a, long long r, const Places<T>& row, const DrawRow& set, float raw_top, float top, u64 floor_rank, bool tiled, double* tile, double* s_wave)
{
    constexpr int kWaves = NT / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, groups = row.groups();
    auto all_groups = [&](auto f) {                                  // every thread of a wave, also where the wave reaches beyond the row
        for (int g0 = 0; g0 < groups; g0 += 4 * NT) {
            float l[4][4];
            row.load_many(g0 + tid, NT, groups, l);
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (g0 + q * NT < groups) f(l[q], g0 + q * NT + tid);
        }
    };
    const DrawFloor floor(floor_rank);
    auto mass4 = [&](const float (&l)[4], int g, double (&w)[4]) {
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            w[j] = draw_kept(l[j], 4 * g + j - row.off, floor, top, set);
            sum += w[j];
        }
        return sum;
    };
    if (PICK) {
        // masses of 256 tokens, one wave's groups, in LDS; then the inclusive sums of these
        if (!tiled)
            all_groups([&](const float (&l)[4], int g) {
                double w[4], sum = mass4(l, g, w);
                sum = draw_wave_scan(sum);
                if (lane == 63) tile[g >> 6] = sum;
            });
        __syncthreads();
        const int tiles = (int)((groups + 63) >> 6), per = (tiles + NT - 1) / NT;
        double sum = 0.0, total;
        for (int q = tid * per; q < (tid + 1) * per && q < tiles; q++) sum += tile[q];
        double at = draw_before<NT, double>(sum, s_wave, &total);
        for (int q = tid * per; q < (tid + 1) * per && q < tiles; q++) { at += tile[q]; tile[q] = at; }
        __syncthreads();
        const double log_total = draw_log(total);
        for (long long s = wave; s < a.S; s += kWaves) {             // a wave per draw
            const double want = draw_uniform(a, r * a.S + s) * total;
            const int lo = draw_place([&](int i) { return tile[i]; }, tiles, draw_power(tiles), want);
            // the first token in the tile that exceeds; where rounding leaves none, the last one with weight
            for (int q = lo;;) {
                const int g = q * 64 + lane;
                float l[4];
                row.load(g, groups, l);
                double w[4], incl = draw_wave_scan(mass4(l, g, w));
                double run = (q ? tile[q - 1] : 0.0) + draw_wave_shift(incl);
                int hit = -1, any = -1;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    run += w[j];
                    if (w[j] > 0.0) { any = j; if (hit < 0 && run > want) hit = j; }
                }
                const u64 hits = __ballot(hit >= 0), some = __ballot(any >= 0);
                if (!some) {
                    if (q == 0) break;                               // not with a top that weighs 1
                    q = draw_back([&](int i) { return tile[i]; }, q);
                    continue;
                }
                const int who = hits ? __ffsll((long long)hits) - 1 : 63 - __clzll((long long)some);
                if (lane == who) {
                    const int j = hits ? hit : any;
                    float lj = l[0];
#pragma unroll
                    for (int e = 1; e < 4; e++) lj = e == j ? l[e] : lj;
                    a.indices[r * a.S + s] = 4 * g + j - row.off;
                    if (a.logprobs) a.logprobs[r * a.S + s] = draw_logprob(lj, top, set.inv_t, log_total);
                }
                break;
            }
        }
    } else {
        // the groups' masses in the workspace; then the inclusive sums of these
        double* spans = a.spans + r * a.spans_row;
        const int n = groups;
        all_groups([&](const float (&l)[4], int g) {
            double w[4];
            const double sum = mass4(l, g, w);
            if (g < n) spans[g] = sum;
        });
        __syncthreads();
        double carry = 0.0;
        for (int b = 0; b < n; b += 4 * NT) {
            double v[4], sum = 0.0, all;
#pragma unroll
            for (int j = 0; j < 4; j++) { const int q = b + 4 * tid + j; v[j] = q < n ? spans[q] : 0.0; sum += v[j]; }
            double at = carry + draw_before<NT, double>(sum, s_wave, &all);
#pragma unroll
            for (int j = 0; j < 4; j++) { const int q = b + 4 * tid + j; at += v[j]; if (q < n) spans[q] = at; }
            carry += all;
        }
        if (tid == 0) { a.total[r] = carry; a.tops[r] = raw_top; a.floors[r] = floor_rank; }
    }
}

template <typename T, int NT, bool PICK, bool EXACT>
__global__ __launch_bounds__(NT) void draw_row_kernel(DrawArgs a)
{
    struct Tiles { u64 hi[kDrawBins], lo[kDrawBins]; };
    struct Cand { DrawCand cand; };
    union Fine { DrawFine fine; DrawCand cand; };
    __shared__ std::conditional_t<EXACT, DrawHist, Tiles> hist;      // the bins, then the candidates' masses by tile
    __shared__ std::conditional_t<EXACT, Fine, Cand> sh;
    __shared__ double tile[PICK ? kDrawWaveTiles : 1];
    __shared__ DrawCut c;
    const long long r = block_of();
    if (r >= a.R) return;
    const int tid = threadIdx.x, lane = tid & 63;
    if (!EXACT && a.cuts && tid == 0) a.left[r] = 0;
    Places<T> row(a, r);
    const int groups = row.groups();
    const DrawRow set = draw_row(a, r);
    float top = -__builtin_inff();
    constexpr int kAhead = 2;                                        // groups in flight per thread, here and below: 256 rows of 131072, one input repeated, 113 us with 2, 114 with 4, 121 with 8, 116 with 1
    for (int g = tid; g < groups; g += kAhead * NT) {
        float l[kAhead][4];
        row.load_many(g, NT, groups, l);
#pragma unroll
        for (int q = 0; q < kAhead; q++)
#pragma unroll
            for (int j = 0; j < 4; j++) top = fmaxf(top, l[q][j]);
    }
    top = draw_max<NT>(top, c.wave_f);
    if (!set.valid || top == -__builtin_inff()) {
        if (PICK) {
            for (long long s = tid; s < a.S; s += NT) { a.indices[r * a.S + s] = -1; if (a.logprobs) a.logprobs[r * a.S + s] = -__builtin_inff(); }
        } else if (tid == 0) a.total[r] = -1.0;
        return;
    }
    const float raw_top = top;
    top = row.finite_top(top);
    auto all_groups = [&](auto f) {                                  // every thread of a wave, also where the wave reaches beyond the row
        for (int g0 = 0; g0 < groups; g0 += kAhead * NT) {
            float l[kAhead][4];
            row.load_many(g0 + tid, NT, groups, l);
#pragma unroll
            for (int q = 0; q < kAhead; q++)
                if (g0 + q * NT < groups) f(l[q], g0 + q * NT + tid);
        }
    };
    const bool by_k = set.k < a.V, by_p = set.p < 1.0;
    u64 floor_rank = 0;
    bool tiled = false;                                              // the tiles' masses are there already
    if (by_k || by_p) {
        for (int b = tid; b < kDrawBins; b += NT) hist.hi[b] = 0;
        __syncthreads();
        const float units = (float)(set.inv_t * 0x1.71547652b82fep+0);
        all_groups([&](const float (&l)[4], int g) {
            if (__all(row.whole(g)))                                 // no choice per token: 3 us of a row of 131072
#pragma unroll
                for (int j = 0; j < 4; j++) draw_near_add(hist.hi, l[j], top, set.scale, units);
            else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (l[j] == l[j]) draw_near_add(hist.hi, l[j], top, set.scale, units);
        });
        __syncthreads();
        draw_bracket<NT>(c, [&](int b) { return draw_near_count(hist.hi[b]); }, [&](int b) { return draw_near_mass(hist.hi[b]); }, set, a.V, by_k, by_p);
        const int bk = c.near.bk, lo = by_p ? c.near.lo : bk, hi = by_p ? c.near.hi : bk;
        if (tid == 0) c.slots = 0;
        if (PICK) for (int q = tid; q < kDrawWaveTiles; q += NT) { hist.hi[q] = 0; hist.lo[q] = 0; tile[q] = 0.0; }
        __syncthreads();
        // 64-bit weights: of all tokens for the total of a top p, in front of the bracket for its sum and for the tiles
        const float lo_t = (float)lo, hi_t = (float)(hi + 1), bk_t = (float)(by_k ? bk : kDrawBins), front = fminf(lo_t, bk_t);
        double above = 0.0, total = 0.0;
        auto pass = [&](auto kind, auto least) {
            all_groups([&](const float (&l)[4], int g) {
                float t[4];
                bool in[4], some = false, sums = kind == kAll;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    t[j] = draw_depth(l[j], top, set.scale);
                    in[j] = l[j] == l[j] && ((t[j] >= lo_t && t[j] < hi_t) || (t[j] >= bk_t && t[j] < bk_t + 1.0f));
                    some |= in[j];
                    sums |= t[j] < (kind == kUpto ? bk_t : front);
                }
                if (__any(some))
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (in[j]) {
                            const uint32_t slot = atomicAdd(&c.slots, 1u);
                            if (slot < (uint32_t)(NT < kDrawCand ? NT : kDrawCand)) sh.cand.rank[slot] = draw_rank(l[j], 4 * g + j - row.off);
                        }
                if (!__any(sums)) return;                            // its tile has been cleared
                double sum = draw_group_sums<kind.value, least.value>(l, t, front, bk_t, top, set, above, total);
                if (PICK && lo > 0) {
                    sum = draw_wave_scan(sum);
                    if (lane == 63) tile[g >> 6] = sum;
                }
            });
        };
        auto pass_of = [&](auto kind) {
            if (set.min_p > 0.0) pass(kind, std::true_type{});
            else pass(kind, std::false_type{});
        };
        if (!by_p) pass_of(std::integral_constant<int, kNone>{});
        else if (by_k) pass_of(std::integral_constant<int, kUpto>{});
        else pass_of(std::integral_constant<int, kAll>{});
        __syncthreads();
        if (by_p) draw_sums<NT>(above, total, c.wave_2);
        __syncthreads();
        if (draw_decide<NT>(c, sh.cand, set, top, by_k, by_p, above, total)) {
            floor_rank = c.floor_rank;
            if (PICK) {
                if (tid < (int)c.slots) {                            // the kept candidates' weights, as whole numbers: any order gives the same sums
                    const u64 rank = sh.cand.rank[tid];
                    const double w = draw_weight(draw_rank_logit(rank), top, set.inv_t);
                    if (rank >= floor_rank && !(w < set.min_p)) {
                        const int q = (draw_rank_index(rank) + row.off) >> 8;
                        uint32_t wh, wl;
                        draw_limbs(w, wh, wl);
                        atomicAdd(&hist.hi[q], (u64)wh);
                        atomicAdd(&hist.lo[q], (u64)wl);
                    }
                }
                __syncthreads();
                const int tiles = (int)((groups + 63) >> 6);
                for (int q = tid; q < tiles; q += NT) tile[q] += limbs(hist.hi[q], hist.lo[q]);
                tiled = true;
            }
        } else if constexpr (EXACT) {
            __syncthreads();
            floor_rank = draw_exact_floor<T, NT>(a, row, set, top, c, hist, sh.fine, sh.cand);
        } else {                                                     // left to draw_exact_kernel
            if (tid == 0) { a.left[r] = 1; a.tops[r] = raw_top; }
            return;
        }
        __syncthreads();
    }
    draw_row_draws<T, NT, PICK>(a, r, row, set, raw_top, top, floor_rank, tiled, tile, c.wave_d);
}

// the rows that the kernel before left: their cuts exactly, from the first histogram on, then their draws
template <typename T, bool PICK>
__global__ __launch_bounds__(kDrawExact) void draw_exact_kernel(DrawArgs a)
{
    constexpr int NT = kDrawExact;
    __shared__ DrawHist hist;
    __shared__ union { DrawFine fine; DrawCand cand; } sh;
    __shared__ double tile[PICK ? kDrawWaveTiles : 1];
    __shared__ DrawCut c;
    const long long r = block_of();
    if (r >= a.R || !a.left[r]) return;
    Places<T> row(a, r);
    const DrawRow set = draw_row(a, r);
    const float raw_top = a.tops[r], top = row.finite_top(raw_top);
    const u64 floor_rank = draw_exact_floor<T, NT>(a, row, set, top, c, hist, sh.fine, sh.cand);
    draw_row_draws<T, NT, PICK>(a, r, row, set, raw_top, top, floor_rank, false, tile, c.wave_d);
}

// The draw within a group whose masses begin at `run`: the first token that exceeds, or where rounding leaves none the last one with weight; -1: none
// has any.
template <typename T>
__device__ __forceinline__ int draw_in_group(const Places<T>& row, int g, const float (&l)[4], double run, double want, const DrawFloor& floor, float top, const DrawRow& set, float& at_l)
{
    int index = -1; bool found = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = 4 * g + j - row.off;
        const double w = draw_kept(l[j], i, floor, top, set);
        run += w;
        if (!found && w > 0.0) { index = i; at_l = l[j]; found = run > want; }
    }
    return index;
}

// a thread per draw: the group by bisection, then its tokens one after the other
template <typename T>
__global__ __launch_bounds__(kBlock) void draw_pick_kernel(DrawArgs a, long long n)
{
    const long long t = block_of() * kBlock + threadIdx.x;
    if (t >= n) return;
    const long long r = t / a.S;
    const double total = a.total[r];
    if (!(total > 0.0)) { a.indices[t] = -1; if (a.logprobs) a.logprobs[t] = -__builtin_inff(); return; }
    Places<T> row(a, r);
    const DrawRow set = draw_row(a, r);
    const float top = row.finite_top(a.tops[r]);
    const DrawFloor floor(a.floors[r]);
    const double* spans = a.spans + r * a.spans_row;
    const double want = draw_uniform(a, t) * total;
    const int lo = draw_place([&](int i) { return spans[i]; }, row.groups(), draw_power(row.groups()), want);
    int index = -1; float at_l = 0.0f;
    for (int q = lo;; q = draw_back([&](int i) { return spans[i]; }, q)) {
        float l[4];
        row.load(q, row.groups(), l);
        index = draw_in_group(row, q, l, q ? spans[q - 1] : 0.0, want, floor, top, set, at_l);
        if (index >= 0 || q == 0) break;
    }
    a.indices[t] = index;
    if (a.logprobs) a.logprobs[t] = draw_logprob(at_l, top, set.inv_t, draw_log(total));
}

// ---- a few long rows, in parts over the card -------------------------------------------------------------------------------------
constexpr int kDrawPart = 256;                      // threads of a part's workgroup
constexpr int kDrawFewWalkers = 32;
constexpr int kDrawWalk = 512;                      // threads of a workgroup that walks several parts

// the walkers' tops together; where a row may be cut, draw_near_kernel has left the result
template <int NT>
__device__ __forceinline__ float draw_row_top(const DrawArgs& a, long long r, float* s_f, bool known)
{
    if (known) return a.tops[r];
    float top = -__builtin_inff();
    for (int w = threadIdx.x; w < a.walkers; w += NT) top = fmaxf(top, a.walk_top[r * a.walkers + w]);
    return draw_max<NT>(top, s_f);
}

// f(l, g) for a walker's share of the row's groups, every thread of a wave; four groups' loads in flight
template <int NT, typename T, typename F>
__device__ __forceinline__ void draw_walk(const DrawArgs& a, const Places<T>& row, F f)
{
    const int groups = row.groups();
    const int each = ((groups + a.walkers - 1) / a.walkers + 63) & ~63;
    const int g0 = (int)blockIdx.x * each, g1 = g0 + each < groups ? g0 + each : groups;
    for (int g = g0; g < g1; g += 4 * NT) {
        float l[4][4];
        row.load_many(g + (int)threadIdx.x, NT, g1, l);
#pragma unroll
        for (int q = 0; q < 4; q++)
            if (g + q * NT < g1) f(l[q], g + q * NT + (int)threadIdx.x);
    }
}

template <typename T>
__global__ __launch_bounds__(kDrawWalk) void draw_part_top_kernel(DrawArgs a)
{
    __shared__ float s_f[kDrawWalk / 64];
    const long long r = blockIdx.y;
    Places<T> row(a, r);
    float top = -__builtin_inff();
    draw_walk<kDrawWalk>(a, row, [&](const float (&l)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; j++) top = fmaxf(top, l[j]);
    });
    top = draw_max<kDrawWalk>(top, s_f);
    if (threadIdx.x == 0) {
        a.walk_top[r * a.walkers + blockIdx.x] = top;
        if (blockIdx.x == 0 && a.cuts) a.list_n[r] = 0;
    }
}

template <typename T>
__global__ __launch_bounds__(kDrawWalk) void draw_part_hist_kernel(DrawArgs a)
{
    __shared__ u64 bins[kDrawBins];
    __shared__ float s_f[kDrawWalk / 64];
    const long long r = blockIdx.y;
    const DrawRow set = draw_row(a, r);
    const bool by_k = set.k < a.V, by_p = set.p < 1.0;
    float top = draw_row_top<kDrawWalk>(a, r, s_f, false);
    if (!set.valid || top == -__builtin_inff() || (!by_k && !by_p)) return;
    for (int b = threadIdx.x; b < kDrawBins; b += kDrawWalk) bins[b] = 0;
    __syncthreads();
    Places<T> row(a, r);
    top = row.finite_top(top);
    const float units = (float)(set.inv_t * 0x1.71547652b82fep+0);
    draw_walk<kDrawWalk>(a, row, [&](const float (&l)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (l[j] == l[j]) draw_near_add(bins, l[j], top, set.scale, units);
    });
    __syncthreads();
    const long long at = (r * a.walkers + blockIdx.x) * kDrawBins;
    for (int b = threadIdx.x; b < kDrawBins; b += kDrawWalk) a.hist[at + b] = bins[b];
}

// 64 bins to a workgroup, its waves share the walkers out
__global__ __launch_bounds__(1024) void draw_sum_hist_kernel(DrawArgs a)
{
    __shared__ uint32_t s_n[16][64];
    __shared__ u64 s_m[16][64];
    const long long r = blockIdx.y;
    const DrawRow set = draw_row(a, r);
    if (!set.valid || (set.k >= a.V && !(set.p < 1.0))) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bin = blockIdx.x * 64 + lane;
    uint32_t n = 0; u64 m = 0;
#pragma unroll 8
    for (int w = wave; w < a.walkers; w += 16) {
        const u64 v = a.hist[(r * a.walkers + w) * kDrawBins + bin];
        n += draw_near_count(v); m += draw_near_mass(v);
    }
    s_n[wave][lane] = n; s_m[wave][lane] = m;
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < 16; w++) { n += s_n[w][lane]; m += s_m[w][lane]; }
        a.row_n[r * kDrawBins + bin] = n; a.row_m[r * kDrawBins + bin] = m;
    }
}

// one workgroup per row: its top, and the bracket from the walkers' histograms where they are few, else from their sum
__global__ __launch_bounds__(1024) void draw_near_kernel(DrawArgs a)
{
    constexpr int NT = 1024;
    __shared__ uint32_t count[kDrawBins];
    __shared__ u64 mass[kDrawBins];
    __shared__ DrawCut c;
    const long long r = blockIdx.x;
    const DrawRow set = draw_row(a, r);
    const bool by_k = set.k < a.V, by_p = set.p < 1.0;
    const float top = draw_row_top<NT>(a, r, c.wave_f, false);
    if (threadIdx.x == 0) a.tops[r] = top;
    if (!set.valid || (!by_k && !by_p)) return;
    for (int b = threadIdx.x; b < kDrawBins; b += NT) {
        uint32_t n = 0; u64 m = 0;
        if (a.walkers <= kDrawFewWalkers) {
#pragma unroll 4
            for (int w = 0; w < a.walkers; w++) {
                const u64 v = a.hist[(r * a.walkers + w) * kDrawBins + b];
                n += draw_near_count(v); m += draw_near_mass(v);
            }
        } else { n = a.row_n[r * kDrawBins + b]; m = a.row_m[r * kDrawBins + b]; }
        count[b] = n; mass[b] = m;
    }
    __syncthreads();
    draw_bracket<NT>(c, [&](int b) { return count[b]; }, [&](int b) { return mass[b]; }, set, a.V, by_k, by_p);
    if (threadIdx.x == 0) a.near[r] = c.near;
}

__device__ __forceinline__ bool draw_all_listed(const DrawNear& near, bool by_k) { return by_k && near.to_bk <= kDrawExact; }

template <typename T>
__global__ __launch_bounds__(kDrawWalk) void draw_part_pass_kernel(DrawArgs a)
{
    constexpr int kStash = 512, kWaves = kDrawWalk / 64;             // ranks that a wave holds back for one atomic on the row's list
    __shared__ u64 s_list[kWaves][kStash];
    __shared__ uint32_t s_held[kWaves + 1];
    __shared__ double s_2[kWaves][2];
    __shared__ float s_f[kWaves];
    const long long r = blockIdx.y;
    const DrawRow set = draw_row(a, r);
    const bool by_k = set.k < a.V, by_p = set.p < 1.0;
    float top = draw_row_top<kDrawWalk>(a, r, s_f, true);
    if (!set.valid || top == -__builtin_inff() || (!by_k && !by_p)) return;
    const DrawNear near = a.near[r];
    Places<T> row(a, r);
    top = row.finite_top(top);
    // a short list takes everything up to bin bk: the row ends in draw_floor_kernel then
    const bool listed = draw_all_listed(near, by_k);
    const int bk = near.bk, lo = listed ? 0 : by_p ? near.lo : bk, hi = listed ? bk : by_p ? near.hi : bk;
    const float lo_t = (float)lo, hi_t = (float)(hi + 1), bk_t = (float)(by_k ? bk : kDrawBins), front = fminf(lo_t, bk_t);
    const bool apart = by_k && (bk < lo || bk > hi);
    const int lane = threadIdx.x & 63;
    u64* stash = s_list[threadIdx.x >> 6];
    double above = 0.0, total = 0.0;
    int held = 0;                                                    // the same in every lane
    auto flush_to = [&](uint32_t at) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int q = lane; q < held; q += 64)
            if ((long long)at + q < a.list_most) a.list[r * a.list_most + at + q] = stash[q];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        held = 0;
    };
    auto flush = [&]() {
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&a.list_n[r], (uint32_t)held);
        flush_to((uint32_t)__builtin_amdgcn_readfirstlane((int)at));
    };
    auto pass = [&](auto kind) {
        draw_walk<kDrawWalk>(a, row, [&](const float (&l)[4], int g) {
            float t[4];
            bool in[4], some = false, sums = kind == kAll;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                t[j] = draw_depth(l[j], top, set.scale);
                in[j] = l[j] == l[j] && t[j] >= lo_t && t[j] < hi_t;
                if (apart) in[j] = in[j] || (l[j] == l[j] && t[j] >= bk_t && t[j] < bk_t + 1.0f);
                some |= in[j];
                sums |= t[j] < bk_t;
            }
            if (kind != kNone && __any(sums)) draw_group_sums<kind.value, false>(l, t, front, bk_t, top, set, above, total);
            if (__any(some)) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const u64 who = __ballot(in[j]);
                    if (in[j]) stash[held + __popcll(who & ((1ull << lane) - 1))] = draw_rank(l[j], 4 * g + j - row.off);
                    held += __popcll(who);
                }
                if (held > kStash - 256) flush();
            }
        });
    };
    if (listed || !by_p) pass(std::integral_constant<int, kNone>{});
    else if (by_k) pass(std::integral_constant<int, kUpto>{});
    else pass(std::integral_constant<int, kAll>{});
    // what is left, with one atomic for the workgroup: atomics on one address take some 10 ns each
    if (lane == 0) s_held[threadIdx.x >> 6] = (uint32_t)held;
    __syncthreads();
    uint32_t ahead = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) { if (w == (int)(threadIdx.x >> 6)) ahead = all; all += s_held[w]; }
    if (threadIdx.x == 0) s_held[kWaves] = all ? atomicAdd(&a.list_n[r], all) : 0;
    __syncthreads();
    flush_to(s_held[kWaves] + ahead);
    draw_sums<kDrawWalk>(above, total, s_2);
    if (threadIdx.x == 0) {
        a.sums[(r * a.walkers + blockIdx.x) * 2] = above;
        a.sums[(r * a.walkers + blockIdx.x) * 2 + 1] = total;
    }
}

// Draws that the one workgroup of a row with a short list makes itself (512 at a time); of more the whole card makes them.  One row of 265754, k = 161: 8192 draws 38 us by the workgroup, 40 by the card; 54914: 66, 40.
constexpr int64_t kDrawInFloor = 8192;
// one workgroup per row: the cuts among the list's tokens, of any number; -> a.floors
template <typename T>
__global__ __launch_bounds__(kDrawExact) void draw_floor_kernel(DrawArgs a)
{
    constexpr int NT = kDrawExact;
    __shared__ DrawHist hist;
    __shared__ union { DrawFine fine; DrawCand cand; } sh;
    __shared__ DrawCut c;
    const long long r = blockIdx.x;
    const int tid = threadIdx.x;
    // all loads first: each is a round trip through the caches
    const DrawRow set = draw_row(a, r);
    const DrawNear near = a.near[r];
    float top = a.tops[r];
    const long long n = a.list_n[r];
    const u64 first_rank = a.list[r * a.list_most + tid];            // list_most is 4096 at least
    const double first_u = tid < a.S ? draw_uniform(a, r * a.S + tid) : 0.0;
    double above = tid < a.walkers ? a.sums[(r * a.walkers + tid) * 2] : 0.0, total = tid < a.walkers ? a.sums[(r * a.walkers + tid) * 2 + 1] : 0.0;       // at most 512
    const bool by_k = set.k < a.V, by_p = set.p < 1.0;
    if (!set.valid || top == -__builtin_inff() || (!by_k && !by_p)) { if (tid == 0) a.floors[r] = 0; return; }
    Places<T> row(a, r);
    top = row.finite_top(top);
    if (tid == 0) c.near = near;
    draw_sums<NT>(above, total, c.wave_2);
    const u64* list = a.list + r * a.list_most;
    bool done = false;
    const bool all_listed = draw_all_listed(c.near, by_k);
    if (all_listed) {                                                // the row's first to_bk tokens, of which the first k count
        if (tid == 0) { c.near.lo = 0; c.near.hi = c.near.bk; }
        above = total = 0.0;
        __syncthreads();
    }
    if (n <= NT) {
        if (tid < n) sh.cand.rank[tid] = first_rank;
        if (tid == 0) c.slots = (uint32_t)n;
        __syncthreads();
        done = draw_decide<NT>(c, sh.cand, set, top, by_k, by_p, above, total, all_listed);
        if (all_listed && a.S <= kDrawInFloor) {                     // and its draws, from the kept ones in index order
            const u64 rank = tid < n ? sh.cand.rank[tid] : 0;
            const float l = draw_rank_logit(rank);
            const double lw = tid < n && rank >= c.floor_rank ? draw_weight(l, top, set.inv_t) : 0.0;
            const bool in = lw > 0.0 && lw >= set.min_p;
            const int i = draw_rank_index(rank);
            __syncthreads();
            if (tid == 0) c.slots = 0;
            __syncthreads();
            if (in) sh.cand.rank[atomicAdd(&c.slots, 1u)] = (u64)(0x7fffffff - i) << 32 | __builtin_bit_cast(uint32_t, l);
            __syncthreads();
            const int m = (int)c.slots;
            draw_rank_cand<NT>(sh.cand, m);
            const u64 mine = tid < m ? sh.cand.ranked[tid] : 0;
            const float ml = __builtin_bit_cast(float, (uint32_t)mine);
            double mass = 0.0;
            const double w = tid < m ? draw_weight(ml, top, set.inv_t) : 0.0, at = draw_before<NT, double>(w, c.wave_d, &mass) + w;
            double* upto = reinterpret_cast<double*>(sh.cand.rank);
            __syncthreads();
            if (tid < m) upto[tid] = at;
            __syncthreads();
            const double log_mass = draw_log(mass);
            for (long long s = tid; s < a.S; s += NT) {
                const double want = (s == tid ? first_u : draw_uniform(a, r * a.S + s)) * mass;
                const int lo = draw_place([&](int i) { return upto[i]; }, m, draw_power(m), want);
                const u64 v = sh.cand.ranked[lo];
                a.indices[r * a.S + s] = 0x7fffffff - (int)(v >> 32);
                if (a.logprobs) a.logprobs[r * a.S + s] = draw_logprob(__builtin_bit_cast(float, (uint32_t)v), top, set.inv_t, log_mass);
            }
            if (tid == 0) a.floors[r] = ~0ull;                       // done
            return;
        }
    } else if (n <= a.list_most) {
        auto each = [&](auto f) {
            for (long long i = tid; i < n; i += NT) { const u64 rank = list[i]; f(draw_rank_logit(rank), rank); }
        };
        const int bk = c.near.bk, lo = c.near.lo, hi = c.near.hi;
        u64 floor_rank = 0;
        __syncthreads();
        if (by_k) {
            if (tid == 0) { c.above_n = c.near.above_k; c.above_hi = 0; c.above_lo = 0; c.base = total; c.in_bin = (uint32_t)n; }
            __syncthreads();
            draw_resolve<NT>(c, sh.fine, sh.cand, each, top, set.inv_t, set.scale, bk, bk, 0, false, by_p, set.k, 0.0);
            floor_rank = c.floor_rank; total = c.mass;
            __syncthreads();
        }
        done = true;
        if (by_p) {
            const double want = set.p * total;
            if (lo == 0 || above < want) {
                if (tid == 0) { c.above_n = 0; c.above_hi = 0; c.above_lo = 0; c.base = above; c.in_bin = (uint32_t)n; }
                __syncthreads();
                draw_resolve<NT>(c, sh.fine, sh.cand, each, top, set.inv_t, set.scale, lo, hi, floor_rank, true, true, 0, want);
                done = hi == bk || c.mass >= want;                   // or else the bracket was too short
                if (tid == 0 && c.floor_rank < floor_rank) c.floor_rank = floor_rank;
                __syncthreads();
            } else done = false;
        }
    }
    u64 floor_rank = c.floor_rank;
    if (!done) {
        __syncthreads();
        floor_rank = draw_exact_floor<T, NT>(a, row, set, top, c, hist, sh.fine, sh.cand);
    }
    if (tid == 0) a.floors[r] = floor_rank;
}

// the masses of a part: inclusive sums behind every group, counted from the part's start
template <typename T>
__global__ __launch_bounds__(kDrawPart, 5) void draw_part_mass_kernel(DrawArgs a)
{
    __shared__ double s_d[kDrawPart / 64];
    __shared__ float s_f[kDrawPart / 64];
    __shared__ double span[4 * kDrawPart];
    const long long r = blockIdx.y;
    const int tid = threadIdx.x;
    const DrawRow set = draw_row(a, r);
    if (a.cuts && a.floors[r] == ~0ull) return;                      // the row has its draws already
    float top = draw_row_top<kDrawPart>(a, r, s_f, a.cuts);
    double carry = 0.0;
    if (set.valid && top > -__builtin_inff()) {
        Places<T> row(a, r);
        top = row.finite_top(top);
        const DrawFloor floor(a.cuts ? a.floors[r] : 0);
        const int groups = row.groups(), g0 = blockIdx.x * a.part;
        double* spans = a.spans + r * a.spans_row + g0;
        for (int b = 0; b < a.part && g0 + b < groups; b += 4 * kDrawPart) {
            float l[4][4];
            row.load_many(g0 + b + tid, kDrawPart, groups, l);
            __syncthreads();                                         // span[] of the round before has been read
#pragma unroll
            for (int q = 0; q < 4; q++) {
                double sum = 0.0;
#pragma unroll
                for (int j = 0; j < 4; j++) sum += draw_kept(l[q][j], 4 * (g0 + b + q * kDrawPart + tid) + j - row.off, floor, top, set);
                span[q * kDrawPart + tid] = sum;
                __builtin_amdgcn_sched_barrier(0);                   // one group's exps at a time, for five waves a SIMD (six spill, and gain nothing)
            }
            __syncthreads();
            double w[4], all;
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = span[4 * tid + q];
            w[1] += w[0]; w[2] += w[1]; w[3] += w[2];
            const double at = carry + draw_before<kDrawPart, double>(w[3], s_d, &all);
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (b + 4 * tid + q < groups - g0) spans[b + 4 * tid + q] = at + w[q];
            if ((tid & 3) == 3) a.lines[(r * a.spans_row + g0 + b) / 16 + tid / 4] = at + w[3];
            carry += all;
        }
    }
    if (tid == 0) a.part_mass[r * a.parts + blockIdx.x] = carry;
}

// Draws of a row in parts.  What bounds many of them is the chain of loads that wait for each other and the lines that these touch; so the sums behind every 1 / nodes of a
// part lie in LDS, down to 16 groups where they fit, the sums behind every 16 groups lie side by side, and a draw reads one line of each kind of sums and one of tokens.
// Measured: 1 M tokens and draws 36 us, 6 M tokens and 1 M draws 55 us (68 with the steps down to 16 groups in the sums behind each group); two draws of a thread side by
// side 3 and 10 us more, four 6 and 15: with 16 waves a CU the loads of one draw hide behind those of others, and the registers of more cost waves.
constexpr int kDrawMostParts = 2048;
constexpr int kDrawMostNodes = 16384;
constexpr int64_t kDrawManyDraws = 1 << 15;         // from here on the nodes' 128 KB are worth their loading (1 M tokens: 64 draws 20.7 us with them, 19.0 without; 32768: 25.6, 26.4)
constexpr int kDrawPickers = 1024;
template <typename T>
__global__ __launch_bounds__(kDrawPickers) void draw_part_pick_kernel(DrawArgs a)
{
    extern __shared__ double s_sum[];                                // masses in front of each part, then behind each node
    __shared__ double s_d[kDrawPickers / 64];
    __shared__ float s_f[kDrawPickers / 64];
    const long long r = blockIdx.y;
    const int tid = threadIdx.x;
    const DrawRow set = draw_row(a, r);
    if (a.cuts && a.floors[r] == ~0ull) return;
    Places<T> row(a, r);
    const float top = row.finite_top(draw_row_top<kDrawPickers>(a, r, s_f, a.cuts));
    double* s_part = s_sum;
    double* s_node = s_sum + a.parts;                                // a gap after every 32: steps of powers of two would meet in one bank
    const int part_log = __builtin_ctz(a.part), groups = row.groups(), step = a.part >> a.nodes_log;
    const double *spans = a.spans + r * a.spans_row, *lines = a.lines + r * a.spans_row / 16;       // lines: what stands behind every 16th group, side by side
    const int per = (a.parts + kDrawPickers - 1) / kDrawPickers;
    double sum = 0.0, total;
    for (int p = tid * per; p < (tid + 1) * per && p < a.parts; p++) sum += a.part_mass[r * a.parts + p];
    double at = draw_before<kDrawPickers, double>(sum, s_d, &total);
    for (int p = tid * per; p < (tid + 1) * per && p < a.parts; p++) { s_part[p] = at; at += a.part_mass[r * a.parts + p]; }
    __syncthreads();
    const int nodes = a.parts * a.nodes;
    for (int q0 = tid; q0 < nodes; q0 += 8 * kDrawPickers) {         // eight loads in flight: 16 k nodes one by one would be 16 trips
        double v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int q = q0 + j * kDrawPickers < nodes ? q0 + j * kDrawPickers : nodes - 1, last = (q + 1) * step - 1;       // the node's last group
            const bool whole = last < groups && ((q + 1) & (a.nodes - 1));
            const double* at = whole ? lines + last / 16 : a.part_mass + r * a.parts + (q >> a.nodes_log);
            v[j] = *at;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int q = q0 + j * kDrawPickers;
            if (q < nodes) s_node[q + (q >> 5)] = s_part[q >> a.nodes_log] + v[j];
        }
    }
    __syncthreads();
    const DrawFloor floor(a.cuts ? a.floors[r] : 0);
    if (!(total > 0.0)) {
        for (long long s = (long long)blockIdx.x * kDrawPickers + tid; s < a.S; s += (long long)gridDim.x * kDrawPickers) {
            a.indices[r * a.S + s] = -1;
            if (a.logprobs) a.logprobs[r * a.S + s] = -__builtin_inff();
        }
        return;
    }
    const int top_node = draw_power(nodes);
    const double log_total = draw_log(total);
    for (long long s = (long long)blockIdx.x * kDrawPickers + tid; s < a.S; s += (long long)gridDim.x * kDrawPickers) {
        const double want = draw_uniform(a, r * a.S + s) * total;
        int n = 0;
        for (int by = top_node; by; by >>= 1) {                      // as draw_place
            const int i = n + by - 1, j = i < nodes ? i : nodes - 1;
            n = i < nodes - 1 && s_node[j + (j >> 5)] <= want ? n + by : n;
        }
        int lo = n * step;
        const int hi = lo + step < groups ? lo + step - 1 : groups - 1;
        const bool beyond = lo > hi;                                 // rounding beyond the last node with tokens
        lo = beyond ? hi : lo;
        const double base = s_part[lo >> part_log];
        double run = (lo & (a.part - 1)) == 0 ? base : beyond ? base + spans[lo - 1] : s_node[n - 1 + ((n - 1) >> 5)];        // in front of group lo
        for (int by = step >> 1; by >= 16; by >>= 1) {
            const int i = lo + by - 1;
            const double v = base + lines[(i < hi ? i : hi) >> 4];
            const bool on = i < hi && v <= want;
            lo = on ? lo + by : lo;
            run = on ? v : run;
        }
        // the line of 16 sums that is left, in two steps of four ways: each way's load would be one more trip
#pragma unroll
        for (int by = 4; by > 0; by -= 3) {
            const int from = lo;
            double v[3];
#pragma unroll
            for (int j = 0; j < 3; j++) { const int i = from + (j + 1) * by - 1; v[j] = base + spans[i < hi ? i : hi]; }
#pragma unroll
            for (int j = 0; j < 3; j++) {
                const bool on = from + (j + 1) * by - 1 < hi && v[j] <= want;
                lo = on ? from + (j + 1) * by : lo;
                run = on ? v[j] : run;
            }
        }
        float l[4], at_l = 0.0f;
        row.load(lo, groups, l);
        int index = draw_in_group(row, lo, l, run, want, floor, top, set, at_l);
        for (int q = lo; index < 0 && q > 0;) {                      // nothing there: rounding; the last one in front with weight
            q = draw_back([&](int i) { return s_part[i >> part_log] + spans[i]; }, q);
            row.load(q, groups, l);
            index = draw_in_group(row, q, l, s_part[q >> part_log] + (q & (a.part - 1) ? spans[q - 1] : 0.0), want, floor, top, set, at_l);
        }
        a.indices[r * a.S + s] = index;
        if (a.logprobs) a.logprobs[r * a.S + s] = draw_logprob(at_l, top, set.inv_t, log_total);
    }
}

// ---- short rows: W lanes to a row, E tokens to a lane ----------------------------------------------------------------------------
template <int W>
__device__ __forceinline__ uint32_t draw_votes(bool b, int sub)       // lanes of the row that say yes
{
    const u64 v = __ballot(b);
    return W == 64 ? __popcll(v) : __popcll((v >> (sub * W)) & ((1ull << (W & 63)) - 1));
}
// all W lanes of a row get op over them: within 16 lanes by DPP (mirrors reach the other half once a half is equal)
template <int W, typename T, typename Op>
__device__ __forceinline__ T draw_lanes_all(T v, Op op)
{
    if (W >= 2) v = op(v, draw_dpp<0xB1, 0xf>(v));
    if (W >= 4) v = op(v, draw_dpp<0x4E, 0xf>(v));
    if (W >= 8) v = op(v, draw_dpp<0x141, 0xf>(v));
    if (W >= 16) v = op(v, draw_dpp<0x140, 0xf>(v));
    if (W >= 32) v = op(v, __shfl_xor(v, 16, 64));
    if (W >= 64) v = op(v, __shfl_xor(v, 32, 64));
    return v;
}
template <int W>
__device__ __forceinline__ double draw_lanes_sum(double v) { return draw_lanes_all<W>(v, [](double x, double y) { return x + y; }); }
// inclusive sums over the row's lanes
template <int W, typename T>
__device__ __forceinline__ T draw_lanes_scan(T v)
{
    const int at = threadIdx.x % W;
    if (W >= 2) { const T o = draw_dpp<0x111, 0xf>(v); v += at >= 1 ? o : (T)0; }
    if (W >= 4) { const T o = draw_dpp<0x112, 0xf>(v); v += at >= 2 ? o : (T)0; }
    if (W >= 8) { const T o = draw_dpp<0x114, 0xf>(v); v += at >= 4 ? o : (T)0; }
    if (W >= 16) { const T o = draw_dpp<0x118, 0xf>(v); v += at >= 8 ? o : (T)0; }
    // DPP stays within 16 lanes: from there on the last lane of the lower half is added to the upper one
    if (W >= 32) { const T o = __shfl(v, 15, 32); v += (at & 16) ? o : (T)0; }
    if (W >= 64) { const T o = __shfl(v, 31, 64); v += at >= 32 ? o : (T)0; }
    return v;
}

template <typename T, int W, int E>
__global__ __launch_bounds__(kBlock) void draw_short_kernel(DrawArgs a)
{
    constexpr int kRows = 64 / W;
    __shared__ double s_mass[kBlock / 64][64 * E];
    __shared__ float s_l[kBlock / 64][64 * E];
    __shared__ double s_total[kBlock / 64][kRows], s_log[kBlock / 64][kRows], s_inv[kBlock / 64][kRows];
    __shared__ float s_top[kBlock / 64][kRows];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / W, j0 = (lane % W) * E;
    const long long r0 = (block_of() * (kBlock / 64) + wave) * kRows, r = r0 + sub;
    const int V = (int)a.V;
    const bool on = r < a.R;
    const DrawRow set = draw_row(a, on ? r : a.R - 1);
    const T* row = (const T*)a.logits + (on ? r : a.R - 1) * a.row_stride;
    float l[E];
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        if (j0 + e + 4 <= V && ((uintptr_t)(row + j0 + e) & (4 * sizeof(T) - 1)) == 0) {
            const Four<T> f = *(const Four<T>*)(row + j0 + e);
#pragma unroll
            for (int j = 0; j < 4; j++) l[e + j] = draw_logit(f.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) l[e + j] = j0 + e + j < V ? draw_logit(row[j0 + e + j]) : __builtin_nanf("");
        }
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < E; e++) top = fmaxf(top, l[e]);
    top = draw_lanes_all<W>(top, [](float x, float y) { return fmaxf(x, y); });
    const bool live = on && set.valid && top > -__builtin_inff();
    if (__any(top == __builtin_inff())) {                            // as Places has it
        const bool infinite = top == __builtin_inff();
#pragma unroll
        for (int e = 0; e < E; e++) l[e] = !infinite || l[e] != l[e] ? l[e] : l[e] == __builtin_inff() ? 0.0f : -__builtin_inff();
        top = infinite ? 0.0f : top;
    }
    double w[E];
    uint32_t key[E];                                                 // 0: not a token, or cut
    const bool cuts = __any(live && (set.k < a.V || set.p < 1.0));
#pragma unroll
    for (int e = 0; e < E; e++) {
        w[e] = draw_weight(l[e], top, set.inv_t);                    // 0 outside the row
        key[e] = 1u;
        if (cuts) key[e] = l[e] == l[e] ? draw_key(l[e]) : 0u;
    }
    // A cut at the highest key t for which the tokens of key >= t reach k, or `want`: found bit by bit; of the ones at t the first few in index order.
#pragma unroll 1
    for (int cut = 0; cuts && cut < 2; cut++) {
        const bool mine = live && (cut == 0 ? set.k < a.V : set.p < 1.0);
        if (!__any(mine)) continue;
        double want = 0.0;
        if (cut) {
            double sum = 0.0;
#pragma unroll
            for (int e = 0; e < E; e++) sum += key[e] ? w[e] : 0.0;
            want = set.p * draw_lanes_sum<W>(sum);
        }
        uint32_t t = 0;
#pragma unroll 1
        for (int b = 31; b >= 0; b--) {
            const uint32_t up = t | 1u << b;
            bool reached;
            if (cut == 0) {
                uint32_t n = 0;
#pragma unroll
                for (int e = 0; e < E; e++) n += draw_votes<W>(key[e] >= up, sub);
                reached = (long long)n >= set.k;
            } else {
                double sum = 0.0;
#pragma unroll
                for (int e = 0; e < E; e++) sum += key[e] >= up ? w[e] : 0.0;
                reached = draw_lanes_sum<W>(sum) >= want;
            }
            if (reached) t = up;
        }
        uint32_t ties = 0, above = 0, before = 0;
        double mass = 0.0, tie_w = 0.0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            above += draw_votes<W>(key[e] > t, sub);
            mass += key[e] > t ? w[e] : 0.0;
            if (key[e] == t) { ties++; tie_w = w[e]; }
        }
        mass = draw_lanes_sum<W>(mass);
        // ties in the lanes before this one, in all of them, and the weight that they share
        const uint32_t incl = draw_lanes_scan<W>(ties);
        before = incl - ties;
        const uint32_t all = __shfl(incl, W - 1, W);
        tie_w = draw_lanes_all<W>(tie_w, [](double x, double y) { return fmax(x, y); });
        double m = cut == 0 ? (double)set.k - (double)above : tie_w > 0.0 ? ceil((want - mass) / tie_w) : (double)all;
        const uint32_t kept = m < 1.0 ? 1u : m < (double)all ? (uint32_t)m : all;
        if (mine)
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (key[e] == t && t) { if (before >= kept) key[e] = 0; before++; }
                else if (key[e] < t) key[e] = 0;
            }
    }
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (!key[e] || w[e] < set.min_p) w[e] = 0.0;
        sum += w[e];
    }
    const double incl = draw_lanes_scan<W>(sum), up = draw_wave_shift(incl), total = __shfl(incl, W - 1, W);
    double run = lane % W ? up : 0.0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        run += w[e];
        // a token without weight is marked by its sign: sums of neighbouring lanes may differ by a rounding, and it is never drawn
        s_mass[wave][lane * E + e] = w[e] > 0.0 ? run : -run;
        s_l[wave][lane * E + e] = l[e];
    }
    if (lane % W == 0) { s_total[wave][sub] = live ? total : -1.0; s_log[wave][sub] = draw_log(total); s_inv[wave][sub] = set.inv_t; s_top[wave][sub] = top; }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");           // LDS of this wave's own lanes
    __builtin_amdgcn_wave_barrier();
    const int rows = a.R - r0 < kRows ? (int)(a.R - r0) : kRows;
    if (rows <= 0) return;
    const float per_row = __builtin_amdgcn_rcpf((float)a.S);
    const long long first = (long long)blockIdx.z * a.share, behind = (long long)rows * a.S - first < a.share ? (long long)rows * a.S : first + a.share;
    for (long long q = first + lane; q < behind; q += 64) {
        int y = 0;                                                   // q / S: a 64-bit division would cost as much as four exps
        if (kRows > 1) {
            if (a.S < (1 << 18)) {
                y = (int)((float)(int)q * per_row);
                const int left = (int)q - y * (int)a.S;
                y += left < 0 ? -1 : left >= (int)a.S ? 1 : 0;
            } else y = (int)(q / a.S);
        }
        const double all = s_total[wave][y];
        const double* mass = &s_mass[wave][y * W * E];
        long long index = -1;
        float lp = -__builtin_inff();
        if (all > 0.0) {
            const double want = draw_uniform(a, r0 * a.S + q) * all;
            int i = 0;                                               // places behind the row hold its total
#pragma unroll
            for (int step = W * E / 2; step; step >>= 1) i += fabs(mass[i + step - 1]) <= want ? step : 0;
            while (i > 0 && !(mass[i] > 0.0)) i--;
            while (!(mass[i] > 0.0) && i < V - 1) i++;
            index = i;
            lp = draw_logprob(s_l[wave][y * W * E + i], s_top[wave][y], s_inv[wave][y], s_log[wave][y]);
        }
        a.indices[r0 * a.S + q] = index;
        if (a.logprobs) a.logprobs[r0 * a.S + q] = lp;
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
    if (s->V > GSX_DRAW_MAX_V || s->R > 0x7fffffffll || (s->R > GSX_DRAW_MAX_LONG_ROWS && s->V > (int64_t)kDrawWaveTiles * 256 - 4) || s->S > (1ll << 38) || (s->R && s->S > (1ll << 38) / s->R)) return GSX_E_RANGE;
    return GSX_OK;
}

struct DrawLayout {
    enum Way { kShort, kRow, kRowSpans, kParts } way;
    long long spans_row, part, list_most; int parts, nodes, walkers, cuts;
    size_t spans, lines, total, floors, tops, left, walk_top, part_mass, hist, row_n, row_m, near, sums, list, list_n, bytes;
};

// Which way, and its workspace.
static DrawLayout draw_layout(const gsx_draw* s)
{
    DrawLayout l = {};
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += align_up(bytes); return here; };
    const size_t R = (size_t)s->R;
    l.cuts = s->top_ks || s->top_ps || s->temperatures || s->temperature == 0.0f || (s->top_k > 0 && s->top_k < s->V) || s->top_p < 1.0f;
    if (s->V <= kDrawShort) l.way = DrawLayout::kShort;
    else if (s->V > kDrawLong && (s->R <= kDrawFewRows || s->V > (int64_t)kDrawWaveTiles * 256 - 4)) l.way = DrawLayout::kParts;
    else if (s->S <= (s->R <= kDrawCus ? kDrawInRow : kDrawInRowOfMany) && s->V <= (int64_t)kDrawWaveTiles * 256 - 4) l.way = DrawLayout::kRow;
    else l.way = DrawLayout::kRowSpans;
    if (l.way != DrawLayout::kShort) { l.tops = take(R * 4); l.left = take(R * 4); }       // left: one launch's word to the next
    if (l.way == DrawLayout::kRowSpans) {
        l.spans_row = (s->V + 3 + 3) / 4;
        l.spans = take(R * (size_t)l.spans_row * 8);
        l.total = take(R * 8);
        l.floors = take(R * 8);
    }
    if (l.way == DrawLayout::kParts) {
        const int64_t groups = (s->V + 3 + 3) / 4;
        l.part = 4 * kDrawPart;
        while (ceil_div(groups, l.part) > kDrawMostParts) l.part *= 2;
        l.parts = (int)ceil_div(groups, l.part);
        l.spans_row = (int64_t)l.parts * l.part;
        l.nodes = 1;
        if (s->S >= kDrawManyDraws)
            while (l.nodes < l.part / 16 && (int64_t)l.parts * l.nodes * 2 <= kDrawMostNodes) l.nodes *= 2;
        l.walkers = (int)(512 / s->R > 1 ? 512 / s->R : 1);
        if (l.walkers < ceil_div(s->V, kDrawMostInHist / 2)) l.walkers = (int)ceil_div(s->V, kDrawMostInHist / 2);
        if (l.walkers > l.parts) l.walkers = l.parts;
        l.spans = take(R * (size_t)l.spans_row * 8);
        l.lines = take(R * (size_t)l.spans_row / 16 * 8);
        l.floors = take(R * 8);
        l.walk_top = take(R * l.walkers * 4);
        l.part_mass = take(R * l.parts * 8);
        if (l.cuts) {
            l.hist = take(R * l.walkers * kDrawBins * 8);
            if (l.walkers > kDrawFewWalkers) { l.row_n = take(R * kDrawBins * 4); l.row_m = take(R * kDrawBins * 8); }
            l.near = take(R * sizeof(DrawNear));
            l.sums = take(R * l.walkers * 16);
            // 2^24 / R tokens of each row, 4096 at least (131072 at the 128 rows up to which ordinary lengths come here; from 4096 rows on, all of more than 524284
            // tokens, the 4096): a longer list is not kept, and one workgroup finds that row's cuts from the row itself
            int64_t most = (1ll << 24) / s->R;
            if (most < 4096) most = 4096;
            l.list_most = s->V < most ? s->V : most;
            l.list = take(R * (size_t)l.list_most * 8);
            l.list_n = take(R * 4);
        }
    }
    l.bytes = at ? at : 256;
    return l;
}

// A wave makes all draws of its rows while there are waves enough, or few draws; else several take shares of them, each with the rows' cuts and masses of its own.
// us a call, one input repeated, by one wave and in shares: 1 x 300, 1024 draws 14.7, 15.5; 2048: 25, 15.5; 1 M: 12384, 19; 1000 x 30, 1024 draws 86, 15.
constexpr int64_t kDrawShare = 1024, kDrawShareWaves = 4096;
template <typename T, int W, int E>
static void draw_short(const DrawArgs& a, hipStream_t stream)
{
    const int64_t rows = 64 / W, waves = ceil_div(a.R, rows), draws = (a.R < rows ? a.R : rows) * a.S;
    int64_t shares = ceil_div(draws, kDrawShare) < kDrawShareWaves / waves ? ceil_div(draws, kDrawShare) : kDrawShareWaves / waves;
    if (shares < 1) shares = 1;
    DrawArgs b = a;
    b.share = ceil_div(ceil_div(draws, shares), 64) * 64;
    dim3 grid = grid_of(ceil_div(a.R, (kBlock / 64) * rows));
    grid.z = (unsigned)ceil_div(draws, b.share);
    draw_short_kernel<T, W, E><<<grid, dim3(kBlock), 0, stream>>>(b);
}

template <typename T>
static int draw_run(const DrawArgs& a, const DrawLayout& l, hipStream_t stream)
{
    if (a.V <= kDrawShort) {
        if (a.V <= 8) draw_short<T, 2, 4>(a, stream);
        else if (a.V <= 16) draw_short<T, 4, 4>(a, stream);
        else if (a.V <= 32) draw_short<T, 8, 4>(a, stream);
        else if (a.V <= 64) draw_short<T, 16, 4>(a, stream);
        else if (a.V <= 128) draw_short<T, 32, 4>(a, stream);
        else if (a.V <= 256) draw_short<T, 64, 4>(a, stream);
        else draw_short<T, 64, 8>(a, stream);
        GSX_LAUNCH_CHECK();
        return GSX_OK;
    }
    if (l.way == DrawLayout::kParts) {
        const dim3 parts((unsigned)l.parts, (unsigned)a.R), walkers((unsigned)l.walkers, (unsigned)a.R);
        draw_part_top_kernel<T><<<walkers, dim3(kDrawWalk), 0, stream>>>(a);
        if (l.cuts) {
            draw_part_hist_kernel<T><<<walkers, dim3(kDrawWalk), 0, stream>>>(a);
            if (l.walkers > kDrawFewWalkers) draw_sum_hist_kernel<<<dim3(kDrawBins / 64, (unsigned)a.R), dim3(1024), 0, stream>>>(a);
            draw_near_kernel<<<dim3((unsigned)a.R), dim3(1024), 0, stream>>>(a);
            draw_part_pass_kernel<T><<<walkers, dim3(kDrawWalk), 0, stream>>>(a);
            draw_floor_kernel<T><<<dim3((unsigned)a.R), dim3(kDrawExact), 0, stream>>>(a);
        }
        draw_part_mass_kernel<T><<<parts, dim3(kDrawPart), 0, stream>>>(a);
        const int64_t picks = ceil_div(a.S, kDrawPickers);
        const size_t lds = ((size_t)l.parts * l.nodes + l.parts * l.nodes / 32 + 1 + l.parts) * 8;
        GSX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(draw_part_pick_kernel<T>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    (kDrawMostNodes + kDrawMostNodes / 32 + 1 + kDrawMostParts) * 8));
        draw_part_pick_kernel<T><<<dim3((unsigned)(picks < 256 ? picks : 256), (unsigned)a.R), dim3(kDrawPickers), lds, stream>>>(a);
        GSX_LAUNCH_CHECK();
        return GSX_OK;
    }
    const dim3 grid = grid_of(a.R);
    const bool small = a.V <= (a.R <= kDrawCus ? kDrawSmall : kDrawSmallOfMany);
    if (l.way == DrawLayout::kRow) {
        if (small) draw_row_kernel<T, kDrawExact, true, true><<<grid, dim3(kDrawExact), 0, stream>>>(a);
        else draw_row_kernel<T, 1024, true, false><<<grid, dim3(1024), 0, stream>>>(a);
        if (!small && l.cuts) draw_exact_kernel<T, true><<<grid, dim3(kDrawExact), 0, stream>>>(a);
    } else {
        if (small) draw_row_kernel<T, kDrawExact, false, true><<<grid, dim3(kDrawExact), 0, stream>>>(a);
        else draw_row_kernel<T, 1024, false, false><<<grid, dim3(1024), 0, stream>>>(a);
        if (!small && l.cuts) draw_exact_kernel<T, false><<<grid, dim3(kDrawExact), 0, stream>>>(a);
        GSX_LAUNCH_CHECK();
        const int64_t n = a.R * a.S;
        draw_pick_kernel<T><<<grid_of(ceil_div(n, kBlock)), dim3(kBlock), 0, stream>>>(a, n);
    }
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

}  // namespace gsx

using namespace gsx;

GSX_API size_t gsx_draw_workspace_bytes(const gsx_draw* s)
{
    if (draw_check(s) != GSX_OK) return 0;
    return s->R == 0 || s->S == 0 ? 256 : draw_layout(s).bytes;              // nothing to draw: no layout, which shares the card out over the rows
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
    a.logits = s->logits; a.row_stride = s->row_stride; a.R = s->R; a.V = s->V; a.S = s->S;
    a.uniforms = s->uniforms; a.uniforms_f64 = s->uniforms_f64 != 0;
    a.temperature = s->temperature; a.top_p = s->top_p; a.min_p = s->min_p; a.top_k = s->top_k;
    a.inv_t = s->temperature > 0.0f ? 1.0 / (double)s->temperature : 1.0;
    a.temperatures = s->temperatures; a.top_ps = s->top_ps; a.min_ps = s->min_ps; a.top_ks = s->top_ks;
    a.indices = (long long*)s->indices; a.logprobs = s->logprobs;
    a.spans_row = l.spans_row;
    a.part = (int)l.part; a.parts = l.parts; a.nodes = l.nodes; a.nodes_log = __builtin_ctz(l.nodes ? l.nodes : 1); a.lines = (double*)(ws + l.lines); a.walkers = l.walkers; a.cuts = l.cuts; a.list_most = l.list_most;
    a.walk_top = (float*)(ws + l.walk_top); a.part_mass = (double*)(ws + l.part_mass);
    a.hist = (u64*)(ws + l.hist); a.row_n = (uint32_t*)(ws + l.row_n); a.row_m = (u64*)(ws + l.row_m); a.near = (DrawNear*)(ws + l.near);
    a.sums = (double*)(ws + l.sums); a.list = (u64*)(ws + l.list); a.list_n = (uint32_t*)(ws + l.list_n);
    a.spans = (double*)(ws + l.spans); a.total = (double*)(ws + l.total); a.floors = (u64*)(ws + l.floors); a.tops = (float*)(ws + l.tops); a.left = (uint32_t*)(ws + l.left);
    switch (s->dtype) {
    case GSX_F32: return draw_run<float>(a, l, (hipStream_t)stream);
    case GSX_BF16: return draw_run<__bf16>(a, l, (hipStream_t)stream);
    default: return draw_run<_Float16>(a, l, (hipStream_t)stream);
    }
}
