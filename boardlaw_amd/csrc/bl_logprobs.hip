// bl_logprobs.hip -- log probabilities of given moves, entropy and the best alternatives of masked policy rows, and their gradient.
//
// With m = max_j x_j over a row's valid entries, d_j = x_j - m, c = #{j : d_j = 0}, r = sum_{d_j < 0} e^{d_j}, t = sum e^{d_j} d_j:
//     log s = log1p(r + c - 1),   logp_j = d_j - log s,   H = log s - t / (c + r).
// Counting the maxima apart from the sum of the rest keeps log s exact to a rounding of r where one move holds nearly all the mass
// (1 + r would round r away), and two parts of a row join by (c, r, t) -> e^{m1 - m} (c + r), ... as one sum.
//     dx_j = g_a [j = a] + sum_i g_i [j = top_i] - p_j (g_a + sum_i g_i + g_H (logp_j + H)).
// An invalid entry and a logit of -inf are the same thing: probability 0, never an alternative, gradient 0.
//
// One pass over the logits each way.  4096 x 32000 bf16: sums alone 67 us (262 MB at 3.9 TB/s, the VALU busy throughout: 18 instructions per
// entry by the counters, half of them the sums' own, most others the join of a new maximum), with 4 alternatives 100 us (23 per entry), the
// gradient 94 us (524 MB, 5.6 TB/s).  32768 x 81 f16 with masks: 7.5 us and 6.5 us, 4.5 times the bytes' time: instructions per row and the launch.
#include "bl_train.h"

#pragma clang fp contract(off)

using namespace bltrain;

namespace {

constexpr int SHORT = 1024;                 // rows up to here stay in a wave's registers
constexpr int SEGMENT = 4096;               // shortest part of a long row that is worth a workgroup of its own
constexpr long ONE_WAVE = 2048;             // long rows from which on a wave takes one
constexpr long SHARED_WAVE = 4096;          // short rows from which on several share a wave also beyond 256 entries (32768 x 361 f16: k 0 20 -> 10 us,
                                            // k 20 95 -> 52; but 1024 x 361, k 20 8.4 -> 11.7: a wave's own chain is longer)

struct Rows {
    const void* raw; long raw_stride;       // elements
    const uint8_t* valid; long valid_stride;
    const long long* actions;
    long R; int A, k;
    float* logp; float* entropy; long long* top; float* top_logp; float* stats;
    int S; char* parts;                     // parts of a long row, and what they leave for the join
};

struct Grads {
    const void* raw; long raw_stride;
    const uint8_t* valid; long valid_stride;
    const long long* actions; const long long* top; const float* stats; const float* entropy;
    const float* g_logp; const float* g_entropy; const float* g_top;
    long R; int A, k;
    void* d_raw;
    int S;
};

// order-preserving code of a value: NaN above everything, -0 = +0, 0 for an entry that is no alternative
__device__ __forceinline__ unsigned code(float x) {
    const unsigned b = __builtin_bit_cast(unsigned, x + 0.f);
    const unsigned u = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return x == -INFINITY ? 0u : (x != x ? 0xffffffffu : u);
}
__device__ __forceinline__ float value_of(unsigned u) {
    const unsigned b = (u & 0x80000000u) ? (u & 0x7fffffffu) : ~u;
    return u == 0xffffffffu ? NAN : __builtin_bit_cast(float, b);
}

// a row's statistics from its sums; `empty`: nothing valid in it
struct Stat { float m, logs, H; bool empty; };
__device__ __forceinline__ Stat finish(float m, float c, float r, float t) {
    Stat s;
    s.empty = m == -INFINITY && r == r;     // (only NaN in the row: r is NaN)
    const float logs = log1pf(r + (c - 1.f));
    s.logs = s.empty ? 0.f : (m == INFINITY ? NAN : logs);
    s.H = s.empty ? 0.f : s.logs - t / (c + r);
    s.m = s.empty ? 0.f : m;
    return s;
}
__device__ __forceinline__ float given_logp(const Stat& s, float xa, long long a, int A) {
    if (a < 0) return 0.f;
    if (a >= A) return NAN;
    return xa == -INFINITY && s.logs == s.logs ? -INFINITY : (xa - s.m) - s.logs;
}

// m: the maximum so far (-inf: nothing yet), c entries equal to it, r and t over the others
struct Part { float m, c, r, t; };
// N more entries into a lane's sums, p.m their maximum already.  An entry costs one exponential and eight other instructions: -inf needs no test, because
// e^-inf = 0 meets a clamped d (the reference is finite unless it is +inf), and NaN comes through both sums
template <int N> __device__ __forceinline__ void eat(Part& p, const float (&x)[N]) {
    const float ref = fmaxf(p.m, -3.402823466e38f);
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float d = x[i] - ref;
        const bool is = x[i] == ref;
        const float e = is ? 0.f : exp_neg(d);
        c += is; p.r += e; p.t = fmaf(e, fmaxf(d, -3e38f), p.t);
    }
    p.c += (float)c;
}
template <int N> __device__ __forceinline__ float max_of(const float (&x)[N]) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; i++) m = fmaxf(m, x[i]);
    return m;
}

// ---- short rows: G lanes hold a row, N entries each -----------------------------------------------------------------------------
// Entry j of the row is with lane j % G.  Loads are coalesced whatever the rows' alignment; everything else is in registers, the
// reductions are DPP.  What bounds it is instructions per row, not bytes, so up to 256 entries four rows share a wave, and where there are many
// rows four up to 512 and two up to 1024.
template <typename T, int G, int N>
__global__ void __launch_bounds__(256) logprobs_rows_kernel(Rows q) {
    const int gl = threadIdx.x & (G - 1);
    const long at = ((long)blockIdx.x * 256 + threadIdx.x) / G;
    const bool live = at < q.R;
    const long row = live ? at : q.R - 1;
    const T* x0 = (const T*)q.raw + row * q.raw_stride;
    const long long a = q.actions ? q.actions[row] : -1;
    float x[N];
#pragma unroll
    for (int i = 0; i < N; i++) { const int j = gl + G * i; x[i] = (float)x0[j < q.A ? j : q.A - 1]; }
    if (q.valid) {
        const uint8_t* v0 = q.valid + row * q.valid_stride;
        uint8_t v[N];
#pragma unroll
        for (int i = 0; i < N; i++) { const int j = gl + G * i; v[i] = v0[j < q.A ? j : q.A - 1]; }
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = v[i] ? x[i] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = gl + G * i < q.A ? x[i] : -INFINITY;

    Part p = {reduce<G, Max>(max_of(x)), 0.f, 0.f, 0.f};
    eat(p, x);
    float xa = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; i++) xa = (gl + G * i == a) ? x[i] : xa;
    const Stat s = finish(p.m, reduce<G, Sum>(p.c), reduce<G, Sum>(p.r), reduce<G, Sum>(p.t));
    if (q.logp) xa = reduce<G, Max>(xa);
    if (live && gl == 0) {
        if (q.logp) q.logp[row] = given_logp(s, xa, a, q.A);
        q.entropy[row] = s.H;
        if (q.stats) { q.stats[2 * row] = s.m; q.stats[2 * row + 1] = s.logs; }
    }
    if (q.k == 0) return;
    unsigned key[N];
#pragma unroll
    for (int i = 0; i < N; i++) key[i] = code(x[i]);
    unsigned mine = 0; int minej = -1;
    for (int n = 0; n < q.k; n++) {
        unsigned b = 0; int bj = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < N; i++) if (key[i] > b) { b = key[i]; bj = gl + G * i; }
        const unsigned best = reduce_max_u<G>(b);
        // the lowest index among the lanes that hold the best value: the largest of its complements
        const int j = (int)~reduce_max_u<G>(b == best && best ? ~(unsigned)bj : 0u);
#pragma unroll
        for (int i = 0; i < N; i++) key[i] = (gl + G * i == j) ? 0u : key[i];
        if ((n & (G - 1)) == gl) { mine = best; minej = best ? j : -1; }
        if (((n + 1) & (G - 1)) == 0 || n + 1 == q.k) {
            const int o = (n & ~(G - 1)) + gl;
            if (live && o <= n) {
                q.top[row * q.k + o] = minej;
                q.top_logp[row * q.k + o] = mine ? (value_of(mine) - s.m) - s.logs : -INFINITY;
            }
        }
    }
}

template <typename T, int G, int N>
__global__ void __launch_bounds__(256) logprobs_rows_grad_kernel(Grads q) {
    const int gl = threadIdx.x & (G - 1);
    const long at = ((long)blockIdx.x * 256 + threadIdx.x) / G;
    const bool live = at < q.R;
    const long row = live ? at : q.R - 1;
    const T* x0 = (const T*)q.raw + row * q.raw_stride;
    float x[N];
#pragma unroll
    for (int i = 0; i < N; i++) { const int j = gl + G * i; x[i] = (float)x0[j < q.A ? j : q.A - 1]; }
    if (q.valid) {
        const uint8_t* v0 = q.valid + row * q.valid_stride;
        uint8_t v[N];
#pragma unroll
        for (int i = 0; i < N; i++) { const int j = gl + G * i; v[i] = v0[j < q.A ? j : q.A - 1]; }
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = v[i] ? x[i] : -INFINITY;
    }
    const long long a = q.actions ? q.actions[row] : -1;
    const float m = q.stats[2 * row], logs = q.stats[2 * row + 1], H = q.entropy[row];
    const float gH = q.g_entropy ? q.g_entropy[row] : 0.f;
    const float ga = q.g_logp && a >= 0 ? (a < q.A ? q.g_logp[row] : NAN) : 0.f;
    float total = ga;
    if (q.g_top) {
        float own = 0.f;
        for (int n = gl; n < q.k; n += G) own += q.top[row * q.k + n] >= 0 ? q.g_top[row * q.k + n] : 0.f;
        total += reduce<G, Sum>(own);
    }
    T* d0 = (T*)q.d_raw + row * q.A;
    float o[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int j = gl + G * i;
        const float lp = (x[i] - m) - logs, p = exp_neg(lp);
        const float w = total + gH * ((lp < -3e38f ? -3e38f : lp) + H);
        const float g = (j == a ? ga : 0.f) - (p == 0.f ? 0.f : p * w);
        o[i] = x[i] == -INFINITY ? 0.f : g;
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < N; i++) { const int j = gl + G * i; if (j < q.A) d0[j] = (T)o[i]; }
    if (q.g_top) for (int n = gl; n < q.k; n += G) {           // the alternatives' own terms: a lane's second store follows its group's first
        const long long j = q.top[row * q.k + n];
        if (j < 0) continue;
        const float lp = ((float)x0[j] - m) - logs, p = exp_neg(lp);
        const float w = total + gH * ((lp < -3e38f ? -3e38f : lp) + H);
        d0[j] = (T)((j == a ? ga : 0.f) + q.g_top[row * q.k + n] - (p == 0.f ? 0.f : p * w));
    }
}

// ---- long rows: a workgroup takes a part of a row --------------------------------------------------------------------------------
typedef unsigned long long u64;
// (value, index) as one number: larger is better, ties go to the lower index, 0 is nothing
__device__ __forceinline__ u64 pack(float x, int j) { const unsigned u = code(x); return u ? ((u64)u << 32 | (unsigned)~j) : 0ull; }
__device__ __forceinline__ u64 lane_u64(u64 v, int lane) { return (u64)lane_u((unsigned)(v >> 32), lane) << 32 | lane_u((unsigned)v, lane); }

// the best `k` <= 64 so far, lane i holding the i-th
struct Best {
    u64 mine = 0, least = 0;                // least: the k-th, or a bound under it, in every lane
    __device__ __forceinline__ void insert(u64 cand, int k) {           // cand: the same in every lane
        const int lane = threadIdx.x & 63;
        const int p = __builtin_popcountll(__ballot(mine > cand));
        const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(mine >> 32), 0x138, 0xf, 0xf, false);     // from the lane below
        const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)mine, 0x138, 0xf, 0xf, false);
        mine = lane < p ? mine : (lane == p ? cand : ((u64)hi << 32 | lo));
        const u64 kth = lane_u64(mine, k - 1);
        least = kth > least ? kth : least;
    }
    // before the first offers: the k-th largest of the lanes' own maxima bounds the k-th of all from below.  Without it the first entries
    // to come are inserted and driven out again, k (1 + log(entries / k)) times an insertion's 30 instructions
    __device__ __forceinline__ void bound(float top, int k) {
        unsigned u = code(top), best = 0;
        for (int n = 0; n < k; n++) { best = reduce_max_u<64>(u); u = u == best ? 0u : u; }
        least = (u64)best << 32;
    }
    __device__ __forceinline__ void offer(u64 own, int k) {             // own: this lane's candidate
        u64 left = __ballot(own > least);
        while (left) {
            insert(lane_u64(own, __builtin_ctzll(left)), k);
            left &= left - 1;
            left &= __ballot(own > least);
        }
    }
};

__device__ __forceinline__ void join(Part& a, const Part& b) {
    const float m = fmaxf(a.m, b.m);
    const bool ea = a.m == m, eb = b.m == m;
    const float da = a.m - m, db = b.m - m, fa = exp_neg(da), fb = exp_neg(db);
    const float sa = a.c + a.r, sb = b.c + b.r;
    // the entries of the part with the lower maximum are da further down: e^{da} (t + da s).  (e^{da} = 0: nothing of it is left; this
    // also keeps 0 * -inf out where a part has no valid entry.  Equal maxima: the sums add.)
    const float ta = ea ? a.t : (fa == 0.f ? 0.f : fa * (a.t + da * sa)), tb = eb ? b.t : (fb == 0.f ? 0.f : fb * (b.t + db * sb));
    a.r = (ea ? a.r : fa * sa) + (eb ? b.r : fb * sb);
    a.c = (ea ? a.c : 0.f) + (eb ? b.c : 0.f);
    a.t = ta + tb; a.m = m;
}
__device__ __forceinline__ Part wave_join(Part p) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        Part b;
        b.m = __shfl_xor(p.m, o); b.c = __shfl_xor(p.c, o); b.r = __shfl_xor(p.r, o); b.t = __shfl_xor(p.t, o);
        join(p, b);
    }
    return p;
}

template <typename T> __device__ __forceinline__ void finish_row(const Rows& q, long row, const Part& p, const Best& best) {
    const int lane = threadIdx.x & 63;
    const Stat s = finish(p.m, p.c, p.r, p.t);
    if (lane == 0) {
        if (q.logp) {
            const long long a = q.actions[row];
            float xa = -INFINITY;
            if (a >= 0 && a < q.A && (!q.valid || q.valid[row * q.valid_stride + a])) xa = (float)((const T*)q.raw)[row * q.raw_stride + a];
            q.logp[row] = given_logp(s, xa, a, q.A);
        }
        q.entropy[row] = s.H;
        if (q.stats) { q.stats[2 * row] = s.m; q.stats[2 * row + 1] = s.logs; }
    }
    if (lane < q.k) {
        const unsigned u = (unsigned)(best.mine >> 32);
        q.top[row * q.k + lane] = u ? (long long)(int)~(unsigned)best.mine : -1;
        q.top_logp[row * q.k + lane] = u ? (value_of(u) - s.m) - s.logs : -INFINITY;
    }
}

// A part of a row as entries: `head` single ones up to the first 16-byte boundary (the first part's), the vectors v0 .. v1 - 1 behind
// them, the rest from `tail` on (the last part's).
struct Span { int head, v0, v1, tail; };
template <typename T, int VEC> __device__ __forceinline__ Span span_of(const T* x0, int A, int part, int S) {
    Span s;
    int head = VEC == 1 ? 0 : (int)(((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) & 15) / sizeof(T));
    if (head > A) head = A;
    const int nv = (A - head) / VEC;
    s.head = head; s.tail = head + nv * VEC;
    s.v0 = (int)((long)nv * part / S); s.v1 = (int)((long)nv * (part + 1) / S);
    return s;
}
// VEC entries from `j` on as they lie in memory, with their mask; and as floats, -inf where invalid.  Two steps, so that the loads of
// several of them go out before the first is waited for (a mask behind a branch makes every load wait for the one before it)
template <typename T, int VEC, bool MASK> struct Entries {
    vec<T, VEC> x;
    vec<uint8_t, VEC> v;
    __device__ __forceinline__ void fetch(const T* x0, const uint8_t* v0, int j) {
        x = *(const vec<T, VEC>*)(x0 + j);
        if constexpr (MASK) v = *(const vec<uint8_t, VEC>*)(v0 + j);
    }
    __device__ __forceinline__ void get(float (&o)[VEC], bool in) const {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            bool ok = in;
            if constexpr (MASK) ok = ok && v[i];
            o[i] = ok ? (float)x[i] : -INFINITY;
        }
    }
};
template <typename T> __device__ __forceinline__ float entry(const T* x0, const uint8_t* v0, int j) { return !v0 || v0[j] ? (float)x0[j] : -INFINITY; }

// WAVES waves to a part of a row: four, or one where there are rows enough to fill the chip with it -- a wave that sees more of a row
// inserts fewer alternatives that are driven out again, and nothing is joined
template <typename T, int VEC, bool MASK, int WAVES>
__global__ void __launch_bounds__(256) logprobs_long_kernel(Rows q) {
    __shared__ Part parts[4];
    __shared__ u64 lists[4][64];
    constexpr int TH = 64 * WAVES;
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % WAVES, tid = threadIdx.x % TH;
    const long job = (long)blockIdx.x * (4 / WAVES) + threadIdx.x / TH, row = job / q.S;
    const int part = (int)(job - row * q.S);
    if (WAVES == 1 && row >= q.R) return;
    const T* x0 = (const T*)q.raw + row * q.raw_stride;
    const uint8_t* v0 = q.valid ? q.valid + row * q.valid_stride : nullptr;
    const Span s = span_of<T, VEC>(x0, q.A, part, q.S);
    Part p = {-INFINITY, 0.f, 0.f, 0.f};
    Best best;
    constexpr int U = VEC == 1 ? 8 : VEC == 4 ? 4 : 2;       // vectors of a lane in flight: 8 or 16 entries, at 6 to 8 waves per SIMD
    for (int v = s.v0 + tid; __any(v < s.v1); v += TH * U) {
        Entries<T, VEC, MASK> raw[U];
        float x[U][VEC];
#pragma unroll
        for (int u = 0; u < U; u++) { const int at = v + TH * u; raw[u].fetch(x0, v0, s.head + VEC * (at < s.v1 ? at : s.v1 - 1)); }
#pragma unroll
        for (int u = 0; u < U; u++) raw[u].get(x[u], v + TH * u < s.v1);
        float tops[U];
#pragma unroll
        for (int u = 0; u < U; u++) tops[u] = max_of(x[u]);
        const float top = max_of(tops);
        if (top > p.m) { const Part higher = {top, 0.f, 0.f, 0.f}; join(p, higher); }
#pragma unroll
        for (int u = 0; u < U; u++) eat(p, x[u]);
        if (q.k) {
            if (v - tid == s.v0) best.bound(top, q.k);
#pragma unroll
            for (int u = 0; u < U; u++) {
                // (a NaN hides from the maximum but not from the sum)
                u64 hits = __ballot(code(tops[u]) >= (unsigned)(best.least >> 32) || p.r != p.r);
                if constexpr (VEC == 1) { if (hits) best.offer(pack(x[u][0], v + TH * u), q.k); }
                else while (hits) {                 // few: one lane's entries, dealt out to lanes 0 .. VEC - 1
                    const int from = __builtin_ctzll(hits);
                    hits &= hits - 1;
                    float mine = -INFINITY;
#pragma unroll
                    for (int i = 0; i < VEC; i++) { const float o = lane_f(x[u][i], from); mine = lane == i ? o : mine; }
                    best.offer(pack(mine, s.head + VEC * (v - lane + from + TH * u) + lane), q.k);
                }
            }
        }
    }
    // the single entries before the first part's vectors and behind the last's, under 8 each
    if (VEC > 1 && wave == 0) {
        const bool front = part == 0 && lane < s.head, back = part == q.S - 1 && lane >= 8 && lane - 8 < q.A - s.tail;
        if (__any(front || back)) {
            const int j = front ? lane : s.tail + lane - 8;
            const float x[1] = {front || back ? entry(x0, v0, j) : -INFINITY};
            if (x[0] > p.m) { const Part higher = {x[0], 0.f, 0.f, 0.f}; join(p, higher); }
            eat(p, x);
            if (q.k) best.offer(pack(x[0], j), q.k);
        }
    }
    p = wave_join(p);
    if constexpr (WAVES > 1) {
        if (lane == 0) parts[wave] = p;
        lists[wave][lane] = best.mine;
        __syncthreads();
        if (wave) return;
        for (int w = 1; w < WAVES; w++) {
            join(p, parts[w]);
            if (q.k) best.offer(lane < q.k ? lists[w][lane] : 0ull, q.k);
        }
    }
    if (q.S == 1) { finish_row<T>(q, row, p, best); return; }
    char* to = q.parts + job * (sizeof(Part) + 8l * q.k);
    if (lane == 0) *(Part*)to = p;
    if (lane < q.k) ((u64*)(to + sizeof(Part)))[lane] = best.mine;
}

// the parts of a row, in their order
template <typename T>
__global__ void __launch_bounds__(64) logprobs_join_kernel(Rows q) {
    const long row = blockIdx.x;
    const int lane = threadIdx.x;
    const long size = sizeof(Part) + 8l * q.k;
    const char* from = q.parts + row * q.S * size;
    Part p = {-INFINITY, 0.f, 0.f, 0.f};
    if (lane < q.S) p = *(const Part*)(from + lane * size);           // S <= 64
    p = wave_join(p);
    Best best;
    for (int i = lane; __any(i < q.S * q.k); i += 64) {
        u64 own = 0;
        if (i < q.S * q.k) { const int part = i / q.k; own = ((const u64*)(from + part * size + sizeof(Part)))[i - part * q.k]; }
        best.offer(own, q.k);
    }
    finish_row<T>(q, row, p, best);
}

template <typename T, int VEC, bool MASK>
__global__ void __launch_bounds__(256) logprobs_long_grad_kernel(Grads q) {
    const long row = blockIdx.x / q.S;
    const int part = (int)(blockIdx.x - row * q.S), tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const T* x0 = (const T*)q.raw + row * q.raw_stride;
    const uint8_t* v0 = q.valid ? q.valid + row * q.valid_stride : nullptr;
    T* d0 = (T*)q.d_raw + row * q.A;
    const Span s = span_of<T, VEC>(x0, q.A, part, q.S);
    const long long a = q.actions ? q.actions[row] : -1;
    const float m = q.stats[2 * row], logs = q.stats[2 * row + 1], H = q.entropy[row];
    const float gH = q.g_entropy ? q.g_entropy[row] : 0.f;
    const float ga = q.g_logp && a >= 0 ? (a < q.A ? q.g_logp[row] : NAN) : 0.f;
    float total = ga;
    if (q.g_top) {
        const float own = lane < q.k && q.top[row * q.k + lane] >= 0 ? q.g_top[row * q.k + lane] : 0.f;
        total += reduce<64, Sum>(own);
    }
    auto grad = [&](float x, int j) {
        const float lp = (x - m) - logs, pr = exp_neg(lp);
        const float w = total + gH * ((lp < -3e38f ? -3e38f : lp) + H);
        const float g = (j == a ? ga : 0.f) - (pr == 0.f ? 0.f : pr * w);
        return x == -INFINITY ? 0.f : g;
    };
    constexpr int U = VEC == 1 ? 8 : 4;
    for (int v = s.v0 + tid; v < s.v1; v += 256 * U) {
        Entries<T, VEC, MASK> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) { const int at = v + 256 * u; raw[u].fetch(x0, v0, s.head + VEC * (at < s.v1 ? at : s.v1 - 1)); }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = s.head + VEC * (v + 256 * u);
            float x[VEC], o[VEC];
            raw[u].get(x, true);
#pragma unroll
            for (int i = 0; i < VEC; i++) o[i] = grad(x[i], j + i);
            if (v + 256 * u < s.v1) store<T, VEC>(d0 + j, o);
        }
    }
    const int singles = wave == 0 && part == 0 ? s.head : (wave == 1 && part == q.S - 1 ? q.A - s.tail : 0);
    if (VEC > 1 && lane < singles) {
        const int j = (wave == 0 ? 0 : s.tail) + lane;
        d0[j] = (T)grad(entry(x0, v0, j), j);
    }
    if (!q.g_top) return;
    // the alternatives' own terms, over what this workgroup has just written
    __syncthreads();
    const int lo = part == 0 ? 0 : s.head + VEC * s.v0, hi = part == q.S - 1 ? q.A : s.head + VEC * s.v1;
    if (tid < q.k) {
        const long long j = q.top[row * q.k + tid];
        if (j >= lo && j < hi) d0[j] = (T)(grad(entry(x0, v0, (int)j), (int)j) + q.g_top[row * q.k + tid]);
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------
// Parts of a long row: enough workgroups to cover the chip twice, none shorter than SEGMENT entries (a part costs a launch's tail and
// its share of the join), at most 64 (the join holds one per lane).
int parts_of(long R, int A) {
    if (A <= SHORT) return 1;
    const long want = (512 + R - 1) / R, most = A / SEGMENT;
    long s = want < most ? want : most;
    return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}
// Rows whose 16-byte boundaries fall on the same entries in `raw` and in the contiguous result, and on whole words of the mask: V entries of
// each at a time.  Otherwise one by one
bool vectors(const void* raw, long stride, const void* other, const uint8_t* valid, long valid_stride, int A, int size) {
    const int V = 16 / size;
    if ((reinterpret_cast<uintptr_t>(raw) & 15) || (reinterpret_cast<uintptr_t>(other) & 15)) return false;
    if (valid && ((reinterpret_cast<uintptr_t>(valid) % V) || (valid_stride - stride) % V)) return false;
    return stride == A || (stride % V == 0 && A % V == 0);
}

template <typename T, int G, int N> void go_short(const Rows& q, hipStream_t s) {
    hipLaunchKernelGGL((logprobs_rows_kernel<T, G, N>), dim3((unsigned)((q.R * G + 255) / 256)), dim3(256), 0, s, q);
}
template <typename T, int G, int N> void go_short(const Grads& q, hipStream_t s) {
    hipLaunchKernelGGL((logprobs_rows_grad_kernel<T, G, N>), dim3((unsigned)((q.R * G + 255) / 256)), dim3(256), 0, s, q);
}
template <typename T, typename Q> void pick_short(const Q& q, hipStream_t s) {
    if (q.A <= 32) go_short<T, 16, 2>(q, s);
    else if (q.A <= 64) go_short<T, 16, 4>(q, s);
    else if (q.A <= 96) go_short<T, 16, 6>(q, s);
    else if (q.A <= 128) go_short<T, 16, 8>(q, s);
    else if (q.A <= 192) go_short<T, 16, 12>(q, s);
    else if (q.A <= 256) go_short<T, 16, 16>(q, s);
    else if (q.A <= 384 && q.R >= SHARED_WAVE) go_short<T, 16, 24>(q, s);
    else if (q.A <= 512 && q.R >= SHARED_WAVE) go_short<T, 16, 32>(q, s);
    else if (q.A <= 768 && q.R >= SHARED_WAVE) go_short<T, 32, 24>(q, s);
    else if (q.R >= SHARED_WAVE) go_short<T, 32, 32>(q, s);
    else if (q.A <= 512) go_short<T, 64, 8>(q, s);
    else go_short<T, 64, 16>(q, s);
}
template <typename T> int run(const Rows& q, hipStream_t s) {
    if (q.A <= SHORT) { pick_short<T>(q, s); return check_launch(); }
    constexpr int V = 16 / sizeof(T);
    const dim3 grid((unsigned)(q.R * q.S));
    const bool wide = vectors(q.raw, q.raw_stride, q.raw, q.valid, q.valid_stride, q.A, sizeof(T));
    if (q.R >= ONE_WAVE) {
        const dim3 grid4((unsigned)((q.R + 3) / 4));
        if (wide && !q.valid) hipLaunchKernelGGL((logprobs_long_kernel<T, V, false, 1>), grid4, dim3(256), 0, s, q);
        else if (wide) hipLaunchKernelGGL((logprobs_long_kernel<T, V, true, 1>), grid4, dim3(256), 0, s, q);
        else if (!q.valid) hipLaunchKernelGGL((logprobs_long_kernel<T, 1, false, 1>), grid4, dim3(256), 0, s, q);
        else hipLaunchKernelGGL((logprobs_long_kernel<T, 1, true, 1>), grid4, dim3(256), 0, s, q);
        return check_launch();
    }
    if (wide && !q.valid) hipLaunchKernelGGL((logprobs_long_kernel<T, V, false, 4>), grid, dim3(256), 0, s, q);
    else if (wide) hipLaunchKernelGGL((logprobs_long_kernel<T, V, true, 4>), grid, dim3(256), 0, s, q);
    else if (!q.valid) hipLaunchKernelGGL((logprobs_long_kernel<T, 1, false, 4>), grid, dim3(256), 0, s, q);
    else hipLaunchKernelGGL((logprobs_long_kernel<T, 1, true, 4>), grid, dim3(256), 0, s, q);
    if (q.S > 1) hipLaunchKernelGGL((logprobs_join_kernel<T>), dim3((unsigned)q.R), dim3(64), 0, s, q);
    return check_launch();
}
template <typename T> int run(const Grads& q, hipStream_t s) {
    if (q.A <= SHORT) { pick_short<T>(q, s); return check_launch(); }
    constexpr int V = 16 / sizeof(T);
    const dim3 grid((unsigned)(q.R * q.S));
    const bool wide = vectors(q.raw, q.raw_stride, q.d_raw, q.valid, q.valid_stride, q.A, sizeof(T));
    if (wide && !q.valid) hipLaunchKernelGGL((logprobs_long_grad_kernel<T, V, false>), grid, dim3(256), 0, s, q);
    else if (wide) hipLaunchKernelGGL((logprobs_long_grad_kernel<T, V, true>), grid, dim3(256), 0, s, q);
    else if (!q.valid) hipLaunchKernelGGL((logprobs_long_grad_kernel<T, 1, false>), grid, dim3(256), 0, s, q);
    else hipLaunchKernelGGL((logprobs_long_grad_kernel<T, 1, true>), grid, dim3(256), 0, s, q);
    return check_launch();
}

int check_rows(const void* raw, int dtype, long raw_stride, const uint8_t* valid, long valid_stride, long R, int A, int k) {
    if (!raw || R <= 0 || A <= 0 || k < 0 || raw_stride < 0 || (valid && valid_stride < 0)) return BL_EINVAL;
    if (dtype != BL_F32 && dtype != BL_F16 && dtype != BL_BF16) return BL_EINVAL;
    if (k > BL_TOP_MAX || A > BL_LOGPROBS_MAX || R > BL_LOGPROBS_ROWS) return BL_ETOOBIG;      // (the largest grid: 2^24 rows x 64 lanes)
    return BL_OK;
}

}  // namespace

extern "C" {

long bl_logprobs_workspace(long R, int A, int k) {
    if (R <= 0 || A <= 0 || k < 0) return 0;
    const int S = parts_of(R, A);
    return S == 1 ? 0 : R * S * ((long)sizeof(Part) + 8l * k);
}

int bl_logprobs(const void* raw, int dtype, long raw_stride, const uint8_t* valid, long valid_stride, const long long* actions, long R,
                int A, int k, float* logp, float* entropy, long long* top, float* top_logp, float* stats, void* workspace,
                bl_stream_t stream) {
    if (const int rc = check_rows(raw, dtype, raw_stride, valid, valid_stride, R, A, k)) return rc;
    if (!entropy || (actions == nullptr) != (logp == nullptr) || (k > 0 && (!top || !top_logp))) return BL_EINVAL;
    Rows q{raw, raw_stride, valid, valid_stride, actions, R, A, k, logp, entropy, top, top_logp, stats, parts_of(R, A), (char*)workspace};
    if (q.S > 1 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7))) return BL_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    return dtype == BL_F32 ? run<float>(q, s) : dtype == BL_F16 ? run<f16>(q, s) : run<bf16>(q, s);
}

int bl_logprobs_grad(const void* raw, int dtype, long raw_stride, const uint8_t* valid, long valid_stride, const long long* actions,
                     long R, int A, int k, const long long* top, const float* stats, const float* entropy, const float* g_logp,
                     const float* g_entropy, const float* g_top, void* d_raw, bl_stream_t stream) {
    if (const int rc = check_rows(raw, dtype, raw_stride, valid, valid_stride, R, A, k)) return rc;
    if (!stats || !entropy || !d_raw || (g_logp && !actions) || (g_top && (!top || k == 0))) return BL_EINVAL;
    Grads q{raw, raw_stride, valid, valid_stride, actions, top, stats, entropy, g_logp, g_entropy, g_top, R, A, k, d_raw, parts_of(R, A)};
    const hipStream_t s = (hipStream_t)stream;
    return dtype == BL_F32 ? run<float>(q, s) : dtype == BL_F16 ? run<f16>(q, s) : run<bf16>(q, s);
}

}  // extern "C"
