// bl_norm.hip -- the residual stream between two blocks in one pass: norm behind the block, its gate, the residual scale, norm before
// the next block; and the gradient.  Per row of W:
//     n = y / rms(y),  u = sigmoid(gate) post n,  x' = x + alpha u,  h = pre x' / rms(x'),     rms(v) = sqrt(mean v^2 + eps)
// Backward, with xn = x' / rms(x') recomputed from x and y (so it is not the rounded x' that is differentiated) and the two reciprocal
// rms of the forward pass:
//     z  = g_x' + rx (t - xn mean(t xn)),  t = g_h pre;      dx = z;      dpre = sum_rows g_h xn;      dalpha = sum z u
//     dgate = alpha z post n s (1 - s);    dpost = sum_rows alpha z s n;  dy = ry (dn - n mean(dn n)),  dn = alpha z s post
// Everything is computed in f32 and rounded once at its store.  The bound is HBM: every element is read once and written once; a row
// is held in registers by G lanes of 8 elements each, so the two dependent sums of a row cost no second read.  The sums over rows are
// kept per workgroup in registers over all of its rows and added up by a second launch in a fixed order: no atomics, the same bits
// every time.  32768 x 512, f32 stream, f16 branches with gates: forward 42 us for 235 MB (5.5 TB/s), backward 68 us for 369 MB (5.4 TB/s) and
// 4 us for the sums; 4096 x 771 f32 14 + 21 + 4 us; 8192 x 4096 bf16 forward 58 us for 335 MB (5.8 TB/s); a copy of 4 GiB runs at 4.75 TB/s, of 32 MiB at 6.6,
// the data sheet says 8.
#include "bl_train.h"
#include "bl_host.h"

#pragma clang fp contract(off)

using namespace bltrain;

namespace {

struct Norm {
    const void* x; long xs;
    const void* y; long ys;
    const float* alpha; const float* post;
    const void* gate; long gs; int kind;
    const float* pre;
    float eps, inv_w; long R; int W;
    void* xo; void* h; float* stats;        // forward
    const void* gx; long gxs; const void* gh; long ghs;          // backward
    void* dx; void* dy; long dys; void* dgate; long dgs; float* parts;
};

// which of a workgroup's rows: the same for a wave's lanes where a row is a wave's or more, and said so, which makes a row's addresses scalar
template <int G> __device__ __forceinline__ int group_of() {
    const int g = threadIdx.x / G;
    if constexpr (G >= 64) return __builtin_amdgcn_readfirstlane(g);
    return g;
}

// where lane gl's N elements of a row are: VEC == 8 in eights (16-byte accesses), VEC == 1 every G-th
template <int G, int VEC> __device__ __forceinline__ int column(int gl, int i) { return VEC == 8 ? 8 * (gl + G * (i / 8)) + i % 8 : gl + G * i; }

// A lane's elements as they lie in memory, and as floats (0 beyond W).  Two steps, so that all of a row's tensors are on their way before the first is
// waited for; the address is clamped instead of a branch around the load
template <int G, int VEC, int N, typename T> struct Elements {
    vec<T, VEC> v[N / VEC];
    __device__ __forceinline__ void fetch(const T* p, int gl, int W) {
#pragma unroll
        for (int c = 0; c < N / VEC; c++) { const int j = column<G, VEC>(gl, c * VEC); v[c] = *(const vec<T, VEC>*)(p + (j < W ? j : W - VEC)); }
    }
    __device__ __forceinline__ void get(float (&o)[N], int gl, int W) const {
#pragma unroll
        for (int c = 0; c < N / VEC; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) o[c * VEC + i] = column<G, VEC>(gl, c * VEC) < W ? (float)v[c][i] : 0.f;
    }
};
template <int G, int VEC, typename T, int N> __device__ __forceinline__ void read(const T* p, int gl, int W, float (&o)[N]) {
    Elements<G, VEC, N, T> e;
    e.fetch(p, gl, W);
    e.get(o, gl, W);
}
template <int G, int VEC, typename T, int N> __device__ __forceinline__ void write(T* p, int gl, int W, const float (&o)[N]) {
    if constexpr (VEC == 8) {
#pragma unroll
        for (int c = 0; c < N; c += 8) {
            const int j = column<G, 8>(gl, c);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = o[c + i];
            if (j < W) store<T, 8>(p + j, v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) { const int j = gl + G * i; if (j < W) p[j] = (T)o[i]; }
    }
}

// sum over the G lanes of a row, in every one of them.  G > 64: a row is several waves'; `lds` holds a value per wave, two sets of them in
// turn (`set`), so that one barrier per sum is enough
template <int G> __device__ __forceinline__ float row_sum(float v, float* lds, int& set) {
    v = reduce<(G < 64 ? G : 64), Sum>(v);
    if constexpr (G > 64) {
        float* at = lds + 16 * set;
        set ^= 1;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        __syncthreads();
        at += threadIdx.x / G * (G / 64);
        v = at[0];
#pragma unroll
        for (int w = 1; w < G / 64; w++) v += at[w];
    }
    return v;
}

struct Gate { float s, ds; };               // sigmoid and its derivative
__device__ __forceinline__ Gate sigmoid(float g) {
    const float e = __builtin_amdgcn_exp2f(g * -1.44269504088896341f), s = __builtin_amdgcn_rcpf(1.f + e);
    return {s, s == 0.f ? 0.f : e * s * s};
}

// Rows beyond 1.8e19, or under 1e-15 with an eps as small, have squares outside f32's range.  The kernel notes that one of its rows has, and
// these come again behind its loop, from memory instead of registers, with the sums made of values scaled by a power of two.  (A branch behind each sum takes
// registers with it: 8192 x 4096 bf16 34 -> 41 us)
template <typename TX, typename TY, int G> __device__ __forceinline__ void odd_rows(const Norm& q, float* lds, int set) {
    constexpr int ROWS = G > 256 ? 1 : 256 / G;
    const int gl = threadIdx.x & (G - 1);
    const float alpha = q.alpha ? *q.alpha : 1.f;
    for (long r0 = (long)blockIdx.x * ROWS; r0 < q.R; r0 += (long)gridDim.x * ROWS) {
        const long row = r0 + group_of<G>(), at = row < q.R ? row : q.R - 1;
        const TX* x = (const TX*)q.x + at * q.xs;
        const TY* y = (const TY*)q.y + at * q.ys;
        bool odd = false;
        auto inverse_rms = [&](auto value) {
            auto mean = [&](float scale) {
                float ss = 0.f;
#pragma unroll 1
                for (int j = gl; j < q.W; j += G) { const float v = value(j) * scale; ss = fmaf(v, v, ss); }
                return row_sum<G>(ss, lds, set) * q.inv_w + q.eps * scale * scale;
            };
            const float first = mean(1.f), scale = first < 0x1p-100f ? 0x1p100f : first <= 0x1p126f ? 1.f : 0x1p-72f;
            odd = odd || scale != 1.f;
            return __builtin_amdgcn_rsqf(mean(scale)) * scale;
        };
        const float ry = q.post ? inverse_rms([&](int j) { return (float)y[j]; }) : 1.f;
        auto x_out = [&](int j) {
            if (!q.y) return (float)x[j];
            float u = (float)y[j];
            if (q.post) u *= q.post[j] * ry;
            if (q.kind != BL_GATE_NONE)
                u *= sigmoid(q.kind == BL_GATE_CHANNEL ? ((const float*)q.gate)[j] : (float)((const TY*)q.gate)[at * q.gs + (q.kind == BL_GATE_FULL ? j : 0)]).s;
            return fmaf(alpha, u, (float)x[j]);
        };
        const float rx = q.pre ? inverse_rms(x_out) : 1.f;
        if (!odd || row >= q.R) continue;
#pragma unroll 1
        for (int j = gl; j < q.W; j += G) {
            const float v = x_out(j);
            if (q.y) ((TX*)q.xo)[at * q.W + j] = (TX)v;
            if (q.pre) ((TY*)q.h)[at * q.W + j] = (TY)(q.pre[j] * (v * rx));
        }
        if (q.stats && gl == 0) { q.stats[2 * at] = ry; q.stats[2 * at + 1] = rx; }
    }
}

template <typename TX, typename TY, int G, int N, int VEC>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_kernel(Norm q) {
    __shared__ float lds[32];
    constexpr int T = G > 256 ? G : 256, ROWS = T / G;
    const int gl = threadIdx.x & (G - 1);
    int set = 0;
    float post[N], pre[N], gate[N];
    if (q.post) read<G, VEC>(q.post, gl, q.W, post);
    if (q.pre) read<G, VEC>(q.pre, gl, q.W, pre);
    if (q.kind == BL_GATE_CHANNEL) read<G, VEC>((const float*)q.gate, gl, q.W, gate);
    const float alpha = q.alpha ? *q.alpha : 1.f;
    float least = 1.f, most = 1.f;              // reciprocals of rms
    for (long r0 = (long)blockIdx.x * ROWS; r0 < q.R; r0 += (long)gridDim.x * ROWS) {
        const long row = r0 + group_of<G>(), at = row < q.R ? row : q.R - 1;      // (G > 64: one row per workgroup, always live)
        const bool live = row < q.R;
        Elements<G, VEC, N, TX> ex;
        Elements<G, VEC, N, TY> ey, eg;
        ex.fetch((const TX*)q.x + at * q.xs, gl, q.W);
        if (q.y) ey.fetch((const TY*)q.y + at * q.ys, gl, q.W);
        if (q.kind == BL_GATE_FULL) eg.fetch((const TY*)q.gate + at * q.gs, gl, q.W);
        float x[N];
        ex.get(x, gl, q.W);
        float ry = 1.f;
        if (q.y) {
            float y[N];
            ey.get(y, gl, q.W);
            if (q.kind == BL_GATE_FULL) eg.get(gate, gl, q.W);
            if (q.kind == BL_GATE_ROW) {
                const float g = (float)((const TY*)q.gate)[at * q.gs];
#pragma unroll
                for (int i = 0; i < N; i++) gate[i] = g;
            }
            if (q.post) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < N; i++) ss = fmaf(y[i], y[i], ss);
                ry = __builtin_amdgcn_rsqf(row_sum<G>(ss, lds, set) * q.inv_w + q.eps);
#pragma unroll
                for (int i = 0; i < N; i++) y[i] *= post[i] * ry;
            }
            if (q.kind != BL_GATE_NONE)
#pragma unroll
                for (int i = 0; i < N; i++) y[i] *= sigmoid(gate[i]).s;
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = fmaf(alpha, y[i], x[i]);
            if (live) write<G, VEC>((TX*)q.xo + at * q.W, gl, q.W, x);
        }
        float rx = 1.f;
        if (q.pre) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < N; i++) if (column<G, VEC>(gl, i) < q.W) ss = fmaf(x[i], x[i], ss);
            rx = __builtin_amdgcn_rsqf(row_sum<G>(ss, lds, set) * q.inv_w + q.eps);
            float h[N];
#pragma unroll
            for (int i = 0; i < N; i++) h[i] = pre[i] * (x[i] * rx);
            if (live) write<G, VEC>((TY*)q.h + at * q.W, gl, q.W, h);
        }
        if (q.stats && live && gl == 0) { q.stats[2 * at] = ry; q.stats[2 * at + 1] = rx; }
        least = fminf(least, fminf(ry, rx)); most = fmaxf(most, fmaxf(ry, rx));
    }
    const bool odd = least < 0x1p-63f || most > 0x1p50f;
    if constexpr (G == 128) { if (!__syncthreads_or(odd)) return; }        // two rows, which share their barriers
    else if (!__any(odd)) return;                                          // (a row of more lanes is its workgroup's only one: the same in every wave)
    odd_rows<TX, TY, G>(q, lds, set);
}

// A lane's sums over its rows, for dpost, dpre and a gate per channel.  In registers; at 16 waves per workgroup, where a lane has 128 of them
// and needs 150, in LDS (its own places, no bank conflict): 2048 x 8192 f32 / f16 124 us with its launches, 196 with what spilled from registers;
// 2048 x 8191, whose single elements need more addresses, 259 with some spills left (445)
enum { POST, PRE, GATE };
template <int G, int N> struct Columns {
    float v[3][N];
    __device__ __forceinline__ explicit Columns(float*) {
#pragma unroll
        for (int a = 0; a < 3; a++)
#pragma unroll
            for (int i = 0; i < N; i++) v[a][i] = 0.f;
    }
    __device__ __forceinline__ void add(int a, int i, float x, float y) { v[a][i] = fmaf(x, y, v[a][i]); }
    __device__ __forceinline__ float get(int a, int i) const { return v[a][i]; }
};
template <int N> struct Columns<1024, N> {
    float* v;
    __device__ __forceinline__ explicit Columns(float* lds) : v(lds + threadIdx.x) {
#pragma unroll
        for (int i = 0; i < 3 * N; i++) v[1024 * i] = 0.f;
    }
    __device__ __forceinline__ void add(int a, int i, float x, float y) { v[1024 * (a * N + i)] = fmaf(x, y, v[1024 * (a * N + i)]); }
    __device__ __forceinline__ float get(int a, int i) const { return v[1024 * (a * N + i)]; }
};

template <typename TX, typename TY, int G, int N, int VEC>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_grad_kernel(Norm q) {
    extern __shared__ __align__(16) float wide[];
    __shared__ float lds[32];
    constexpr int T = G > 256 ? G : 256, ROWS = T / G;
    __shared__ float cols[ROWS > 1 ? 3 * N * G + 1 : 1];
    const int gl = threadIdx.x & (G - 1);
    int set = 0;
    float post[N], pre[N], gate[N];
    // gains and channel gates: in registers for all rows, or (16 waves) read again where a row needs them
    constexpr bool KEEP = G < 1024;
    auto read_post = [&] { if (q.post) read<G, VEC>(q.post, gl, q.W, post); };
    auto read_pre = [&] { if (q.gh) read<G, VEC>(q.pre, gl, q.W, pre); };
    auto read_gate = [&] { if (q.kind == BL_GATE_CHANNEL) read<G, VEC>((const float*)q.gate, gl, q.W, gate); };
    if (!q.post)
#pragma unroll
        for (int i = 0; i < N; i++) post[i] = 1.f;
    if constexpr (KEEP) { read_post(); read_pre(); read_gate(); }
    const float alpha = q.alpha ? *q.alpha : 1.f;
    Columns<G, N> sums(wide);
    float salpha = 0.f;
    for (long r0 = (long)blockIdx.x * ROWS; r0 < q.R; r0 += (long)gridDim.x * ROWS) {
        const long row = r0 + group_of<G>(), at = row < q.R ? row : q.R - 1;
        const bool live = row < q.R;
        const float ry = q.stats[2 * at], rx = q.stats[2 * at + 1];
        Elements<G, VEC, N, TX> ex, ez;
        Elements<G, VEC, N, TY> ey, eg, et;
        ex.fetch((const TX*)q.x + at * q.xs, gl, q.W);
        if (q.y) ey.fetch((const TY*)q.y + at * q.ys, gl, q.W);
        if (q.kind == BL_GATE_FULL) eg.fetch((const TY*)q.gate + at * q.gs, gl, q.W);
        if (q.gx) ez.fetch((const TX*)q.gx + at * q.gxs, gl, q.W);
        if (q.gh) et.fetch((const TY*)q.gh + at * q.ghs, gl, q.W);
        if constexpr (!KEEP) { read_post(); read_gate(); }
        // (beyond W everything is 0, so nothing there counts; the sigmoid is computed twice rather than held)
        float x[N], z[N], n[N];
        ex.get(x, gl, q.W);
        if (q.y) {
            ey.get(n, gl, q.W);
            if (q.kind == BL_GATE_FULL) eg.get(gate, gl, q.W);
            if (q.kind == BL_GATE_ROW) {
                const float g = (float)((const TY*)q.gate)[at * q.gs];
#pragma unroll
                for (int i = 0; i < N; i++) gate[i] = g;
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                n[i] *= ry;
                const float u = post[i] * n[i];
                x[i] = fmaf(alpha, q.kind != BL_GATE_NONE ? u * sigmoid(gate[i]).s : u, x[i]);
            }
        }
        if (q.gx) ez.get(z, gl, q.W);
        else
#pragma unroll
            for (int i = 0; i < N; i++) z[i] = 0.f;
        if (q.gh) {
            float t[N], c = 0.f;
            et.get(t, gl, q.W);
            if constexpr (!KEEP) read_pre();
#pragma unroll
            for (int i = 0; i < N; i++) {
                x[i] *= rx;                                                          // xn
                if (live) sums.add(PRE, i, t[i], x[i]);
                t[i] *= pre[i];
                c = fmaf(t[i], x[i], c);
            }
            c = row_sum<G>(c, lds, set) * q.inv_w;
            // one column: xn^2 = 1 - eps rx^2, and the difference would cancel
#pragma unroll
            for (int i = 0; i < N; i++) z[i] = fmaf(rx, q.W == 1 ? t[i] * (q.eps * rx * rx) : fmaf(-x[i], c, t[i]), z[i]);
        }
        if (live) write<G, VEC>((TX*)q.dx + at * q.W, gl, q.W, z);
        if (!q.y) continue;
        float c = 0.f, cg = 0.f, dn[N];
        if constexpr (!KEEP) { read_post(); read_gate(); }
        if (q.kind != BL_GATE_NONE) {
            float dg[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const Gate g = sigmoid(gate[i]);
                const float v = alpha * z[i], vn = v * n[i], sp = g.s * post[i];
                if (live) { salpha = fmaf(z[i], n[i] * sp, salpha); sums.add(POST, i, vn, g.s); }
                dn[i] = v * sp;
                c = fmaf(dn[i], n[i], c);
                dg[i] = vn * post[i] * g.ds;
                if (live && q.kind == BL_GATE_CHANNEL) sums.add(GATE, i, dg[i], 1.f);
                cg += dg[i];
            }
            if (q.kind == BL_GATE_FULL && q.dgate && live) write<G, VEC>((TY*)q.dgate + at * q.dgs, gl, q.W, dg);
            if (q.kind == BL_GATE_ROW) {
                cg = row_sum<G>(cg, lds, set);
                if (q.dgate && live && gl == 0) ((TY*)q.dgate)[at * q.dgs] = (TY)cg;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float v = alpha * z[i];
                if (live) { salpha = fmaf(z[i], n[i] * post[i], salpha); sums.add(POST, i, v, n[i]); }
                dn[i] = v * post[i];
                c = fmaf(dn[i], n[i], c);
            }
        }
        if (q.post) {
            c = row_sum<G>(c, lds, set) * q.inv_w;
#pragma unroll
            for (int i = 0; i < N; i++) dn[i] = ry * (q.W == 1 ? dn[i] * (q.eps * ry * ry) : fmaf(-n[i], c, dn[i]));
        }
        if (live) write<G, VEC>((TY*)q.dy + at * q.dys, gl, q.W, dn);
    }
    // this workgroup's sums over its rows: dpost, dpre, dgate per column, then dalpha
    float* out = q.parts + (long)blockIdx.x * (3l * q.W + 1);
    salpha = row_sum<G>(salpha, lds, set);
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int j = column<G, VEC>(gl, i);
            if (j < q.W) { out[j] = sums.get(POST, i); out[q.W + j] = sums.get(PRE, i); out[2 * q.W + j] = sums.get(GATE, i); }
        }
        if (gl == 0) out[3 * q.W] = salpha;
    } else {
        // the workgroup's groups of lanes one after the other: a fixed order
        for (int g = 0; g < ROWS; g++) {
            if (threadIdx.x / G == g) {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int k = gl + G * i;
#pragma unroll
                    for (int a = 0; a < 3; a++) cols[a * N * G + k] = g ? cols[a * N * G + k] + sums.get(a, i) : sums.get(a, i);
                }
                if (gl == 0) cols[3 * N * G] = g ? cols[3 * N * G] + salpha : salpha;
            }
            __syncthreads();
        }
        if (threadIdx.x < G) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int j = column<G, VEC>(gl, i), k = gl + G * i;
                if (j < q.W) { out[j] = cols[k]; out[q.W + j] = cols[N * G + k]; out[2 * q.W + j] = cols[2 * N * G + k]; }
            }
            if (gl == 0) out[3 * q.W] = cols[3 * N * G];
        }
    }
}

// the workgroups' sums added up: 64 columns by 16 parts of the workgroups, then the 16 parts
struct Sums { const float* parts; int blocks, W; float* dpost; float* dpre; float* dgate; float* dalpha; };
__global__ void __launch_bounds__(1024) norm_sums_kernel(Sums q) {
    __shared__ float lds[1024];
    const int C = 3 * q.W + 1, col = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
    float* to = col < q.W ? q.dpost : col < 2 * q.W ? q.dpre : col < 3 * q.W ? q.dgate : col < C ? q.dalpha : nullptr;
    float v = 0.f;
    if (to) {
        const int b0 = (int)((long)q.blocks * part / 16), b1 = (int)((long)q.blocks * (part + 1) / 16);
#pragma unroll 8
        for (int b = b0; b < b1; b++) v += q.parts[(long)b * C + col];
    }
    lds[threadIdx.x] = v;
    __syncthreads();
    if (part || !to) return;
#pragma unroll
    for (int p = 1; p < 16; p++) v += lds[threadIdx.x + 64 * p];
    to[col < 3 * q.W ? col % q.W : 0] = v;
}

// ---- host --------------------------------------------------------------------------------------------------------------------------
// Lanes of a row, 8 elements each: the fewest that hold it -- 16 rows to a wave up to 32 wide, a row to a wave up to 512 (no barrier), to a
// workgroup from 1025 on.  (16 elements per lane need 300 registers in the backward pass: 16384 x 768 f32 114 us with its launches, with 8 per lane in two
// waves 84)
constexpr int N = 8;
int lanes_of(int W) { return W <= 32 ? 4 : W <= 128 ? 16 : W <= 512 ? 64 : W <= 1024 ? 128 : W <= 2048 ? 256 : W <= 4096 ? 512 : 1024; }
// workgroups of the backward pass: each leaves 3 W + 1 sums, so no more than keep the chip full
int blocks_of(long R, int W) {
    const int G = lanes_of(W), rows = G > 256 ? 1 : 256 / G;
    const long need = (R + rows - 1) / rows, most = 512;
    return (int)(need < most ? need : most);
}
bool aligned(const void* p, long stride, int size) { return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * size) % 16 == 0); }

template <typename TX, typename TY, int G, int VEC> int go(const Norm& q, bool grad, hipStream_t s) {
    constexpr int T = G > 256 ? G : 256, ROWS = T / G;
    if (grad) {
        constexpr size_t bytes = G == 1024 ? 3 * N * G * sizeof(float) : 0;
        static size_t raised[64];
        if (!bl_raise_lds_limit((const void*)norm_grad_kernel<TX, TY, G, N, VEC>, bytes, raised)) return BL_ELAUNCH;
        hipLaunchKernelGGL((norm_grad_kernel<TX, TY, G, N, VEC>), dim3((unsigned)blocks_of(q.R, q.W)), dim3(T), bytes, s, q);
    } else {
        const long need = (q.R + ROWS - 1) / ROWS;
        hipLaunchKernelGGL((norm_kernel<TX, TY, G, N, VEC>), dim3((unsigned)(need < 2048 ? need : 2048)), dim3(T), 0, s, q);
    }
    return check_launch();
}
template <typename TX, typename TY, int VEC> int by_lanes(const Norm& q, bool grad, hipStream_t s) {
    switch (lanes_of(q.W)) {
        case 4: return go<TX, TY, 4, VEC>(q, grad, s);
        case 16: return go<TX, TY, 16, VEC>(q, grad, s);
        case 64: return go<TX, TY, 64, VEC>(q, grad, s);
        case 128: return go<TX, TY, 128, VEC>(q, grad, s);
        case 256: return go<TX, TY, 256, VEC>(q, grad, s);
        case 512: return go<TX, TY, 512, VEC>(q, grad, s);
        default: return go<TX, TY, 1024, VEC>(q, grad, s);
    }
}
template <typename TX, typename TY> int by_vec(const Norm& q, bool grad, hipStream_t s) {
    const int sx = sizeof(TX), sy = sizeof(TY);
    bool v = q.W % 8 == 0 && aligned(q.x, q.xs, sx) && aligned(q.y, q.ys, sy) && aligned(q.post, 0, 4) && aligned(q.pre, 0, 4);
    if (q.kind == BL_GATE_FULL) v = v && aligned(q.gate, q.gs, sy) && aligned(q.dgate, q.dgs, sy);
    if (q.kind == BL_GATE_CHANNEL) v = v && aligned(q.gate, 0, 4);
    v = v && aligned(q.xo, q.W, sx) && aligned(q.h, q.W, sy) && aligned(q.gx, q.gxs, sx) && aligned(q.gh, q.ghs, sy) && aligned(q.dx, q.W, sx) && aligned(q.dy, q.dys, sy);
    return v ? by_lanes<TX, TY, 8>(q, grad, s) : by_lanes<TX, TY, 1>(q, grad, s);
}
int by_type(const Norm& q, int tx, int ty, bool grad, hipStream_t s) {
    if (tx == BL_F32 && ty == BL_F32) return by_vec<float, float>(q, grad, s);
    if (tx == BL_F32 && ty == BL_F16) return by_vec<float, f16>(q, grad, s);
    if (tx == BL_F32 && ty == BL_BF16) return by_vec<float, bf16>(q, grad, s);
    if (tx == BL_F16 && ty == BL_F16) return by_vec<f16, f16>(q, grad, s);
    if (tx == BL_BF16 && ty == BL_BF16) return by_vec<bf16, bf16>(q, grad, s);
    return BL_EINVAL;
}
int check_norm(const Norm& q) {
    if (!q.x || q.R <= 0 || q.W <= 0 || !(q.eps >= 0.f) || q.xs < 0 || q.ys < 0 || q.gs < 0) return BL_EINVAL;
    if (q.kind < BL_GATE_NONE || q.kind > BL_GATE_ROW || (q.kind != BL_GATE_NONE) != (q.gate != nullptr)) return BL_EINVAL;
    if (!q.y && (q.kind != BL_GATE_NONE || q.post || !q.pre)) return BL_EINVAL;
    return q.W > BL_NORM_MAX ? BL_ETOOBIG : BL_OK;
}

}  // namespace

extern "C" {

int bl_norm_residual(const void* x, int x_dtype, long x_stride, const void* y, int y_dtype, long y_stride, const float* alpha,
                     const float* post, const void* gate, int gate_kind, long gate_stride, const float* pre, float eps, long R, int W,
                     void* x_out, void* h, float* stats, bl_stream_t stream) {
    Norm q{};
    q.x = x; q.xs = x_stride; q.y = y; q.ys = y_stride; q.alpha = alpha; q.post = post; q.gate = gate; q.gs = gate_stride; q.kind = gate_kind;
    q.pre = pre; q.eps = eps; q.inv_w = 1.f / (float)W; q.R = R; q.W = W; q.xo = x_out; q.h = h; q.stats = stats;
    if (const int rc = check_norm(q)) return rc;
    if ((y != nullptr) != (x_out != nullptr) || (pre != nullptr) != (h != nullptr)) return BL_EINVAL;
    return by_type(q, x_dtype, y_dtype, false, (hipStream_t)stream);
}

long bl_norm_residual_workspace(long R, int W) { return R <= 0 || W <= 0 || W > BL_NORM_MAX ? 0 : 4l * blocks_of(R, W) * (3l * W + 1); }

int bl_norm_residual_grad(const void* x, int x_dtype, long x_stride, const void* y, int y_dtype, long y_stride, const float* alpha,
                          const float* post, const void* gate, int gate_kind, long gate_stride, const float* pre, float eps, long R,
                          int W, const float* stats, const void* g_x, long g_x_stride, const void* g_h, long g_h_stride, void* d_x,
                          void* d_y, long d_y_stride, void* d_gate, long d_gate_stride, float* d_alpha, float* d_post, float* d_pre,
                          void* workspace, bl_stream_t stream) {
    Norm q{};
    q.x = x; q.xs = x_stride; q.y = y; q.ys = y_stride; q.alpha = alpha; q.post = post; q.gate = gate; q.gs = gate_stride; q.kind = gate_kind;
    q.pre = pre; q.eps = eps; q.inv_w = 1.f / (float)W; q.R = R; q.W = W; q.stats = (float*)stats;
    q.gx = g_x; q.gxs = g_x_stride; q.gh = g_h; q.ghs = g_h_stride; q.dx = d_x; q.dy = d_y; q.dys = d_y_stride;
    q.dgate = gate_kind == BL_GATE_CHANNEL ? nullptr : d_gate; q.dgs = d_gate_stride; q.parts = (float*)workspace;
    if (const int rc = check_norm(q)) return rc;
    if (!stats || !d_x || !workspace || (y != nullptr) != (d_y != nullptr) || (g_h && !pre) || g_x_stride < 0 || g_h_stride < 0 || d_y_stride < 0 || d_gate_stride < 0) return BL_EINVAL;
    if (const int rc = by_type(q, x_dtype, y_dtype, true, (hipStream_t)stream)) return rc;
    if (!d_alpha && !d_post && !d_pre && !(gate_kind == BL_GATE_CHANNEL && d_gate)) return BL_OK;
    Sums t{q.parts, blocks_of(R, W), W, d_post, d_pre, gate_kind == BL_GATE_CHANNEL ? (float*)d_gate : nullptr, d_alpha};
    hipLaunchKernelGGL(norm_sums_kernel, dim3((unsigned)((3 * W + 1 + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, t);
    return check_launch();
}

}  // extern "C"
