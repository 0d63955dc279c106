// bl_ortho.hip -- Newton-Schulz orthogonalisation of update matrices, for the learner's hidden weights.
//
//     X = G / (|G|_F + eps);   `steps` times:  A = X X^T,  B = b A + c A^2,  X = a X + B X        (on the side with fewer rows, m <= n)
//
// takes every singular value s to a s + b s^3 + c s^5 and again, i.e. towards 1.  The iteration multiplies what is small by up to 3.4 a
// step: with f16 or bf16 operands the rounding of the large directions drowns the small ones of a low-rank gradient (3.7 % / 30 % of the
// result on rank 8 + 1 % noise).  So every operand is a pair of f16 numbers hi + lo (22 bits and lo's sign), a product is hi hi + hi lo +
// lo hi on v_mfma_f32_32x32x16_f16 with f32 sums (the dropped lo lo is 2^-24 of the product: what f32 rounding costs), 3/16 of the matrix
// rate instead of the f32 MFMA's 1/16.  Operands carry a factor 2^13: entries of X and B stay below 3 (the quintic maps [0, 1.21] into
// itself), so hi < 2^15, and lo keeps its bits above f16's smallest steps down to entries of 2^-14.
//
// Operands lie in the workspace as MFMA fragments: 32 rows x 16 k, lane = row + 32 (k / 8), 8 consecutive k per lane, hi then lo -- a
// wave's load is one contiguous KiB and both operands of P Q^T use the same layout.  The accumulator holds 4 consecutive rows of D per
// lane, which are 4 consecutive k of D^T as an operand: writing D^T costs nothing, writing D as well goes through LDS once per tile.
// A and A^2 are symmetric: only the tiles on and above the diagonal are computed.
#include "bl_train.h"

#pragma clang fp contract(off)

using namespace bltrain;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float SCALE = 8192.f, UNSCALE = 1.f / 8192.f;
constexpr int TILE = 64, MANY = 32, PARTS = 32;
constexpr int FRAG = 512;                   // halves of one fragment, hi or lo

struct Mats { const void* in[MANY]; void* out[MANY]; };

int up(int v) { return (v + TILE - 1) / TILE * TILE; }

// halves from one fragment pair to the next are 2 FRAG; (rb, kb): 32 rows, 16 k
__device__ __forceinline__ long frag_at(int rb, int kb, int KB) { return ((long)rb * KB + kb) * (2 * FRAG); }

__device__ __forceinline__ void split(float v, f16& hi, f16& lo) { hi = (f16)v; lo = (f16)(v - (float)hi); }

// ---- |G|^2 in parts, in f64: neither 2^100 nor 2^-100 as a loss scale overflows or vanishes ----
template <typename T> __global__ void __launch_bounds__(256) norm_parts_kernel(Mats q, long total, double* parts) {
    __shared__ double lds[4];
    const T* g = (const T*)q.in[blockIdx.y];
    const long i0 = total * blockIdx.x / PARTS, i1 = total * (blockIdx.x + 1) / PARTS;
    double s = 0.;
    for (long i = i0 + threadIdx.x; i < i1; i += 256) { const double v = (double)(float)g[i]; s += v * v; }
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.y * PARTS + blockIdx.x] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// ---- X and X^T as operands, zero beyond (m, n).  A workgroup takes 32 rows x 32 columns; tall: G is n x m ----
template <typename T>
__global__ void __launch_bounds__(256) lay_out_kernel(Mats q, int m, int n, int tall, float eps, const double* parts, f16* X, f16* XT, long sx) {
    __shared__ float t[32][33];
    const T* g = (const T*)q.in[blockIdx.z];
    double ss = 0.;
    for (int p = 0; p < PARTS; p++) ss += parts[blockIdx.z * PARTS + p];
    const double inv = (double)SCALE / (sqrt(ss) + (double)eps);
    const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
    for (int e = threadIdx.x; e < 1024; e += 256) {
        const int i = e >> 5, j = e & 31;                       // i: the slow index of G
        const int r = tall ? r0 + j : r0 + i, c = tall ? c0 + i : c0 + j;
        float v = 0.f;
        if (r < m && c < n) v = (float)((double)(float)g[tall ? (long)c * m + r : (long)r * n + c] * inv);
        t[tall ? j : i][tall ? i : j] = v;
    }
    __syncthreads();
    // 2 fragments each way, 4 x 64 lanes of 8 values
    const int part = threadIdx.x >> 6, lane = threadIdx.x & 63, k0 = 16 * (part & 1) + 8 * (lane >> 5), row = lane & 31;
    half8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; i++) { f16 a, b; split(part < 2 ? t[row][k0 + i] : t[k0 + i][row], a, b); hi[i] = a; lo[i] = b; }
    const int KX = gridDim.x * 2, KT = gridDim.y * 2;           // 16-wide k blocks of X and of X^T
    f16* to = part < 2 ? X + blockIdx.z * sx + frag_at(blockIdx.y, 2 * blockIdx.x + part, KX)
                       : XT + blockIdx.z * sx + frag_at(blockIdx.x, 2 * blockIdx.y + (part - 2), KT);
    *(half8*)(to + lane * 8) = hi;
    *(half8*)(to + FRAG + lane * 8) = lo;
}

// ---- D = beta S + gamma P Q^T, tile by tile --------------------------------------------------------------------------------------
enum { GRAM, POLY, NEXT, LAST };            // A;  B;  X and X^T;  the result
struct Product {
    const f16* P; const f16* Q; long sp, sq;        // operands, and from one matrix to the next (halves)
    const f16* S; long ss;                          // the summand, laid out like the (transposed) result; null: none
    f16* D; f16* DT; long sd, sdt;                  // D^T as an operand, D as an operand (null: not wanted)
    int M, N, K;                                    // padded
    float beta, gamma;
    int m, n, tall, dtype;                          // LAST
    int count;
};
template <int MODE>
__global__ void __launch_bounds__(256) product_kernel(Product p, Mats q) {
    __shared__ uint32_t turn[4][32][33];
    const int tn = p.N / TILE, tm = p.M / TILE, per = (MODE == GRAM || MODE == POLY) ? tm * (tm + 1) / 2 : tm * tn;
    const int z = blockIdx.x / per;
    int t = blockIdx.x - z * per, I, J;
    if constexpr (MODE == GRAM || MODE == POLY) { J = 0; while ((J + 1) * (J + 2) / 2 <= t) J++; I = t - J * (J + 1) / 2; }
    else { I = t / tn; J = t - I * tn; }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int rb = 2 * I + (wave >> 1), cb = 2 * J + (wave & 1), KB = p.K / 16;
    const f16* P = p.P + z * p.sp + frag_at(rb, 0, KB) + lane * 8;
    const f16* Q = p.Q + z * p.sq + frag_at(cb, 0, KB) + lane * 8;
    float16v acc = {};
#pragma unroll 4
    for (int kb = 0; kb < KB; kb++) {
        const half8 ph = *(const half8*)(P + (long)kb * 2 * FRAG), pl = *(const half8*)(P + (long)kb * 2 * FRAG + FRAG);
        const half8 qh = *(const half8*)(Q + (long)kb * 2 * FRAG), ql = *(const half8*)(Q + (long)kb * 2 * FRAG + FRAG);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc, 0, 0, 0);
    }
    // lane: column c = lane % 32 of D, rows 8 g + 4 (lane / 32) + 0..3.  As an operand (D^T): row c, 4 consecutive k
    const int c = lane & 31, h = lane >> 5, MB = p.M / 16;
    float v[16];
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const long at = frag_at(cb, 2 * rb + (g >> 1), MB) + (c + 32 * (g & 1)) * 8 + 4 * h;
        half4 sh = {}, sl = {};
        if (p.S) { sh = *(const half4*)(p.S + z * p.ss + at); sl = *(const half4*)(p.S + z * p.ss + at + FRAG); }
        half4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float s = (float)sh[i] + (float)sl[i];
            const float d = fmaf(p.gamma, acc[4 * g + i], p.beta * s);
            f16 a, b; split(d, a, b); hi[i] = a; lo[i] = b;
            v[4 * g + i] = d;
        }
        if constexpr (MODE != LAST) { *(half4*)(p.D + z * p.sd + at) = hi; *(half4*)(p.D + z * p.sd + at + FRAG) = lo; }
    }
    if constexpr (MODE == LAST) {
        // D is n x m
#pragma unroll
        for (int g = 0; g < 16; g++) {
            const int r = 32 * rb + 8 * (g >> 2) + 4 * h + (g & 3), col = 32 * cb + c;
            if (r < p.n && col < p.m) {
                const long at = p.tall ? (long)r * p.m + col : (long)col * p.n + r;
                const float d = v[g] * UNSCALE;
                if (p.dtype == BL_F32) ((float*)q.out[z])[at] = d;
                else if (p.dtype == BL_F16) ((f16*)q.out[z])[at] = (f16)d;
                else ((bf16*)q.out[z])[at] = (bf16)d;
            }
        }
    } else if (MODE == NEXT || I != J) {
        // D itself as an operand: through LDS, a wave's 32 x 32 its own
#pragma unroll
        for (int g = 0; g < 16; g++) {
            f16 a, b; split(v[g], a, b);
            turn[wave][8 * (g >> 2) + 4 * h + (g & 3)][c] = (uint32_t)__builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront"); __builtin_amdgcn_wave_barrier();
        const int NB = p.N / 16;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            half8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t w = turn[wave][c][16 * s + 8 * h + i];
                hi[i] = __builtin_bit_cast(f16, (uint16_t)w); lo[i] = __builtin_bit_cast(f16, (uint16_t)(w >> 16));
            }
            f16* to = p.DT + z * p.sdt + frag_at(rb, 2 * cb + s, NB) + lane * 8;
            *(half8*)to = hi;
            *(half8*)(to + FRAG) = lo;
        }
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------
struct Plan { long x, a, norm; long total(int count) const { return count * (3 * x + 2 * a) * (long)sizeof(f16) + norm; } };
Plan plan_of(int m, int n) {                // halves of one matrix: X (and each X^T), A (and B); bytes of the norms' parts
    const long mp = up(m), np = up(n);
    return {2 * mp * np, 2 * mp * mp, MANY * PARTS * (long)sizeof(double)};
}
template <int MODE> void multiply(const Product& p, const Mats& q, hipStream_t s) {
    const int tm = p.M / TILE, tn = p.N / TILE;
    const long per = (MODE == GRAM || MODE == POLY) ? (long)tm * (tm + 1) / 2 : (long)tm * tn;
    hipLaunchKernelGGL((product_kernel<MODE>), dim3((unsigned)(per * p.count)), dim3(256), 0, s, p, q);
}

}  // namespace

extern "C" {

long bl_orthogonalize_workspace(int count, int rows, int cols) {
    if (count <= 0 || rows <= 0 || cols <= 0 || rows > BL_ORTHO_MAX || cols > BL_ORTHO_MAX) return 0;
    const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    return plan_of(m, n).total(count < MANY ? count : MANY);
}

int bl_orthogonalize(const void* const* host_in, void* const* host_out, int count, int dtype, int rows, int cols, int steps, float eps,
                     void* workspace, bl_stream_t stream) {
    if (!host_in || !host_out || !workspace || count <= 0 || rows <= 0 || cols <= 0 || steps <= 0 || !(eps >= 0.f)) return BL_EINVAL;
    if (dtype != BL_F32 && dtype != BL_F16 && dtype != BL_BF16) return BL_EINVAL;
    if (rows > BL_ORTHO_MAX || cols > BL_ORTHO_MAX) return BL_ETOOBIG;
    for (int i = 0; i < count; i++) if (!host_in[i] || !host_out[i]) return BL_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    const int tall = rows > cols, m = tall ? cols : rows, n = tall ? rows : cols, mp = up(m), np = up(n);
    const Plan plan = plan_of(m, n);
    for (int i0 = 0; i0 < count; i0 += MANY) {
        const int c = count - i0 < MANY ? count - i0 : MANY;
        Mats q{};
        for (int i = 0; i < c; i++) { q.in[i] = host_in[i0 + i]; q.out[i] = host_out[i0 + i]; }
        double* parts = (double*)workspace;
        f16* X = (f16*)((char*)workspace + plan.norm);
        f16* XT[2] = {X + c * plan.x, X + 2 * c * plan.x};
        f16* A = X + 3 * c * plan.x;
        f16* B = A + c * plan.a;
        const dim3 ng(PARTS, c), lg(np / 32, mp / 32, c);
        if (dtype == BL_F32) {
            hipLaunchKernelGGL((norm_parts_kernel<float>), ng, dim3(256), 0, s, q, (long)m * n, parts);
            hipLaunchKernelGGL((lay_out_kernel<float>), lg, dim3(256), 0, s, q, m, n, tall, eps, parts, X, XT[0], plan.x);
        } else if (dtype == BL_F16) {
            hipLaunchKernelGGL((norm_parts_kernel<f16>), ng, dim3(256), 0, s, q, (long)m * n, parts);
            hipLaunchKernelGGL((lay_out_kernel<f16>), lg, dim3(256), 0, s, q, m, n, tall, eps, parts, X, XT[0], plan.x);
        } else {
            hipLaunchKernelGGL((norm_parts_kernel<bf16>), ng, dim3(256), 0, s, q, (long)m * n, parts);
            hipLaunchKernelGGL((lay_out_kernel<bf16>), lg, dim3(256), 0, s, q, m, n, tall, eps, parts, X, XT[0], plan.x);
        }
        for (int it = 0; it < steps; it++) {
            f16 *from = XT[it & 1], *to = XT[(it & 1) ^ 1];
            // acc carries SCALE^2
            multiply<GRAM>(Product{X, X, plan.x, plan.x, nullptr, 0, A, A, plan.a, plan.a, mp, mp, np, 0.f, UNSCALE, 0, 0, 0, 0, c}, q, s);
            multiply<POLY>(Product{A, A, plan.a, plan.a, A, plan.a, B, B, plan.a, plan.a, mp, mp, mp, NS_B, NS_C * UNSCALE, 0, 0, 0, 0, c}, q, s);
            // X^T B: n x m, whose transpose a X + B X is written over X (nobody reads X here but the lane that replaces it)
            const Product next{from, B, plan.x, plan.a, X, plan.x, X, to, plan.x, plan.x, np, mp, mp, NS_A, UNSCALE, m, n, tall, dtype, c};
            if (it + 1 < steps) multiply<NEXT>(next, q, s);
            else multiply<LAST>(next, q, s);
        }
        if (const int rc = check_launch()) return rc;
    }
    return BL_OK;
}

}  // extern "C"
