// bl_ortho.hip -- Newton-Schulz orthogonalisation of update matrices, for the learner's hidden weights.
//
//     X = G / (|G|_F + eps);   `steps` times:  A = X X^T,  B = b A + c A^2,  X = a X + B X        (on the side with fewer rows, m <= n)
//
// takes every singular value s to a s + b s^3 + c s^5 and again, i.e. towards 1.  The iteration multiplies what is small by up to 3.4 a
// step: with f16 or bf16 operands the rounding of the large directions drowns the small ones of a low-rank gradient (3.7 % / 30 % of the
// result on rank 8 + 1 % noise).  So every operand (beyond few rows, below) is a pair of f16 numbers hi + lo (22 bits and lo's sign), a product is hi hi + hi lo +
// lo hi on v_mfma_f32_32x32x16_f16 with f32 sums (the dropped lo lo is up to 2^-22 of the product, 2^-24 typically: what f32 rounding costs), a third
// of the f16 matrix rate where the f32 MFMA has a sixteenth.  Operands carry a factor 2^13: entries of X and B stay below 3 (the quintic maps [0, 1.21] into
// itself), so hi < 2^15, and lo keeps its bits above f16's smallest steps down to entries of 2^-14.
//
// Operands lie in the workspace as MFMA fragments: 32 rows x 16 k, lane = row + 32 (k / 8), 8 consecutive k per lane, hi then lo -- a
// wave's load is one contiguous KiB and both operands of P Q^T use the same layout.  The accumulator holds 4 consecutive rows of D per
// lane, which are 4 consecutive k of D^T as an operand: writing D^T costs nothing, writing D as well goes through LDS once per tile.
// A and A^2 are symmetric: only the tiles on and above the diagonal are computed.
#include <type_traits>
#include "bl_train.h"
#include "bl_host.h"

#pragma clang fp contract(off)

using namespace bltrain;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float SCALE = 8192.f, UNSCALE = 1.f / 8192.f;
constexpr int PAD = 128, MANY = 32, PARTS = 64;
constexpr int FRAG = 512;                   // halves of one fragment, hi or lo

struct Mats { const void* in[MANY]; void* out[MANY]; };

int up(int v) { return v <= 64 ? 64 : (v + PAD - 1) / PAD * PAD; }        // whole tiles of 64, or of 128

// halves from one fragment pair to the next are 2 FRAG; (rb, kb): 32 rows, 16 k
__device__ __forceinline__ long frag_at(int rb, int kb, int KB) { return ((long)rb * KB + kb) * (2 * FRAG); }

__device__ __forceinline__ void split(float v, f16& hi, f16& lo) { hi = (f16)v; lo = (f16)(v - (float)hi); }

// 1 / (|G| + eps); 0 for a zero matrix without an eps, whose result is zeros too
__device__ __forceinline__ double reciprocal(double square, float eps) { const double d = sqrt(square) + (double)eps; return d == 0. ? 0. : 1. / d; }

// ---- |G|^2 in parts, in f64: neither 2^100 nor 2^-100 as a loss scale overflows or vanishes ----
template <typename T> __global__ void __launch_bounds__(256) norm_parts_kernel(Mats q, long total, double* parts) {
    __shared__ double lds[4];
    const T* g = (const T*)q.in[blockIdx.y];
    constexpr int V = 16 / sizeof(T);
    const bool wide = (reinterpret_cast<uintptr_t>(g) & 15) == 0;
    const long nv = wide ? total / V : 0, i0 = nv * blockIdx.x / PARTS, i1 = nv * (blockIdx.x + 1) / PARTS;
    double s = 0.;
    for (long i = i0 + threadIdx.x; i < i1; i += 256) {
        float v[V];
        load<T, V>(g + i * V, v);
#pragma unroll
        for (int k = 0; k < V; k++) s += (double)v[k] * (double)v[k];
    }
    const long rest = total - nv * V, j0 = nv * V + rest * blockIdx.x / PARTS, j1 = nv * V + rest * (blockIdx.x + 1) / PARTS;
    for (long i = j0 + threadIdx.x; i < j1; i += 256) { const double v = (double)(float)g[i]; s += v * v; }
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
    double ss = parts[blockIdx.z * PARTS + (threadIdx.x & 63)];
    for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o);
    const double inv = (double)SCALE * reciprocal(ss, eps);
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
// The summand of a wave's 32 x 32 of D, at fragment row rb and fragment column cb.  A lane holds column c = lane % 32 of D, rows
// 8 g + 4 (lane / 32) + 0..3: as an operand (D^T), row c and 4 consecutive k
struct Summand { half4 hi[4], lo[4]; };
__device__ __forceinline__ long place(int rb, int cb, int g, int MB) {
    const int lane = threadIdx.x & 63;
    return frag_at(cb, 2 * rb + (g >> 1), MB) + ((lane & 31) + 32 * (g & 1)) * 8 + 4 * (lane >> 5);
}
__device__ __forceinline__ void fetch_summand(Summand& s, const f16* S, int rb, int cb, int MB) {
#pragma unroll
    for (int g = 0; g < 4; g++) { const f16* at = S + place(rb, cb, g, MB); s.hi[g] = *(const half4*)at; s.lo[g] = *(const half4*)(at + FRAG); }
}

template <typename T> __device__ __forceinline__ void store_tall(T* out, const float (&v)[16], int r0, int col, int n, int m) {
#pragma unroll
    for (int g = 0; g < 16; g++) { const int r = r0 + 8 * (g >> 2) + (g & 3); if (r < n && col < m) out[(long)r * m + col] = (T)(v[g] * UNSCALE); }
}
template <typename T> __device__ __forceinline__ void store_wide(T* out, const float (*t)[33], int r0, int c0, int n, int m) {
    const int lane = threadIdx.x & 63;
    float o[16];
#pragma unroll
    for (int i = 0; i < 16; i++) o[i] = t[2 * i + (lane >> 5)][lane & 31];
#pragma unroll
    for (int i = 0; i < 16; i++) {              // two rows of the result at a time, 32 consecutive entries of each
        const int c = c0 + 2 * i + (lane >> 5), r = r0 + (lane & 31);
        if (r < n && c < m) out[(long)c * n + r] = (T)(o[i] * UNSCALE);
    }
}
// a wave's 32 x 32 of D, which is n x m, as the result: as it is where the input was tall, else transposed, through LDS
__device__ __forceinline__ void store_result(const Product& p, void* out, const float (&v)[16], int rb, int cb, uint32_t (*turn)[33]) {
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    if (p.tall) {
        if (p.dtype == BL_F32) store_tall((float*)out, v, 32 * rb + 4 * h, 32 * cb + c, p.n, p.m);
        else if (p.dtype == BL_F16) store_tall((f16*)out, v, 32 * rb + 4 * h, 32 * cb + c, p.n, p.m);
        else store_tall((bf16*)out, v, 32 * rb + 4 * h, 32 * cb + c, p.n, p.m);
        return;
    }
    float (*t)[33] = (float (*)[33])turn;
#pragma unroll
    for (int g = 0; g < 16; g++) t[c][8 * (g >> 2) + 4 * h + (g & 3)] = v[g];
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront"); __builtin_amdgcn_wave_barrier();
    if (p.dtype == BL_F32) store_wide((float*)out, t, 32 * rb, 32 * cb, p.n, p.m);
    else if (p.dtype == BL_F16) store_wide((f16*)out, t, 32 * rb, 32 * cb, p.n, p.m);
    else store_wide((bf16*)out, t, 32 * rb, 32 * cb, p.n, p.m);
}

// mirror: D is wanted as an operand too
template <int MODE>
__device__ __forceinline__ void epilogue(const Product& p, const Mats& q, const float16v& acc, const Summand& sum, int z, int rb, int cb, bool mirror, uint32_t (*turn)[33]) {
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5, MB = p.M / 16;
    float v[16];
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const long at = place(rb, cb, g, MB);
        half4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float d = MODE == GRAM ? p.gamma * acc[4 * g + i] : fmaf(p.gamma, acc[4 * g + i], p.beta * ((float)sum.hi[g][i] + (float)sum.lo[g][i]));
            f16 a, b; split(d, a, b); hi[i] = a; lo[i] = b;
            v[4 * g + i] = d;
        }
        if constexpr (MODE != LAST) { *(half4*)(p.D + z * p.sd + at) = hi; *(half4*)(p.D + z * p.sd + at + FRAG) = lo; }
    }
    if constexpr (MODE == LAST) {
        store_result(p, q.out[z], v, rb, cb, turn);
    } else if (mirror) {
        // D itself as an operand: through LDS, a wave's 32 x 32 its own (its DS operations go in order)
#pragma unroll
        for (int g = 0; g < 16; g++) {
            f16 a, b; split(v[g], a, b);
            turn[8 * (g >> 2) + 4 * h + (g & 3)][c] = (uint32_t)__builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront"); __builtin_amdgcn_wave_barrier();
        const int NB = p.N / 16;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            half8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t w = turn[c][16 * s + 8 * h + i];
                hi[i] = __builtin_bit_cast(f16, (uint16_t)w); lo[i] = __builtin_bit_cast(f16, (uint16_t)(w >> 16));
            }
            f16* to = p.DT + z * p.sdt + frag_at(rb, 2 * cb + s, NB) + lane * 8;
            *(half8*)to = hi;
            *(half8*)(to + FRAG) = lo;
        }
    }
}

// Which tile of which matrix a workgroup has.  Consecutive workgroups go to the 8 XCDs in turn: each of them gets consecutive tiles, whose
// operands its L2 then holds
struct Tile { int z, I, J; };
template <bool SYM, int ROWS, int COLS> __host__ __device__ __forceinline__ int tiles_in(int M, int N) {
    const int tm = M / ROWS, tn = N / COLS;
    if constexpr (!SYM) return tm * tn;
    else if constexpr (ROWS == COLS) return tn * (tn + 1) / 2;
    else { static_assert(ROWS == 2 * COLS, "two columns of tiles to a row of them"); return tm * (tm + 1); }
}
template <bool SYM, int ROWS, int COLS> __device__ __forceinline__ Tile tile_of(const Product& p) {
    const int per = tiles_in<SYM, ROWS, COLS>(p.M, p.N);
    const int total = per * p.count, share = total / 8, extra = total % 8, xcd = blockIdx.x % 8;
    const int id = xcd * share + (xcd < extra ? xcd : extra) + blockIdx.x / 8;
    Tile t;
    t.z = id / per;
    const int i = id - t.z * per;
    if constexpr (SYM) {                        // the tiles on and above the diagonal, (double) column by column
        constexpr int F = ROWS / COLS;          // column j of F columns has j + 1 tiles in each
        int j = (int)((sqrtf(8.f * (i / F) + 1.f) - 1.f) * .5f);
        while (F * j * (j + 1) / 2 > i) j--;
        while (F * (j + 1) * (j + 2) / 2 <= i) j++;
        const int in = i - F * j * (j + 1) / 2;
        t.J = F * j + in / (j + 1); t.I = in % (j + 1);
    } else { const int tn = p.N / COLS; t.I = i / tn; t.J = i - t.I * tn; }
    return t;
}

// 16 k of 32 F rows of P and 64 rows of Q
template <int F> struct Frags { half8 ph[F], pl[F], qh[2], ql[2]; };
template <int F> __device__ __forceinline__ void multiply_add(const Frags<F>& f, float16v (&acc)[F][2]) {
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.pl[i], f.qh[j], acc[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ph[i], f.ql[j], acc[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ph[i], f.qh[j], acc[i][j], 0, 0, 0);
}

// Few tiles: a workgroup of four waves computes 64 x 64 of D, every wave all of it over a quarter of K, straight from memory into
// registers; the quarters are added through LDS in a fixed order.  A wave multiplies 12 times per 8 KiB it loads and waits for nobody.
// Four matrices of 512: 7 to 10 us a product on 144 or 256 workgroups, of which a launch that does nothing takes 2.4, adding the quarters 1.1, the
// loop 4.5 -- 256 KiB per workgroup through its CU's L1 is 1.7 at its full 64 bytes a clock, and the operands were written by other XCDs.
template <int MODE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 2))) product_64_kernel(Product p, Mats q) {
    extern __shared__ __align__(16) char smem[];
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    constexpr int D = 2;                                    // blocks of 16 k on their way (1, 2, 3, 4: 4 x 128 x 128 86, 88, 95, 101 us for 5 steps, 4 x 512 x 512 155, 153, 159, 158)
    const Tile t = tile_of<SYM, 64, 64>(p);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, KB = p.K / 16, n = KB / 4;
    const int rb = 2 * t.I + (wave >> 1), cb = 2 * t.J + (wave & 1);        // this wave's 32 x 32 in the end
    Summand sum;
    if constexpr (MODE != GRAM) fetch_summand(sum, p.S + t.z * p.ss, rb, cb, p.M / 16);
    // a row of fragments is contiguous; what is asked for beyond it is not loaded and reads as zero
    const int bytes = KB * 4 * FRAG;
    const f16* P = p.P + t.z * p.sp + frag_at(2 * t.I, 0, KB);
    const f16* Q = p.Q + t.z * p.sq + frag_at(2 * t.J, 0, KB);
    __amdgpu_buffer_rsrc_t rows[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        rows[i] = __builtin_amdgcn_make_buffer_rsrc((void*)((i < 2 ? P : Q) + (i & 1) * frag_at(1, 0, KB)), 0, bytes, 0x00020000);
    auto fetch = [&](Frags<2>& f, int kb) {                    // kb of this wave's n
        const int at = kb < n ? ((wave * n + kb) * 4 * FRAG + lane * 16) : bytes;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            f.ph[i] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(rows[i], at, 0, 0));
            f.pl[i] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(rows[i], at + 2 * FRAG, 0, 0));
            f.qh[i] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(rows[2 + i], at, 0, 0));
            f.ql[i] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(rows[2 + i], at + 2 * FRAG, 0, 0));
        }
    };
    Frags<2> f[D];
#pragma unroll
    for (int d = 0; d < D; d++) fetch(f[d], d);
    float16v acc[2][2] = {};
    for (int k = 0; k < n; k += D) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            multiply_add(f[d], acc);
            fetch(f[d], k + d + D);
        }
    }
    // lds[tile][wave][value][lane]: every wave leaves the three tiles that are not its own
    float* lds = (float*)smem;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i != wave)
#pragma unroll
            for (int v = 0; v < 16; v += 4)
                *(float4*)(lds + ((i * 4 + wave) * 4 + v / 4) * 256 + lane * 4) = make_float4(acc[i >> 1][i & 1][v], acc[i >> 1][i & 1][v + 1], acc[i >> 1][i & 1][v + 2], acc[i >> 1][i & 1][v + 3]);
    __syncthreads();
    float16v own = wave == 0 ? acc[0][0] : wave == 1 ? acc[0][1] : wave == 2 ? acc[1][0] : acc[1][1], total = {};
#pragma unroll
    for (int w = 0; w < 4; w++)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
            float4 o = make_float4(own[v], own[v + 1], own[v + 2], own[v + 3]);
            if (w != wave) o = *(const float4*)(lds + ((wave * 4 + w) * 4 + v / 4) * 256 + lane * 4);
            total[v] += o.x; total[v + 1] += o.y; total[v + 2] += o.z; total[v + 3] += o.w;
        }
    __syncthreads();
    epilogue<MODE>(p, q, total, sum, t.z, rb, cb, !SYM || t.I != t.J, (uint32_t (*)[33])(smem + wave * 32 * 33 * 4));
}

// Many tiles: a workgroup of four waves computes 64 F x 128 of D, each wave 32 F x 64.  16 k at a time go through LDS, which holds four such
// stages: while stage s is multiplied, the fragments of stage s + 1 are read, stage s + 3 is written from registers and stage s + 7
// sets out for them -- one barrier per stage, nothing to wait for behind it, and four stages of products for a load to arrive.
// Stages beyond the last are loaded from the last again and never used, so that a stage is one straight run of instructions, dealt
// out between the products by the scheduling groups.  F = 4 takes 72 KiB of LDS traffic to 768 cycles of products (F = 2: 48 to 384, which is
// all that LDS has).  Eight matrices of 1024: 59 us for B X (51.5 GFLOP in the three products, 870 TFLOP/s where a large library f16 product reaches
// 1314), 47 for X X^T and 49 for A A on 160 workgroups: what they lack is the other 96 CUs.  The matrix units are busy 56 % of the cycles.
template <int MODE, int F>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) product_wide_kernel(Product p, Mats q) {
    extern __shared__ __align__(16) char smem[];
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    constexpr int NL = F + 2, STAGE = NL * 2048;            // 16-byte loads of a thread per stage; halves
    f16* lds = (f16*)smem;
    const Tile t = tile_of<SYM, 64 * F, 128>(p);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave >> 1, wn = wave & 1;
    const int KB = p.K / 16;
    // load i: rows of fragments 2 i and 2 i + 1, half of the workgroup each
    const long mine = frag_at(threadIdx.x >> 7, 0, KB) + (threadIdx.x & 127) * 8;
    const f16* P = p.P + t.z * p.sp + frag_at(2 * F * t.I, 0, KB) + mine;
    const f16* Q = p.Q + t.z * p.sq + frag_at(4 * t.J, 0, KB) + mine;
    half8 r[4][NL];
    auto fetch = [&](half8 (&r)[NL], int s) {
        const long at = (long)(s < KB ? s : KB - 1) * 2 * FRAG;
#pragma unroll
        for (int i = 0; i < NL; i++) r[i] = *(const half8*)((i < F ? P + frag_at(2 * i, 0, KB) : Q + frag_at(2 * (i - F), 0, KB)) + at);
    };
    auto put = [&](const half8 (&r)[NL], int slot) {
#pragma unroll
        for (int i = 0; i < NL; i++) *(half8*)(lds + slot * STAGE + i * 2048 + threadIdx.x * 8) = r[i];
    };
    auto read = [&](Frags<F>& f, int slot) {
        const f16* ps = lds + slot * STAGE + F * wm * 2 * FRAG + lane * 8;
        const f16* qs = lds + slot * STAGE + (2 * F + 2 * wn) * 2 * FRAG + lane * 8;
#pragma unroll
        for (int i = 0; i < F; i++) { f.ph[i] = *(const half8*)(ps + i * 2 * FRAG); f.pl[i] = *(const half8*)(ps + i * 2 * FRAG + FRAG); }
#pragma unroll
        for (int i = 0; i < 2; i++) { f.qh[i] = *(const half8*)(qs + i * 2 * FRAG); f.ql[i] = *(const half8*)(qs + i * 2 * FRAG + FRAG); }
    };
#pragma unroll
    for (int s = 0; s < 4; s++) fetch(r[s], s);
#pragma unroll
    for (int s = 0; s < 3; s++) { put(r[s], s); fetch(r[s], s + 4); }
    float16v acc[F][2] = {};
    Frags<F> f[2];
    __syncthreads();
    read(f[0], 0);
    auto stage = [&](auto slot_, int s) {                   // stage s, in slot s % 4
        constexpr int slot = decltype(slot_)::value, next = (slot + 1) % 4, free = (slot + 3) % 4;
        __builtin_amdgcn_sched_barrier(0);
        read(f[(slot + 1) & 1], next);
        put(r[free], free);
        fetch(r[free], s + 7);
        multiply_add<F>(f[slot & 1], acc);
        // what LDS does comes first, so that the barrier finds it done; the loads go under the last products
#pragma unroll
        for (int i = 0; i < NL; i++) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if constexpr (F == 4) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < NL; i++) { __builtin_amdgcn_sched_group_barrier(0x020, 1, 0); __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); }
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
    };
    for (int s = 0; s < KB; s += 4) {                       // (K is a multiple of 128)
        stage(std::integral_constant<int, 0>(), s);
        stage(std::integral_constant<int, 1>(), s + 1);
        stage(std::integral_constant<int, 2>(), s + 2);
        stage(std::integral_constant<int, 3>(), s + 3);
    }
#pragma unroll
    for (int i = 0; i < F; i++) {
        const int rb = 2 * F * t.I + F * wm + i;
        Summand sum[2];
        if constexpr (MODE != GRAM) {
#pragma unroll
            for (int j = 0; j < 2; j++) fetch_summand(sum[j], p.S + t.z * p.ss, rb, 4 * t.J + 2 * wn + j, p.M / 16);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int cb = 4 * t.J + 2 * wn + j;
            // D^T of this 32 x 32 is stored in any case; D unless the tile that holds (cb, rb) is computed and stores it
            const bool mirror = !SYM || rb / 4 < (cb / (2 * F)) * (F / 2);
            epilogue<MODE>(p, q, acc[i][j], sum[j], t.z, rb, cb, mirror, (uint32_t (*)[33])(smem + wave * 32 * 33 * 4));
        }
    }
}

// ---- m <= 64 and n <= 64 NB <= 128 (mostly m > 32): one workgroup takes a matrix through all of it in LDS ------------------------------------------
// 15 dependent products of a few hundred cycles each: launches (3 to 5 us apiece) would be nearly all of the time.  Here products cost next
// to nothing, so operands are three f16 numbers (33 bits) and a product six: a small matrix is often nearly singular, and sums this
// short leave f32 so little error of their own that 22 bits would show.
constexpr int TRIPLE = 3 * FRAG;
__device__ __forceinline__ int triple_at(int rb, int kb, int KB) { return (rb * KB + kb) * TRIPLE; }
__device__ __forceinline__ void split(float v, f16 (&o)[3]) {
    o[0] = (f16)v;
    const float r = v - (float)o[0];
    o[1] = (f16)r;
    o[2] = (f16)(r - (float)o[1]);
}
template <typename T, int NB>
__global__ void __launch_bounds__(256) ortho_small_kernel(Mats q, Product p, int steps, float eps) {
    extern __shared__ __align__(16) char smem[];
    __shared__ double sums[4];
    constexpr int NP = 64 * NB, EACH = 64 * NP / 256;
    f16 *X = (f16*)smem, *XT = X + 3 * 64 * NP, *A = XT + 3 * 64 * NP, *B = A + 3 * 64 * 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5, m = p.m, n = p.n;
    const T* g = (const T*)q.in[blockIdx.x];
    // element (row, k) of an operand with KB blocks of 16 k
    auto set = [&](f16* to, int row, int k, int KB, const f16 (&s)[3]) {
        to += triple_at(row >> 5, k >> 4, KB) + ((row & 31) + 32 * ((k >> 3) & 1)) * 8 + (k & 7);
#pragma unroll
        for (int i = 0; i < 3; i++) to[i * FRAG] = s[i];
    };
    T raw[EACH];                                // (clamped addresses and no branch: all of them on their way at once)
    float v[EACH];
    double ss = 0.;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int e = threadIdx.x + 256 * i, r = min(p.tall ? e % 64 : e / NP, m - 1), col = min(p.tall ? e / 64 : e % NP, n - 1);
        raw[i] = g[p.tall ? col * m + r : r * n + col];
    }
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int e = threadIdx.x + 256 * i, r = p.tall ? e % 64 : e / NP, col = p.tall ? e / 64 : e % NP;
        v[i] = r < m && col < n ? (float)raw[i] : 0.f;
        ss += (double)v[i] * (double)v[i];
    }
    for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o);
    if (lane == 0) sums[wave] = ss;
    __syncthreads();
    const double inv = (double)SCALE * reciprocal((sums[0] + sums[1]) + (sums[2] + sums[3]), eps);
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int e = threadIdx.x + 256 * i, r = p.tall ? e % 64 : e / NP, col = p.tall ? e / 64 : e % NP;
        f16 s[3];
        split((float)((double)v[i] * inv), s);
        set(X, r, col, NP / 16, s);
        set(XT, col, r, 4, s);
    }
    __syncthreads();
    // 32 x 32 of P Q^T at fragment row rb and column cb; what is padding of K alone is left out
    auto product = [&](const f16* P, const f16* Q, int rb, int cb, int KB, int k) {
        float16v acc = {};
        for (int kb = 0; kb < (k + 15) / 16; kb++) {
            half8 a[3], b[3];
#pragma unroll
            for (int i = 0; i < 3; i++) {
                a[i] = *(const half8*)(P + triple_at(rb, kb, KB) + i * FRAG + lane * 8);
                b[i] = *(const half8*)(Q + triple_at(cb, kb, KB) + i * FRAG + lane * 8);
            }
            // the smallest first; lo mid, mid lo and lo lo are under 2^-33 of the product
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[2], b[0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[2], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], acc, 0, 0, 0);
        }
        return acc;
    };
    // a lane's 4 consecutive k of D^T, group `k`
    auto spot = [&](int rb, int cb, int k, int MB) { return triple_at(cb, 2 * rb + (k >> 1), MB) + (c + 32 * (k & 1)) * 8 + 4 * h; };
    // beta s + gamma acc into D^T, its values kept.  The summands are the same lane's values of the product before, in f32
    auto finish = [&](float16v& acc, const float16v& s, f16* D, int rb, int cb, int MB, float beta, float gamma) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            half4 o[3];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                acc[4 * k + i] = fmaf(gamma, acc[4 * k + i], beta * s[4 * k + i]);
                f16 t[3];
                split(acc[4 * k + i], t);
                o[0][i] = t[0]; o[1][i] = t[1]; o[2][i] = t[2];
            }
#pragma unroll
            for (int i = 0; i < 3; i++) *(half4*)(D + spot(rb, cb, k, MB) + i * FRAG) = o[i];
        }
    };
    const int rb = wave >> 1, cb = wave & 1;
    float16v x[NB];                             // this lane's entries of X^T
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const f16* from = X + spot(rb + 2 * j, cb, k, NP / 16);
            const half4 hi = *(const half4*)from, mid = *(const half4*)(from + FRAG), lo = *(const half4*)(from + 2 * FRAG);
#pragma unroll
            for (int i = 0; i < 4; i++) x[j][4 * k + i] = (float)hi[i] + ((float)mid[i] + (float)lo[i]);
        }
    for (int it = 0; it < steps; it++) {
        float16v a = product(X, X, rb, cb, NP / 16, n);
        finish(a, a, A, rb, cb, 4, 0.f, UNSCALE);
        __syncthreads();
        float16v b = product(A, A, rb, cb, 4, m);
        finish(b, a, B, rb, cb, 4, NS_B, NS_C * UNSCALE);
        __syncthreads();
        // X^T B, NP x 64: blocks rb + 2 j of its rows; X is each lane's own to replace, X^T only when every wave has read it
        float16v next[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) next[j] = product(XT, B, rb + 2 * j, cb, 4, m);
#pragma unroll
        for (int j = 0; j < NB; j++) { finish(next[j], x[j], X, rb + 2 * j, cb, NP / 16, NS_A, UNSCALE); x[j] = next[j]; }
        __syncthreads();
        if (it + 1 == steps) {                  // (A and B are free: the way to the result)
#pragma unroll
            for (int j = 0; j < NB; j++) {
                float o[16];
#pragma unroll
                for (int i = 0; i < 16; i++) o[i] = next[j][i];
                store_result(p, q.out[blockIdx.x], o, rb + 2 * j, cb, (uint32_t (*)[33])((char*)A + wave * 32 * 33 * 4));
            }
            break;
        }
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                f16 s[3];
                split(next[j][i], s);
                set(XT, 32 * (rb + 2 * j) + 8 * (i >> 2) + 4 * h + (i & 3), 32 * cb + c, 4, s);
            }
        __syncthreads();
    }
}

// ---- few rows: the iteration on the m x m side, in f64 --------------------------------------------------------------------------------
// Every X of the iteration is Q G with Q a polynomial of G G^T, so that with A = X X^T the steps are  P = a I + b A + c A^2,  Q = P Q,  A = P A P
// and G comes in twice: for its Gram matrix and for Q G.  Sums over few rows leave f32 so little error of its own that operands of 22 bits would
// show (against the f32 form's: 8 x 129 2.7 times, 2 x 500 likewise, 32 x 200 1.55, 64 x 300 1.04), and 33 bits with f32 sums still do (8 x 8 1.75).  m x m
// products on v_mfma_f64_16x16x4_f64 are few, and what is left is the result's own rounding.  A column's sums over k may be taken
// in any order, so a lane loads 4 consecutive k; one fragment is both operands of a Gram product.
// Where it is used: up to 32 rows at any width, up to 64 beyond 128 wide.  us, beside the kernels above: 4 x 16 x 16 10.9 (19.2), 4 x 32 x 32 18.3 (21.2),
// 4 x 8 x 400 15 (90), 4 x 32 x 200 27 (84), 4 x 64 x 300 85 (88), 64 x 1000 86 (102), 64 x 16384 133 (515); but 4 x 48 x 48 38 (23), 4 x 64 x 64 69 (25), 4 x 64 x 128 78 (41),
// where three f16 numbers are as exact as f32.  The steps' f64 products bound it: 69 of 85 us at 64 x 300.
// Up to 6 steps: a direction that G does not have is in A with its rounding, 2^-53 and of either sign, which a step multiplies by 3.4445^2, and in Q with 3.4445 a step:
// 41 times a step in Q G.  Ones of 20 x 24 are 7e-9, 4e-8, 2e-6, 6e-5 off behind 5, 6, 7, 8 steps (the f32 form 3e-6) and diverge behind 12; X X^T has no such
// direction, and the kernels above take any number of steps.
typedef double d4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ d4 mfma(double x, double y, d4 acc) { return __builtin_amdgcn_mfma_f64_16x16x4f64(x, y, acc, 0, 0, 0); }
// rows of 16 MT doubles, an odd number of 16s apart: the four rows that a fragment's lanes read lie in different banks
constexpr int ONE_PART = 256, MOST_PARTS = 32, FEW_STEPS = 6;
template <int MT> struct Few { static constexpr int MP = 16 * MT, LD = MP | 16, TILES = MT * (MT + 1) / 2, SIZE = MP * LD; };
// tile t of those on and above the diagonal, column by column
__device__ __forceinline__ void tile_at(int t, int& a, int& b) { b = 0; while (t > b) t -= ++b; a = t; }
// a lane's 4 values of tile (a, b) of a product: row l / 16 + 4 i, column l % 16
template <int LD> __device__ __forceinline__ int few_at(int a, int b, int i) { return (16 * a + (threadIdx.x >> 4 & 3) + 4 * i) * LD + 16 * b + (threadIdx.x & 15); }
template <int LD> __device__ __forceinline__ int few_mirror(int a, int b, int i) { return (16 * b + (threadIdx.x & 15)) * LD + 16 * a + (threadIdx.x >> 4 & 3) + 4 * i; }

// Gram matrix of columns c0 .. c1 - 1 of G into `to`: the waves take 16 columns in turn and are added in their order
template <typename T, int MT> __device__ __forceinline__ void gram_few(const T* g, int m, int n, int tall, int c0, int c1, double* to) {
    using F = Few<MT>;
    const int wave = threadIdx.x >> 6, i = threadIdx.x & 15, h = threadIdx.x >> 4 & 3;
    d4 acc[F::TILES] = {};
    for (int k = c0 + 16 * wave; k < c1; k += 64) {
        T raw[MT][4];
#pragma unroll
        for (int r = 0; r < MT; r++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int row = min(16 * r + i, m - 1), col = min(k + 4 * h + c, c1 - 1);
                raw[r][c] = g[tall ? (long)col * m + row : (long)row * n + col];
            }
#pragma unroll
        for (int c = 0; c < 4; c++) {
            double x[MT];
#pragma unroll
            for (int r = 0; r < MT; r++) x[r] = 16 * r + i < m && k + 4 * h + c < c1 ? (double)(float)raw[r][c] : 0.;
#pragma unroll
            for (int b = 0, t = 0; b < MT; b++)
#pragma unroll
                for (int a = 0; a <= b; a++, t++) acc[t] = mfma(x[a], x[b], acc[t]);
        }
    }
    for (int w = 0; w < 4; w++) {
        if (wave == w) {
#pragma unroll
            for (int b = 0, t = 0; b < MT; b++)
#pragma unroll
                for (int a = 0; a <= b; a++, t++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int at = few_at<F::LD>(a, b, j);
                        const double v = w ? to[at] + acc[t][j] : acc[t][j];
                        to[at] = v;
                        if (w == 3 && a != b) to[few_mirror<F::LD>(a, b, j)] = v;
                    }
        }
        __syncthreads();
    }
}
// a part of the columns per workgroup; whole matrices of MP x MP, added up by few_rows_kernel
template <typename T, int MT> __global__ void __launch_bounds__(256) few_gram_kernel(Mats q, int m, int n, int tall, double* parts) {
    extern __shared__ __align__(16) char smem[];
    using F = Few<MT>;
    double* A = (double*)smem;
    gram_few<T, MT>((const T*)q.in[blockIdx.y], m, n, tall, (int)((long)n * blockIdx.x / gridDim.x), (int)((long)n * (blockIdx.x + 1) / gridDim.x), A);
    double* to = parts + ((long)blockIdx.y * gridDim.x + blockIdx.x) * F::MP * F::MP;
    for (int e = threadIdx.x; e < F::MP * F::MP; e += 256) to[e] = A[e / F::MP * F::LD + e % F::MP];
}

// S = 0: one workgroup takes a matrix through all of it.  Otherwise from the Gram matrix's S parts, each of a matrix's workgroups through the (same)
// steps and then its own columns of Q G: that costs what a launch of its own for the steps would, without the launch
template <typename T, int MT>
__global__ void __launch_bounds__(256) few_rows_kernel(Mats q, int m, int n, int tall, int steps, float eps, const double* parts, int S) {
    extern __shared__ __align__(16) char smem[];
    using F = Few<MT>;
    constexpr int MP = F::MP, LD = F::LD, EACH = (F::TILES + 3) / 4;
    double *A = (double*)smem, *P = A + F::SIZE, *Q = P + F::SIZE;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, h = lane >> 4;
    const T* g = (const T*)q.in[blockIdx.y];
    if (S == 0) gram_few<T, MT>(g, m, n, tall, 0, n, A);
    else {
        for (int e = threadIdx.x; e < MP * MP; e += 256) {
            const double* from = parts + (long)blockIdx.y * S * MP * MP + e;
            double v = 0.;
#pragma unroll 4
            for (int s = 0; s < S; s++) v += from[(long)s * MP * MP];
            A[e / MP * LD + e % MP] = v;
        }
        __syncthreads();
    }
    double trace = lane < MP ? A[lane * LD + lane] : 0.;        // |G|^2: neither 2^100 nor 2^-100 as a loss scale overflows or vanishes
    for (int o = 32; o; o >>= 1) trace += __shfl_xor(trace, o);
    const double inv = reciprocal(trace, eps);
    __syncthreads();
    for (int e = threadIdx.x; e < F::SIZE; e += 256) A[e] *= inv * inv;        // (what lies between the rows is nobody's)
    __syncthreads();
    // a product of two symmetric matrices that commute, which is symmetric: its tiles on and above the diagonal, dealt out to the waves
    auto product = [&](const double* x, const double* y, d4 (&acc)[EACH]) {
        int a[EACH], b[EACH];
#pragma unroll
        for (int u = 0; u < EACH; u++) { tile_at(min(wave + 4 * u, F::TILES - 1), a[u], b[u]); acc[u] = d4{}; }
#pragma unroll
        for (int k = 0; k < MP; k += 4)
#pragma unroll
            for (int u = 0; u < EACH; u++) acc[u] = mfma(x[(k + h) * LD + 16 * a[u] + i], y[(k + h) * LD + 16 * b[u] + i], acc[u]);
    };
    auto put = [&](double* to, auto value) {                 // value(place, i-th of tile u)
#pragma unroll
        for (int u = 0; u < EACH; u++) {
            int a, b;
            tile_at(wave + 4 * u, a, b);
            if (wave + 4 * u < F::TILES)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int at = few_at<LD>(a, b, j);
                    const double v = value(at, u, j);
                    to[at] = v;
                    if (a != b) to[few_mirror<LD>(a, b, j)] = v;
                }
        }
    };
    for (int it = 0; it < steps; it++) {
        const bool last = it + 1 == steps;
        d4 r[EACH], s[EACH];
        product(A, A, r);
        put(P, [&](int at, int u, int j) { return (at / LD == at % LD ? 3.4445 : 0.) + (-4.7750 * A[at] + 2.0315 * r[u][j]); });
        __syncthreads();
        if (it) product(P, Q, r);
        if (!last) product(P, A, s);
        __syncthreads();
        put(Q, [&](int at, int u, int j) { return it ? r[u][j] : inv * P[at]; });
        if (!last) put(A, [&](int, int u, int j) { return s[u][j]; });
        __syncthreads();
        if (last) break;
        product(P, A, s);
        __syncthreads();
        put(A, [&](int, int u, int j) { return s[u][j]; });
        __syncthreads();
    }
    // Q G, 16 columns of a wave at a time, read before they are written.  A tall G is its transpose here, and so is its tile
    T* out = (T*)q.out[blockIdx.y];
    for (int c0 = (blockIdx.x * 4 + wave) * 16; c0 < n; c0 += gridDim.x * 64) {
        T raw[MP / 4];
        double x[MP / 4];
#pragma unroll
        for (int k = 0; k < MP / 4; k++) {
            const int row = min(4 * k + h, m - 1), col = min(c0 + i, n - 1);
            raw[k] = g[tall ? (long)col * m + row : (long)row * n + col];
        }
#pragma unroll
        for (int k = 0; k < MP / 4; k++) x[k] = 4 * k + h < m && c0 + i < n ? (double)(float)raw[k] : 0.;
#pragma unroll
        for (int a = 0; a < MT; a++) {
            d4 acc = {};
#pragma unroll
            for (int k = 0; k < MP / 4; k++) {
                const double y = Q[(4 * k + h) * LD + 16 * a + i];
                acc = tall ? mfma(x[k], y, acc) : mfma(y, x[k], acc);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int row = 16 * a + (tall ? i : h + 4 * j), col = c0 + (tall ? h + 4 * j : i);
                if (row < m && col < n) out[tall ? (long)col * m + row : (long)row * n + col] = (T)(float)acc[j];
            }
        }
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------
struct Plan { long x, a, norm; long total(int count) const { return count * (3 * x + 2 * a) * (long)sizeof(f16) + norm; } };
Plan plan_of(int m, int n) {                // halves of one matrix: X (and each X^T), A (and B); bytes of the norms' parts
    const long mp = up(m), np = up(n);
    return {2 * mp * np, 2 * mp * mp, MANY * PARTS * (long)sizeof(double)};
}
bool few_rows(int m, int n) { return m <= 32 || (m <= 64 && n > 128); }        // ... and up to FEW_STEPS
// parts of a Gram matrix, by the columns alone (a matrix's result does not depend on its batch)
int few_parts(int n) { return n <= ONE_PART ? 0 : (n + ONE_PART - 1) / ONE_PART < MOST_PARTS ? (n + ONE_PART - 1) / ONE_PART : MOST_PARTS; }
long few_bytes(int count, int m, int n) { const long mp = (m + 15) / 16 * 16, s = few_parts(n); return count * (s > 0 ? s : 1) * mp * mp * (long)sizeof(double); }
template <int MODE, int F> bool wide(const Product& p, const Mats& q, hipStream_t s) {
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    constexpr size_t bytes = 4 * (F + 2) * 4096;
    static size_t raised[64];
    if (!bl_raise_lds_limit((const void*)product_wide_kernel<MODE, F>, bytes, raised)) return false;
    hipLaunchKernelGGL((product_wide_kernel<MODE, F>), dim3((unsigned)(tiles_in<SYM, 64 * F, 128>(p.M, p.N) * p.count)), dim3(256), bytes, s, p, q);
    return true;
}
template <int MODE> bool multiply(const Product& p, const Mats& q, hipStream_t s) {
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    // The larger tile wherever it fills the chip well enough.  us for all 15 products of 5 steps on tiles of 64 x 64 / 128 x 128 / 256 x 128:
    // 8 matrices of 512: 220 / 256 / 389; of 1024, one: 206 / 338 / 557, two: 309 / 364 / 572, four: 502 / 443 / 596, eight: 845 / 840 / 757; one of 2048:
    // 942 / 753 / 1010.  128 x 128 pays from 136 tiles on (72 .. 128 do not), 256 x 128 where tiles of 128 x 128 are more than the 256 CUs and a second round
    // of them begins.  Whole calls on 128 x 128 / 256 x 128, in tiles of 128 x 128 for X X^T: 24 x 512 x 1024, 240 tiles: 614 / 696; 7 x 1024 x 1024, 252: 587 / 693; 26 x 512 x 512, 260:
    // 491 / 461; 2 x 2048 x 2048, 272: 1303 / 1219; B X alone, 3 x 1280 x 1280, 300: 597 / 542.
    const bool whole = p.M % 128 == 0 && p.N % 128 == 0;
    const int tiles = whole ? tiles_in<SYM, 128, 128>(p.M, p.N) * p.count : 0;
    if (tiles > 256 && p.M % 256 == 0) return wide<MODE, 4>(p, q, s);
    if (tiles > 128) return wide<MODE, 2>(p, q, s);
    hipLaunchKernelGGL((product_64_kernel<MODE>), dim3((unsigned)(tiles_in<SYM, 64, 64>(p.M, p.N) * p.count)), dim3(256), 65536, s, p, q);
    return true;
}

template <typename T, int NB> bool small(const Product& p, const Mats& q, int steps, float eps, hipStream_t s) {
    constexpr size_t bytes = 3 * sizeof(f16) * (2 * 64 * 64 * NB + 2 * 64 * 64);
    static size_t raised[64];
    if (!bl_raise_lds_limit((const void*)ortho_small_kernel<T, NB>, bytes, raised)) return false;
    hipLaunchKernelGGL((ortho_small_kernel<T, NB>), dim3(p.count), dim3(256), bytes, s, q, p, steps, eps);
    return true;
}
template <typename T, int MT> int few(const Mats& q, int c, int m, int n, int tall, int steps, float eps, double* parts, hipStream_t s) {
    using F = Few<MT>;
    constexpr size_t one = F::SIZE * sizeof(double);
    static size_t raised[64];
    if (!bl_raise_lds_limit((const void*)few_rows_kernel<T, MT>, 3 * one, raised)) return BL_ELAUNCH;
    const int S = few_parts(n), most = (n + 63) / 64, want = 256 / c;
    if (S) hipLaunchKernelGGL((few_gram_kernel<T, MT>), dim3(S, c), dim3(256), one, s, q, m, n, tall, parts);
    hipLaunchKernelGGL((few_rows_kernel<T, MT>), dim3(S == 0 ? 1 : want < most ? want : most, c), dim3(256), 3 * one, s, q, m, n, tall, steps, eps, parts, S);
    return check_launch();
}
template <typename T> int run(const Mats& q, int c, int m, int n, int tall, int dtype, int steps, float eps, const Plan& plan, void* workspace, hipStream_t s) {
    const int mp = up(m), np = up(n);
    double* parts = (double*)workspace;
    if (few_rows(m, n) && steps <= FEW_STEPS)
        return m <= 16 ? few<T, 1>(q, c, m, n, tall, steps, eps, parts, s) : m <= 32 ? few<T, 2>(q, c, m, n, tall, steps, eps, parts, s)
             : m <= 48 ? few<T, 3>(q, c, m, n, tall, steps, eps, parts, s) : few<T, 4>(q, c, m, n, tall, steps, eps, parts, s);
    if (m <= 64 && n <= 128) {
        Product p{};
        p.m = m; p.n = n; p.tall = tall; p.dtype = dtype; p.count = c;
        if (!(n <= 64 ? small<T, 1>(p, q, steps, eps, s) : small<T, 2>(p, q, steps, eps, s))) return BL_ELAUNCH;
        return check_launch();
    }
    f16* X = (f16*)((char*)workspace + plan.norm);
    f16* XT[2] = {X + c * plan.x, X + 2 * c * plan.x};
    f16* A = X + 3 * c * plan.x;
    f16* B = A + c * plan.a;
    hipLaunchKernelGGL((norm_parts_kernel<T>), dim3(PARTS, c), dim3(256), 0, s, q, (long)m * n, parts);
    hipLaunchKernelGGL((lay_out_kernel<T>), dim3(np / 32, mp / 32, c), dim3(256), 0, s, q, m, n, tall, eps, parts, X, XT[0], plan.x);
    for (int it = 0; it < steps; it++) {
        f16 *from = XT[it & 1], *to = XT[(it & 1) ^ 1];
        // acc carries SCALE^2
        bool ok = multiply<GRAM>(Product{X, X, plan.x, plan.x, nullptr, 0, A, A, plan.a, plan.a, mp, mp, np, 0.f, UNSCALE, 0, 0, 0, 0, c}, q, s);
        ok = ok && multiply<POLY>(Product{A, A, plan.a, plan.a, A, plan.a, B, B, plan.a, plan.a, mp, mp, mp, NS_B, NS_C * UNSCALE, 0, 0, 0, 0, c}, q, s);
        // X^T B: n x m, whose transpose a X + B X is written over X (nobody reads X here but the lane that replaces it)
        const Product next{from, B, plan.x, plan.a, X, plan.x, X, to, plan.x, plan.x, np, mp, mp, NS_A, UNSCALE, m, n, tall, dtype, c};
        ok = ok && (it + 1 < steps ? multiply<NEXT>(next, q, s) : multiply<LAST>(next, q, s));
        if (!ok) return BL_ELAUNCH;
    }
    return check_launch();
}

}  // namespace

extern "C" {

long bl_orthogonalize_workspace(int count, int rows, int cols) {
    if (count <= 0 || rows <= 0 || cols <= 0 || rows > BL_ORTHO_MAX || cols > BL_ORTHO_MAX) return 0;
    const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    if (count > MANY) count = MANY;
    const long all = plan_of(m, n).total(count), few = few_rows(m, n) ? few_bytes(count, m, n) : 0;       // (whatever the steps)
    return all > few ? all : few;
}

int bl_orthogonalize(const void* const* host_in, void* const* host_out, int count, int dtype, int rows, int cols, int steps, float eps,
                     void* workspace, bl_stream_t stream) {
    if (!host_in || !host_out || !workspace || count <= 0 || rows <= 0 || cols <= 0 || steps <= 0 || !(eps >= 0.f)) return BL_EINVAL;
    if (dtype != BL_F32 && dtype != BL_F16 && dtype != BL_BF16) return BL_EINVAL;
    if (rows > BL_ORTHO_MAX || cols > BL_ORTHO_MAX) return BL_ETOOBIG;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return BL_EINVAL;
    for (int i = 0; i < count; i++) if (!host_in[i] || !host_out[i]) return BL_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    const int tall = rows > cols, m = tall ? cols : rows, n = tall ? rows : cols;
    const Plan plan = plan_of(m, n);
    for (int i0 = 0; i0 < count; i0 += MANY) {
        const int c = count - i0 < MANY ? count - i0 : MANY;
        Mats q{};
        for (int i = 0; i < c; i++) { q.in[i] = host_in[i0 + i]; q.out[i] = host_out[i0 + i]; }
        const int rc = dtype == BL_F32 ? run<float>(q, c, m, n, tall, dtype, steps, eps, plan, workspace, s)
                     : dtype == BL_F16 ? run<f16>(q, c, m, n, tall, dtype, steps, eps, plan, workspace, s) : run<bf16>(q, c, m, n, tall, dtype, steps, eps, plan, workspace, s);
        if (rc) return rc;
    }
    return BL_OK;
}

}  // extern "C"
