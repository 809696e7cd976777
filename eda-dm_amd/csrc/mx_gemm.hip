// Product of microscaled operands on the block-scaled matrix instructions (v_mfma_scale_f32_16x16x128_f8f6f4):
//   out[m][n] = sum_b 2^(sa[m][b] - 127 + sw[n][b] - 127) sum_{k in block b} a[m][k] w[n][k]  (+ bias[n])
// with a in e4m3 or e2m1 and w in e2m1, both as they lie in memory (rows of blocks; no weight is re-packed), 32-bit accumulation.
//
// Operand layout of the 16 x 16 x 128 instruction, lane l = 16 q + r: a 4-bit operand's lane holds the 32 elements of block q of
// row r; an 8-bit operand's lane holds elements 16 q .. 16 q + 15 of each half of row r; either way lane l gives the scale of
// block q of row r.  w goes in as the first operand, so that a lane ends up with four neighbouring columns of one output row.
//
// Precision.  Within a group of products the instruction keeps 13 binary places below the largest exponent.  The 4 x 4-bit products
// (and 8 x 4-bit ones within 8 binades) are inside that and sum exactly; e4m3 spans 18 binades, and what falls below is cut off: a
// relative error of a few 1e-6 of the result, which a 16-bit output's rounding (2e-3) hides.  For a 32-bit output the 8-bit operand is
// split by the top bit of its exponent into two operands of 8 binades each, both exact, at twice the matrix work.
#include "mx_common.h"
#include "../../include/edadm.h"

typedef int mx_i8 __attribute__((ext_vector_type(8)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));

struct MxArgs {
    const uint8_t *A, *As, *W, *Ws;
    int64_t lda, ldas, ldw, ldws;      // bytes
    const float* bias;
    void* out;
    int64_t ldo;                       // elements
    int64_t M, N;
    int nblk;                          // blocks of 32 along K
};

__device__ __forceinline__ mx_i8 frag4(uint4 a) { return mx_i8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}; }
__device__ __forceinline__ mx_i8 frag8(uint4 a, uint4 b) { return mx_i8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w}; }

// e4m3 codes with exponent fields 8 .. 15 / 0 .. 7, zeros elsewhere (bytes: the field's top bit is bit 6)
__device__ __forceinline__ mx_i8 part_hi(mx_i8 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) { const uint32_t m = (uint32_t)c[i] & 0x40404040u; c[i] = (int)((uint32_t)c[i] & (((m << 1) - (m >> 6)) | 0x80808080u)); }
    return c;
}
__device__ __forceinline__ mx_i8 part_lo(mx_i8 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) { const uint32_t m = (uint32_t)c[i] & 0x40404040u; c[i] = (int)((uint32_t)c[i] & ~((m << 1) - (m >> 6))); }
    return c;
}

template <int AF, bool EXACT>
__device__ __forceinline__ mx_f4 mx_mma16(mx_i8 w, mx_i8 a, mx_f4 c, uint32_t sw, uint32_t sa) {
    if constexpr (AF == MX_FP4) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 4, 4, 0, (int)sw, 0, (int)sa);
    else if constexpr (!EXACT) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 4, 0, 0, (int)sw, 0, (int)sa);
    else {
        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, part_lo(a), c, 4, 0, 0, (int)sw, 0, (int)sa);
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, part_hi(a), c, 4, 0, 0, (int)sw, 0, (int)sa);
    }
}

// four neighbouring columns of row m
template <int ODT> __device__ __forceinline__ void mx_out4(const MxArgs& a, int64_t m, int64_t n, mx_f4 v) {
    if (m >= a.M || n >= a.N) return;
    if (n + 4 <= a.N) {
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += a.bias[n + i];
        }
        const int64_t at = m * a.ldo + n;
        // rows may start at any element: a vector store where this one is aligned for it
        if constexpr (ODT == MX_F32) {
            float* p = (float*)a.out + at;
            if (((uintptr_t)p & 15) == 0) *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
            else { p[0] = v[0]; p[1] = v[1]; p[2] = v[2]; p[3] = v[3]; }
        } else {
            uint16_t* p = (uint16_t*)a.out + at;
            const uint32_t x = mx_pair<ODT>(v[0], v[1]), y = mx_pair<ODT>(v[2], v[3]);
            if (((uintptr_t)p & 7) == 0) *(uint2*)p = make_uint2(x, y);
            else { p[0] = (uint16_t)x; p[1] = (uint16_t)(x >> 16); p[2] = (uint16_t)y; p[3] = (uint16_t)(y >> 16); }
        }
    } else {
        for (int i = 0; i < 4 && n + i < a.N; ++i) {
            const float s = a.bias ? v[i] + a.bias[n + i] : v[i];
            if constexpr (ODT == MX_F32) ((float*)a.out)[m * a.ldo + n + i] = s;
            else ((uint16_t*)a.out)[m * a.ldo + n + i] = (uint16_t)mx_pair<ODT>(s, 0.f);
        }
    }
}

// ------------------------------------------------------------------------------------------------ few rows
// A workgroup owns 16 NT columns and 16 MT rows; its waves take the K-steps of 128 in turn, fetch their operands straight into
// registers (UK steps of them in flight) and add their sums in LDS in the order of the waves.  Bound by reading w once.
template <int AF, int MT, int NT, int UK, bool EXACT, int ODT>
__global__ __launch_bounds__(512) void k_mx_rows(MxArgs a, int strips) {
    constexpr int WAVES = 8;
    __shared__ mx_f4 red[WAVES][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)(blockIdx.x % strips) * (16 * NT), m0 = (int64_t)(blockIdx.x / strips) * (16 * MT);
    const int steps = (a.nblk + 3) / 4;
    const uint8_t *wp[NT], *wsp[NT], *ap[MT], *asp[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t n = min(n0 + 16 * j + r, a.N - 1);              // rows past the end: read the last one, store nothing
        wp[j] = a.W + n * a.ldw + q * 16;
        wsp[j] = a.Ws + n * a.ldws + q;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = min(m0 + 16 * i + r, a.M - 1);
        ap[i] = a.A + m * a.lda + q * 16;
        asp[i] = a.As + m * a.ldas + q;
    }
    mx_f4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mx_f4{0, 0, 0, 0};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int s0 = wave; s0 < steps; s0 += WAVES * UK) {
        uint4 w[UK][NT], x[UK][MT], y[UK][MT];
        uint32_t sw[UK][NT], sa[UK][MT];
#pragma unroll
        for (int u = 0; u < UK; ++u) {
            const int b = (s0 + u * WAVES) * 4;                       // first block of the step
            const bool in = b + q < a.nblk;                           // blocks past the end: zeros under any finite scale
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                w[u][j] = in ? *(const uint4*)(wp[j] + (int64_t)b * 16) : zero;
                sw[u][j] = in ? wsp[j][b] : 127u;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if constexpr (AF == MX_FP4) x[u][i] = in ? *(const uint4*)(ap[i] + (int64_t)b * 16) : zero;
                else {
                    x[u][i] = b + (q >> 1) < a.nblk ? *(const uint4*)(ap[i] + (int64_t)b * 32) : zero;
                    y[u][i] = b + 2 + (q >> 1) < a.nblk ? *(const uint4*)(ap[i] + (int64_t)b * 32 + 64) : zero;
                }
                sa[u][i] = in ? asp[i][b] : 127u;
            }
        }
#pragma unroll
        for (int u = 0; u < UK; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const mx_i8 fa = AF == MX_FP4 ? frag4(x[u][i]) : frag8(x[u][i], y[u][i]);
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = mx_mma16<AF, EXACT>(frag4(w[u][j]), fa, acc[i][j], sw[u][j], sa[u][i]);
            }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) red[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * NT * 64; e += WAVES * 64) {
        const int tile = e >> 6, l = e & 63;
        mx_f4 v = red[0][tile][l];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) v += red[k][tile][l];
        mx_out4<ODT>(a, m0 + 16 * (tile / NT) + (l & 15), n0 + 16 * (tile % NT) + 4 * (l >> 4), v);
    }
}

// ------------------------------------------------------------------------------------------------ host side
template <int AF, bool EXACT, int ODT> static int launch_rows(const MxArgs& a, hipStream_t st) {
    const int64_t mt = (a.M + 15) / 16;
    const int m = mt >= 4 ? 4 : mt == 3 ? 3 : (int)mt;
    const int64_t strips = (a.N + 15) / 16, chunks = (mt + m - 1) / m;
    if (strips > 0x7fffffff || strips * chunks > 0x7fffffff) return EDADM_EINVAL;
    const unsigned grid = (unsigned)(strips * chunks);
    if (m == 1) k_mx_rows<AF, 1, 1, 5, EXACT, ODT><<<grid, 512, 0, st>>>(a, (int)strips);
    else if (m == 2) k_mx_rows<AF, 2, 1, 3, EXACT, ODT><<<grid, 512, 0, st>>>(a, (int)strips);
    else if (m == 3) k_mx_rows<AF, 3, 1, 2, EXACT, ODT><<<grid, 512, 0, st>>>(a, (int)strips);
    else k_mx_rows<AF, 4, 1, 2, EXACT, ODT><<<grid, 512, 0, st>>>(a, (int)strips);
    return edadm_launch_status();
}

template <int AF, bool EXACT, int ODT> static int launch_mx(const MxArgs& a, hipStream_t st) { return launch_rows<AF, EXACT, ODT>(a, st); }

static inline bool mx_side_ok(const uint8_t* c, int64_t ld, const uint8_t* s, int64_t lds, int64_t rows, int64_t nb, int fmt) {
    return c && s && (uintptr_t)c % 16 == 0 && ld >= nb * (fmt == MX_FP4 ? 16 : 32) && (rows <= 1 || ld % 16 == 0) && lds >= nb;
}

extern "C" int edadm_mx_gemm(const uint8_t* A, int64_t lda, const uint8_t* As, int64_t ldas, int afmt, const uint8_t* W, int64_t ldw,
                             const uint8_t* Ws, int64_t ldws, int64_t M, int64_t N, int64_t K, const float* bias, void* out, int64_t ldo,
                             int odt, void* stream) {
    const int64_t nb = (K + 31) / 32;
    if (M < 0 || N < 0 || K < 1 || nb > (1 << 24) || (afmt != MX_FP4 && afmt != MX_FP8) || odt < MX_F32 || odt > MX_F16) return EDADM_EINVAL;
    if (M == 0 || N == 0) return 0;
    if (!mx_side_ok(A, lda, As, ldas, M, nb, afmt) || !mx_side_ok(W, ldw, Ws, ldws, N, nb, MX_FP4) || !out || ldo < N) return EDADM_EINVAL;
    const MxArgs a = {A, As, W, Ws, lda, ldas, ldw, ldws, bias, out, ldo, M, N, (int)nb};
    hipStream_t st = (hipStream_t)stream;
    if (afmt == MX_FP4)
        return odt == MX_F32 ? launch_mx<MX_FP4, false, MX_F32>(a, st) : odt == MX_BF16 ? launch_mx<MX_FP4, false, MX_BF16>(a, st) : launch_mx<MX_FP4, false, MX_F16>(a, st);
    return odt == MX_F32 ? launch_mx<MX_FP8, true, MX_F32>(a, st) : odt == MX_BF16 ? launch_mx<MX_FP8, false, MX_BF16>(a, st) : launch_mx<MX_FP8, false, MX_F16>(a, st);
}
