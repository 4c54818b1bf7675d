// The root-mean-square norm in front of a linear with the residual's addition and the quantizer, in one
// pass: h = x + res, r = 1 / sqrt(mean(h^2) + eps), and QACT (fp32.quantize_mx, opentpu/fp32.py:321-343)
// of (h * r) * gamma, the products QACT's RSCALE and CSCALE make (docs/isa.md:447-452): with the r this
// kernel gives, otpu_qact of its fp32 h gives the same bits.
//
// Bound by memory: x and res are read and h, the bytes and the offsets written once (fp32 13 bytes an
// element), the row held in registers between the sum of squares, the maximum and the quantizing.
// 16384 x 4096 fp32: 168 us, 5.2 TB/s, as a large copy; 1 x 1024: 3.3 us, a launch and two trips to memory.
#include "otpu_common.h"

namespace otpu {

struct NormArgs {
    const void* x; int64_t ldx;
    const void* res; int64_t ldr;   // or NULL
    const float* gamma;
    int K; float eps;
    void* h; int64_t ldh;           // or NULL
    float* r;                       // or NULL
    int8_t* q; int64_t ldq;
    float* S;
    uint8_t* d; int64_t ldd;
};

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// 16 bytes of a row as fp32 values, and back (to 16 bits: rounded to nearest even)
template <int DT> struct Row;
template <> struct Row<OTPU_F32> {
    static constexpr int V = 4;
    static __device__ __forceinline__ void load(const void* p, int64_t i, float (&f)[V]) {
        const v4f t = *reinterpret_cast<const v4f*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = t[j];
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float (&f)[V]) {
        *reinterpret_cast<v4f*>(static_cast<float*>(p) + i) = v4f{f[0], f[1], f[2], f[3]};
    }
};
template <typename VT, typename ET>
struct Row16 {
    static constexpr int V = 8;
    static __device__ __forceinline__ void load(const void* p, int64_t i, float (&f)[V]) {
        const VT t = *reinterpret_cast<const VT*>(static_cast<const ET*>(p) + i);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = (float)t[j];
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float (&f)[V]) {
        VT t;
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = (ET)f[j];
        *reinterpret_cast<VT*>(static_cast<ET*>(p) + i) = t;
    }
};
template <> struct Row<OTPU_BF16> : Row16<v8bf, __bf16> {};
template <> struct Row<OTPU_F16> : Row16<v8h, _Float16> {};

__device__ __forceinline__ float wave_sum_f32(float v) {
    v += bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(v), 0xB1, 0xF, 0xF, false));
    v += bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(v), 0x4E, 0xF, 0xF, false));
    v += bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(v), 0x141, 0xF, 0xF, false));
    v += bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(v), 0x140, 0xF, 0xF, false));
    const auto a = __builtin_amdgcn_permlane16_swap(fbits(v), fbits(v), false, false);
    v = bitsf(a[0]) + bitsf(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(v), false, false);
    return bitsf(b[0]) + bitsf(b[1]);
}

// TPR threads a row (a wave of a workgroup of four, or a workgroup of 256 or 1024), CPT pieces of 16
// bytes of x a thread
template <int DT, bool ROW, int CPT, int TPR>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_qact_kernel(NormArgs a, int M) {
    using R = Row<DT>;
    constexpr int V = R::V, W = TPR / 64;
    __shared__ float rsum[W];
    __shared__ uint32_t rmax[W];
    const int row = TPR == 64 ? (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : (int)blockIdx.x;
    if (row >= M) return;                                  // (TPR 64 only: a whole wave, no barrier below)
    const int lane = threadIdx.x & (TPR - 1), K = a.K, nc = K / V;
    const int64_t ox = (int64_t)row * a.ldx, orr = (int64_t)row * a.ldr;

    float v[CPT][V];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = lane + TPR * k;
        if (c < nc) R::load(a.x, ox + (int64_t)c * V, v[k]);
        else
#pragma unroll
            for (int j = 0; j < V; ++j) v[k][j] = 0.f;
    }
    if (a.res) {
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            const int c = lane + TPR * k;
            if (c < nc) {
                float u[V];
                R::load(a.res, orr + (int64_t)c * V, u);
#pragma unroll
                for (int j = 0; j < V; ++j) v[k][j] = fadd(v[k][j], u[j]);
            }
        }
    }
    float ss = 0.f;                                        // the sum of squares: in fp32 throughout
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = lane + TPR * k;
        if (a.h && c < nc) R::store(a.h, (int64_t)row * a.ldh + (int64_t)c * V, v[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) ss = __builtin_fmaf(v[k][j], v[k][j], ss);
    }
    ss = wave_sum_f32(ss);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) rsum[threadIdx.x >> 6] = ss;
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) ss += rsum[w];
    }
    const float r = ftz(1.0f / __builtin_sqrtf(ss / (float)K + a.eps));
    uint32_t m = 0, gm[CPT];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = lane + TPR * k;
        gm[k] = 0;
        if (c < nc) {
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const v4f g = *reinterpret_cast<const v4f*>(a.gamma + (int64_t)c * V + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[k][j + i] = fmul(fmul(v[k][j + i], r), g[i]);
                    gm[k] = max(gm[k], fbits(v[k][j + i]) & 0x7FFFFFFFu);
                }
            }
        }
        m = max(m, gm[k]);
    }
    uint32_t amax = wave_max_dpp(m, 64);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) rmax[threadIdx.x >> 6] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) amax = max(amax, rmax[w]);
    }
    const float fa = bitsf(amax);
    const float inv = amax ? fmul(127.0f, recip(fa)) : 0.0f;
    if (lane == 0) {
        a.S[row] = amax ? fmul(fa, bitsf(0x3C010204u)) : 0.0f;   // amax * f32(1/127)
        if (a.r) a.r[row] = r;
    }
    uint32_t* qr = reinterpret_cast<uint32_t*>(a.q + (int64_t)row * a.ldq);
    uint8_t* dr = a.d ? a.d + (int64_t)row * a.ldd : nullptr;
    constexpr int GL = 32 / V;                             // lanes a group
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int c = lane + TPR * k;
        int dg = 0;
        if constexpr (!ROW) {
            const uint32_t g = wave_max_dpp(gm[k], GL);
            dg = (int)(amax >> 23) - (int)(g >> 23) - ((g & 0x7FFFFFu) > (amax & 0x7FFFFFu));
            dg = g ? (dg < 0 ? 0 : (dg > 31 ? 31 : dg)) : 0;
        }
        const float sc = fmul(inv, pow2f(dg));
        uint32_t p[V / 4];
#pragma unroll
        for (int j = 0; j < V / 4; ++j)
            p[j] = (uint32_t)(q8(fmul(v[k][4 * j], sc)) & 0xFF) | ((uint32_t)(q8(fmul(v[k][4 * j + 1], sc)) & 0xFF) << 8)
                 | ((uint32_t)(q8(fmul(v[k][4 * j + 2], sc)) & 0xFF) << 16) | ((uint32_t)(q8(fmul(v[k][4 * j + 3], sc)) & 0xFF) << 24);
        if (c < nc) {
            if constexpr (V == 8) reinterpret_cast<uint2*>(qr)[c] = make_uint2(p[0], p[1]);
            else qr[c] = p[0];
            if (dr && c % GL == 0) dr[c / GL] = (uint8_t)dg;
        }
    }
}

template <int DT, bool ROW, int CPT>
static void launch_tpr(const NormArgs& a, int M, int tpr, hipStream_t s) {
    if (tpr == 64) norm_qact_kernel<DT, ROW, CPT, 64><<<(M + 3) / 4, 256, 0, s>>>(a, M);
    else if (tpr == 256) norm_qact_kernel<DT, ROW, CPT, 256><<<M, 256, 0, s>>>(a, M);
    else norm_qact_kernel<DT, ROW, CPT, 1024><<<M, 1024, 0, s>>>(a, M);
}

template <int DT, bool ROW>
static void launch_norm(const NormArgs& a, int M, hipStream_t s) {
    // A wave a row up to two pieces a lane (no barrier), a workgroup of 256 up to eight a thread, else of 1024:
    // pieces past eight would not stay in registers.
    const int nc = a.K / Row<DT>::V;
    const int tpr = nc <= 128 ? 64 : (nc <= 2048 ? 256 : 1024);
    const int per = (nc + tpr - 1) / tpr;
    if (per <= 1) launch_tpr<DT, ROW, 1>(a, M, tpr, s);
    else if (per <= 2) launch_tpr<DT, ROW, 2>(a, M, tpr, s);
    else if (per <= 4) launch_tpr<DT, ROW, 4>(a, M, tpr, s);
    else launch_tpr<DT, ROW, 8>(a, M, tpr, s);
}

}  // namespace otpu

using namespace otpu;

static bool al(const void* p, int a) { return ((uintptr_t)p & (uintptr_t)(a - 1)) == 0; }

extern "C" int otpu_norm_qact(const void* x, int64_t ldx, const void* res, int64_t ldr, int dtype, int M, int K,
                              const float* gamma, float eps, int flags, void* h, int64_t ldh, float* r, int8_t* q,
                              int64_t ldq, float* S, uint8_t* d, int64_t ldd, otpu_stream_t stream) {
    if (flags & ~OTPU_Q_ROW) return otpu_fail(OTPU_EINVAL, "norm_qact: unknown flags %#x", flags);
    const int row = flags & OTPU_Q_ROW;
    if (dtype != OTPU_F32 && dtype != OTPU_BF16 && dtype != OTPU_F16)
        return otpu_fail(OTPU_EFORMAT, "norm_qact: type %d", dtype);
    if (M < 0 || M >= (1 << 22) || K < 32 || K % 32 || K > OTPU_NORM_COLS)
        return otpu_fail(OTPU_EINVAL, "norm_qact: M %d, K %d (a multiple of 32, at most %d)", M, K, OTPU_NORM_COLS);
    if (!(eps >= 0.f)) return otpu_fail(OTPU_EINVAL, "norm_qact: eps %g", (double)eps);
    if (M == 0) return OTPU_OK;
    if (!x || !gamma || !q || !S || (!d && !row)) return otpu_fail(OTPU_EINVAL, "norm_qact: a NULL operand");
    if (ldx < K || (res && ldr < K) || (h && ldh < K) || ldq < K || (d && ldd < K / 32))
        return otpu_fail(OTPU_EINVAL, "norm_qact: rows shorter than %d columns", K);
    const int v = dtype == OTPU_F32 ? 4 : 8;
    if (!al(x, 16) || ldx % v || (res && (!al(res, 16) || ldr % v)) || (h && (!al(h, 16) || ldh % v)) || !al(gamma, 16) ||
        !al(q, v) || ldq % v || !al(S, 4) || (r && !al(r, 4)))
        return otpu_fail(OTPU_EALIGN, "norm_qact: rows of x, res and h and gamma 16-byte aligned, rows of q %d-byte aligned", v);
    NormArgs a = {x, ldx, res, ldr, gamma, K, eps, h, ldh, r, q, ldq, S, d, ldd};
    const hipStream_t s = (hipStream_t)stream;
    switch (2 * dtype + (row ? 1 : 0)) {
        case 2 * OTPU_F32: launch_norm<OTPU_F32, false>(a, M, s); break;
        case 2 * OTPU_F32 + 1: launch_norm<OTPU_F32, true>(a, M, s); break;
        case 2 * OTPU_BF16: launch_norm<OTPU_BF16, false>(a, M, s); break;
        case 2 * OTPU_BF16 + 1: launch_norm<OTPU_BF16, true>(a, M, s); break;
        case 2 * OTPU_F16: launch_norm<OTPU_F16, false>(a, M, s); break;
        default: launch_norm<OTPU_F16, true>(a, M, s); break;
    }
    return otpu_launch_check("norm_qact");
}
