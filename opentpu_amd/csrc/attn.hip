// Attention for a batch that shares a long prefix: each query sees all P keys of the shared prefix and
// its own sequence's keys up to its own place.  The softmax is split over key segments with a running
// maximum m and sum l of each (o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s), so the prefix is
// multiplied once by the rows of every sequence together and each sequence's cache by its own rows.
//
//   segment_kernel   one segment's share of the keys for a tile of rows: partial o, m, l
//   combine_kernel   the partials of a row joined, rounded to the output's type; the row's lse
//   weights_kernel   the own keys' weights from the finished lse, added to the running sums
#include "otpu_common.h"

namespace otpu {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

#define INL __attribute__((always_inline))

// a 16-bit type: the 32 x 32 x 16 product and the rounding of two fp32 values (to nearest even)
struct BF16 {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    typedef __bf16 e;
    static __device__ __forceinline__ v16f mma(v8s a, v8s b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static constexpr uint16_t INF = 0x7F80, ONE = 0x3F80;
};
struct F16 {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    typedef _Float16 e;
    static __device__ __forceinline__ v16f mma(v8s a, v8s b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static constexpr uint16_t INF = 0x7C00, ONE = 0x3C00;
};

struct AttnArgs {
    const char* q; int64_t qb, qt, qh;       // byte strides of sequence, token, head
    const char* pk; int64_t pks, pkh;        // prefix: of token, head
    const char* pv; int64_t pvs, pvh;
    const char* k; int64_t kb, kt, kh;       // own: of sequence, token, head
    const char* v; int64_t vb, vt, vh;
    const int32_t* lens;
    char* out; int64_t ob, ot, oh;
    float* weights;                          // [B, Hkv, T] or NULL
    int P, T, B, Lq, Hq, Hkv, G, D;
    float scale2;                            // scale * log2(e)
    int sp, ss;                              // splits of the prefix, of the own keys
    float* po;                               // partial o [sp + ss][rows][D]
    float* pm;                               // m [sp + ss][rows]
    float* pl;                               // l [sp + ss][rows]
    float* lse;                              // [rows]: log2 of the softmax's sum
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// direct-to-LDS load: 16 bytes a lane, lane L's at lds + 16 L
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 : : "v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
__device__ __forceinline__ void wait_all_dma() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }
__device__ __forceinline__ void bar() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

__device__ __forceinline__ float swap32_max(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(v), false, false);
    return fmaxf(bitsf(p[0]), bitsf(p[1]));
}
__device__ __forceinline__ float swap32_sum(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(v), false, false);
    return bitsf(p[0]) + bitsf(p[1]);
}

// A workgroup's shape: WR waves of 32 rows each times WK shares of the keys, KT keys a wave a step.
template <int DP_, int WR_, int WK_, int KT_>
struct Shape {
    static constexpr int DP = DP_, WR = WR_, WK = WK_, KT = KT_;
    static constexpr int NW = WR * WK;                     // waves
    static constexpr int BM = WR * 32;                     // rows
    static constexpr int NKEY = WK * KT;                   // keys a step
    static constexpr int CR = DP / 8;                      // 16-byte chunks a key
    static constexpr int KB = NKEY * DP * 2;               // bytes of a step's keys (and of its values)
    static constexpr int STAGE = 2 * KB;
    static constexpr int LOADS = KB / 1024 / NW;           // direct loads a wave issues for the keys
    static constexpr int MERGE = (WK - 1) * WR * 64 * (DP / 2 + 2) * 4;
    static constexpr int LDS = 2 * STAGE > MERGE ? 2 * STAGE : MERGE;
    static_assert(KB % (1024 * NW) == 0, "whole direct loads");
};

// chunk c of key row r lies in slot c ^ f(r): the 8 (16) rows that lanes read together at one c on
// distinct banks; of value row r: the 4 rows that a transposing read takes, two chunks each
template <int CR> __device__ __forceinline__ int kswz(int r) { return r & (CR < 16 ? CR - 1 : 15); }
template <int CR> __device__ __forceinline__ int vswz(int r) { return (2 * r) & (CR < 16 ? CR - 1 : 15); }

// The rows of a tile against keys [key0, key1) of a segment; lim: how many of the segment's keys this
// lane's row sees.
template <class E, class S, bool FULL, bool OWN>
__device__ __forceinline__ void segment_tile(const AttnArgs& a, char* lds, const char* kbase, int64_t kstride,
                                             const char* vbase, int64_t vstride, int key0, int key1, int lim,
                                             const char* qrow, bool valid, int slot, int64_t row) {
    constexpr int DP = S::DP, KT = S::KT, CR = S::CR, KS = DP / 16, DT = DP / 32, TT = KT / 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % S::WR, wk = wave / S::WR;
    const int r32 = lane & 31, hh = lane >> 5;
    const int64_t rows = (int64_t)a.B * a.Lq * a.Hq;
    float* const pm = a.pm + slot * rows + row;
    float* const pl = a.pl + slot * rows + row;

    const int n = key1 - key0;
    if (n <= 0) {                                          // (uniform over the workgroup)
        if (wk == 0 && valid && hh == 0) { *pm = -__builtin_inff(); *pl = 0.f; }
        return;
    }
    if constexpr (!FULL) {                                 // columns past D: zeros that no load overwrites
        for (int i = threadIdx.x; i < 2 * S::STAGE / 16; i += S::NW * 64)
            reinterpret_cast<v4u*>(lds)[i] = v4u{0, 0, 0, 0};
        bar();
    }
    // the row's query: B operand of K Q^T
    v8s qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int c = 2 * s + hh;
        if (FULL || c * 8 < a.D) qf[s] = *reinterpret_cast<const v8s*>(qrow + c * 16);
        else qf[s] = v8s{0, 0, 0, 0, 0, 0, 0, 0};
    }
    const uint32_t lds0 = lds_addr(lds);
    const int steps = (n + S::NKEY - 1) / S::NKEY;
    constexpr int RPL = 64 / CR;                           // key rows a direct load covers
    auto issue = [&](int i) INL {
        const char* kb = kbase + (int64_t)(key0 + i * S::NKEY) * kstride;
        const char* vb = vbase + (int64_t)(key0 + i * S::NKEY) * vstride;
        const uint32_t at = lds0 + (uint32_t)(i & 1) * S::STAGE;
        const int last = n - 1 - i * S::NKEY;              // rows past the segment's end: its last key
#pragma unroll
        for (int u = 0; u < S::LOADS; ++u) {
            const int r = (wave * S::LOADS + u) * RPL + lane / CR, sl = lane % CR;
            const int rr = min(r, last);
            const int ck = sl ^ kswz<CR>(r), cv = sl ^ vswz<CR>(r);
            const uint32_t to = (uint32_t)(wave * S::LOADS + u) * 1024u;
            if (FULL || ck * 8 < a.D) dma16(kb, (uint32_t)rr * (uint32_t)kstride + 16u * ck, at + to);
            if (FULL || cv * 8 < a.D) dma16(vb, (uint32_t)rr * (uint32_t)vstride + 16u * cv, at + S::KB + to);
        }
    };
    issue(0);

    v16f o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    float m = -__builtin_inff(), l = 0.f;
    const float c2 = a.scale2;
    // the first key that some row of this wave does not see
    int first = lim;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) first = min(first, __shfl_xor(first, x, 64));
    first = __builtin_amdgcn_readfirstlane(first);

    for (int i = 0; i < steps; ++i) {
        wait_all_dma();
        bar();
        if (i + 1 < steps) issue(i + 1);
        const char* const ks = lds + (i & 1) * S::STAGE;
        const char* const vs = ks + S::KB;
        const int at = key0 + i * S::NKEY + wk * KT;       // the wave's first key
        if (at >= key1) continue;

        v16f s[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
            const int kr = wk * KT + t * 32 + r32;
            const char* const krow = ks + kr * (DP * 2);
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                const v8s kf = *reinterpret_cast<const v8s*>(krow + (((2 * x + hh) ^ kswz<CR>(kr)) << 4));
                s[t] = E::mma(kf, qf[x], s[t]);
            }
        }
        const bool masked = at + KT > first;               // (uniform) keys that a row does not see
        if (masked) {
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (at + t * 32 + 8 * (r / 4) + 4 * hh + r % 4 >= lim) s[t][r] = -__builtin_inff();
        }
        float mt = s[0][0];
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[t][r]);
        mt = swap32_max(mt) * c2;
        // the maximum is raised, and o and l scaled, only where a score passes it by more than 2^8: the
        // weights stay below 2^8, exact in the same relative terms
        if (__any(mt > m + 8.f)) {
            const float mn = fmaxf(m, mt);
            const float al = mn > -__builtin_inff() ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
            m = mn;
            l *= al;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[t][r] *= al;
        }
        const float mu = m > -__builtin_inff() ? m : 0.f;  // (a row that has seen no key yet)
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], c2, -mu));
                l += s[t][r];
            }
        // o^T += V^T P^T: registers 8j .. 8j+7 of a score tile are this lane's keys 16j + 4 hh + 0..3
        // and 16j + 8 + 4 hh + 0..3, the order in which the values' transposing reads give them
        auto values = [&](int t, int j, int d) INL {
            typedef __attribute__((address_space(3))) v4s lv4s;
            const int kr = wk * KT + t * 32 + 16 * j + 4 * hh + (lane & 15) / 4;
            const int c = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            const char* const p0 = vs + kr * (DP * 2) + ((c ^ vswz<CR>(kr)) << 4) + 8 * (lane & 1);
            const char* const p1 = vs + (kr + 8) * (DP * 2) + ((c ^ vswz<CR>(kr + 8)) << 4) + 8 * (lane & 1);
            const v4s a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)p0);
            const v4s a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)p1);
            return __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        if (OWN && masked) {
            // an infinity or NaN among the values of a key that some row does not see would reach that
            // row as 0 * inf: such a step multiplies the finite values alone, and then adds the others to
            // the rows that see them
            uint32_t bad = 0;
            constexpr uint32_t EX = E::INF * 0x10001u, LO = (0x8000u - E::INF) * 0x10001u;
#pragma unroll 1
            for (int x = lane; x < KT * CR; x += 64) {
                const v4u w = reinterpret_cast<const v4u*>(vs + wk * KT * (DP * 2))[x];
                bad |= ((w[0] & EX) + LO) | ((w[1] & EX) + LO) | ((w[2] & EX) + LO) | ((w[3] & EX) + LO);
            }
            if (__any((bad & 0x80008000u) != 0)) {
#pragma unroll 1
                for (int kind = 0; kind < 4; ++kind) {     // finite, inf, -inf, NaN
                    const float add = kind == 1 ? __builtin_inff() : (kind == 2 ? -__builtin_inff() : __builtin_nanf(""));
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        __builtin_amdgcn_sched_barrier(0); // (not all columns at once: registers)
                        v16f c;
#pragma unroll
                        for (int r = 0; r < 16; ++r) c[r] = kind == 0 ? o[d][r] : 0.f;
#pragma unroll
                        for (int t = 0; t < TT; ++t)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                v8s va = values(t, j, d);
                                typename E::v8 p;
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const int key = at + t * 32 + 16 * j + 8 * (e / 4) + 4 * hh + e % 4;
                                    p[e] = (typename E::e)(kind == 0 ? s[t][8 * j + e] : (key < lim ? 1.f : 0.f));
                                    const uint16_t x = (uint16_t)va[e];
                                    const int is = (x & 0x7FFF) < E::INF ? 0 : ((x & 0x7FFF) > E::INF ? 3 : (x >> 15) + 1);
                                    va[e] = (short)(kind == is ? (kind == 0 ? x : E::ONE) : 0);
                                }
                                c = E::mma(va, __builtin_bit_cast(v8s, p), c);
                            }
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[d][r] = kind == 0 ? c[r] : (c[r] > 0.f ? o[d][r] + add : o[d][r]);
                    }
                }
                continue;
            }
        }
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                typename E::v8 p;
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = (typename E::e)s[t][8 * j + e];
                const v8s pb = __builtin_bit_cast(v8s, p);
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] = E::mma(values(t, j, d), pb, o[d]);
            }
    }
    l = swap32_sum(l);

    // the key shares of a row tile joined through LDS (o and l relative to a common m)
    if constexpr (S::WK > 1) {
        constexpr int ST = DP / 2 + 2;
        float* const x = reinterpret_cast<float*>(lds);
        bar();
        if (wk > 0) {
            float* const y = x + (((wk - 1) * S::WR + wr) * ST) * 64 + lane;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) y[(t * 16 + r) * 64] = o[t][r];
            y[(DP / 2) * 64] = m;
            y[(DP / 2 + 1) * 64] = l;
        }
        bar();
        if (wk > 0) return;
#pragma unroll
        for (int w = 1; w < S::WK; ++w) {
            const float* const y = x + (((w - 1) * S::WR + wr) * ST) * 64 + lane;
            const float m1 = y[(DP / 2) * 64], mn = fmaxf(m, m1);
            const float e0 = m > -__builtin_inff() ? __builtin_amdgcn_exp2f(m - mn) : 0.f;
            const float e1 = m1 > -__builtin_inff() ? __builtin_amdgcn_exp2f(m1 - mn) : 0.f;
            l = l * e0 + y[(DP / 2 + 1) * 64] * e1;
            m = mn;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[t][r] = o[t][r] * e0 + y[(t * 16 + r) * 64] * e1;
        }
    }
    if (!valid) return;
    if (hh == 0) { *pm = m; *pl = l; }
    float* const po = a.po + (slot * rows + row) * a.D;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = t * 32 + 8 * r + 4 * hh;
            if (FULL || d < a.D)
                *reinterpret_cast<v4f*>(po + d) = v4f{o[t][4 * r], o[t][4 * r + 1], o[t][4 * r + 2], o[t][4 * r + 3]};
        }
}

// Prefix: workgroup (head, row tile, split), the heads spread over the XCDs and a split's row tiles next
// to each other, so that one L2 serves them the same keys.  Own: workgroup (sequence, head, row tile,
// split).
template <class E, class S, bool FULL, bool OWN>
__global__ __launch_bounds__(S::NW * 64) void segment_kernel(AttnArgs a, int tiles) {
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Lq * a.G;
    const int h = blockIdx.x % a.Hkv;
    int x = blockIdx.x / a.Hkv;
    const int tile = x % tiles;
    x /= tiles;
    const int mrow = tile * S::BM + (wave % S::WR) * 32 + (lane & 31);
    if constexpr (!OWN) {
        const int M = a.B * R, split = x;
        const int mc = min(mrow, M - 1);
        const int b = mc / R, rem = mc - b * R, i = rem / a.G, g = rem - i * a.G;
        const int head = h * a.G + g;
        const int per = (((a.P + a.sp - 1) / a.sp) + 63) & ~63;
        const int key0 = min(split * per, a.P), key1 = min(key0 + per, a.P);
        segment_tile<E, S, FULL, OWN>(a, lds, a.pk + h * a.pkh, a.pks, a.pv + h * a.pvh, a.pvs, key0, key1, key1,
                                 a.q + b * a.qb + i * a.qt + head * a.qh, mrow < M, split,
                                 ((int64_t)b * a.Lq + i) * a.Hq + head);
    } else {
        const int b = x / a.ss, split = x % a.ss;
        const int len = min(max(a.lens[b], 0), a.T);
        const int mc = min(mrow, R - 1);
        const int i = mc / a.G, g = mc - i * a.G, head = h * a.G + g;
        const int ilast = min((tile + 1) * S::BM, R) - 1;
        const int seen = max(len - a.Lq + ilast / a.G + 1, 0);          // keys that the tile's last row sees
        const int per = (((seen + a.ss - 1) / a.ss) + 63) & ~63;
        const int key0 = min(split * per, seen), key1 = min(key0 + per, seen);
        segment_tile<E, S, FULL, OWN>(a, lds, a.k + b * a.kb + h * a.kh, a.kt, a.v + b * a.vb + h * a.vh, a.vt, key0, key1,
                                 min(len - a.Lq + i + 1, key1), a.q + b * a.qb + i * a.qt + head * a.qh, mrow < R,
                                 a.sp + split, ((int64_t)b * a.Lq + i) * a.Hq + head);
    }
}

// a thread: four columns of a row, over the row's partials
template <class E>
__global__ __launch_bounds__(256) void combine_kernel(AttnArgs a) {
    const int64_t rows = (int64_t)a.B * a.Lq * a.Hq;
    const int per = a.D / 4;
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= rows * per) return;
    const int64_t row = t / per;
    const int d = (int)(t - row * per) * 4;
    const int n = a.sp + a.ss;
    float m = -__builtin_inff();
    for (int s = 0; s < n; ++s) m = fmaxf(m, a.pm[s * rows + row]);
    float l = 0.f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < n; ++s) {
        const float ms = a.pm[s * rows + row];
        if (ms == -__builtin_inff()) continue;
        const float w = __builtin_amdgcn_exp2f(ms - m);
        l += w * a.pl[s * rows + row];
        const v4f x = *reinterpret_cast<const v4f*>(a.po + (s * rows + row) * a.D + d);
        o += w * x;
    }
    const float il = l == 0.f ? 0.f : 1.f / l;
    typename E::v4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (typename E::e)(o[j] * il);
    const int head = (int)(row % a.Hq);
    const int64_t bi = row / a.Hq;
    const int i = (int)(bi % a.Lq);
    const int64_t b = bi / a.Lq;
    *reinterpret_cast<typename E::v4*>(a.out + b * a.ob + i * a.ot + head * a.oh + d * 2) = y;
    if (a.lse && d == 0) a.lse[row] = m + __builtin_log2f(l);
}

// Own key weights: a wave takes 32 keys of a (sequence, head) and the R rows in tiles of 32, Q K^T with
// the keys along the columns, so that a lane sums its key's column in registers and nothing is atomic.
template <class E, int DP, bool FULL>
__global__ __launch_bounds__(256) void weights_kernel(AttnArgs a) {
    constexpr int KS = DP / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hh = lane >> 5;
    const int R = a.Lq * a.G;
    const int h = blockIdx.x % a.Hkv;
    int x = blockIdx.x / a.Hkv;
    const int nt = (a.T + 127) / 128;
    const int b = x / nt, t0 = (x % nt) * 128 + wave * 32;
    const int len = min(max(a.lens[b], 0), a.T);
    if (t0 >= len) return;
    const int key = t0 + r32;
    const char* const krow = a.k + b * a.kb + h * a.kh + (int64_t)min(key, len - 1) * a.kt;
    v8s kf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int c = 2 * s + hh;
        if (FULL || c * 8 < a.D) kf[s] = *reinterpret_cast<const v8s*>(krow + c * 16);
        else kf[s] = v8s{0, 0, 0, 0, 0, 0, 0, 0};
    }
    float sum = 0.f;
    for (int m0 = 0; m0 < R; m0 += 32) {
        const int mc = min(m0 + r32, R - 1), i = mc / a.G, g = mc - i * a.G;
        const char* const qrow = a.q + b * a.qb + i * a.qt + (h * a.G + g) * a.qh;
        v16f s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int u = 0; u < KS; ++u) {
            const int c = 2 * u + hh;
            v8s qf = v8s{0, 0, 0, 0, 0, 0, 0, 0};
            if (FULL || c * 8 < a.D) qf = *reinterpret_cast<const v8s*>(qrow + c * 16);
            s = E::mma(qf, kf[u], s);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int mr = m0 + 8 * (r / 4) + 4 * hh + r % 4;
            if (mr < R) {
                const int ii = mr / a.G, gg = mr - ii * a.G;
                if (key <= len - a.Lq + ii)
                    sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.scale2, -a.lse[((int64_t)b * a.Lq + ii) * a.Hq + h * a.G + gg]));
            }
        }
    }
    sum = swap32_sum(sum);
    if (hh == 0 && key < len) a.weights[((int64_t)b * a.Hkv + h) * a.T + key] += sum;
}

// ---- the host's side --------------------------------------------------------------------------

struct Plan {
    int bm_p, bm_o;                          // rows of a tile: prefix, own
    int sp, ss;                              // splits
    int64_t rows;
    int64_t bytes;
};

static int tile_rows(int rows) { return rows <= 32 ? 32 : (rows <= 64 ? 64 : 128); }

static Plan plan(int B, int Lq, int Hq, int Hkv, int D, int P, int T) {
    Plan p;
    const int R = Lq * (Hq / Hkv), cu = otpu_cu_count();
    const int64_t M = (int64_t)B * R;
    p.rows = (int64_t)B * Lq * Hq;
    p.bm_p = tile_rows((int)(M < 128 ? M : 128));
    p.bm_o = tile_rows(R < 128 ? R : 128);
    auto splits = [&](int64_t groups, int keys) {
        if (keys <= 0 || groups <= 0) return 0;
        int64_t s = (cu + groups - 1) / groups;
        const int most = (keys + 255) / 256;
        return (int)(s > most ? most : (s < 1 ? 1 : s));
    };
    p.sp = splits((int64_t)Hkv * ((M + p.bm_p - 1) / p.bm_p), P);
    p.ss = splits((int64_t)B * Hkv * ((R + p.bm_o - 1) / p.bm_o), T);
    const int64_t n = p.sp + p.ss;
    p.bytes = 4 * (n * p.rows * (D + 2) + p.rows) + 256;
    return p;
}

template <class E, class S, bool FULL>
static void launch_segment(const AttnArgs& a, bool own, hipStream_t s) {
    const int64_t m = own ? (int64_t)a.Lq * a.G : (int64_t)a.B * a.Lq * a.G;
    const int tiles = (int)((m + S::BM - 1) / S::BM);
    const int64_t grid = (int64_t)a.Hkv * tiles * (own ? (int64_t)a.B * a.ss : a.sp);
    if (own) segment_kernel<E, S, FULL, true><<<(unsigned)grid, S::NW * 64, 0, s>>>(a, tiles);
    else segment_kernel<E, S, FULL, false><<<(unsigned)grid, S::NW * 64, 0, s>>>(a, tiles);
}

template <class E, int DP, bool FULL>
static void launch_bm(const AttnArgs& a, bool own, int bm, hipStream_t s) {
    if constexpr (DP <= 128) {
        if (bm == 32) launch_segment<E, Shape<DP, 1, 4, 32>, FULL>(a, own, s);
        else if (bm == 64) launch_segment<E, Shape<DP, 2, 4, 32>, FULL>(a, own, s);
        else launch_segment<E, Shape<DP, 4, 2, 64>, FULL>(a, own, s);
    } else {
        if (bm == 32) launch_segment<E, Shape<DP, 1, 2, 32>, FULL>(a, own, s);
        else if (bm == 64) launch_segment<E, Shape<DP, 2, 2, 32>, FULL>(a, own, s);
        else launch_segment<E, Shape<DP, 4, 1, 32>, FULL>(a, own, s);
    }
}

template <class E, int DP, bool FULL>
static void launch_all(const AttnArgs& a, const Plan& p, hipStream_t s) {
    if (a.sp) launch_bm<E, DP, FULL>(a, false, p.bm_p, s);
    if (a.ss) launch_bm<E, DP, FULL>(a, true, p.bm_o, s);
    combine_kernel<E><<<(unsigned)((p.rows * (a.D / 4) + 255) / 256), 256, 0, s>>>(a);
    if (a.weights && a.T)
        weights_kernel<E, DP, FULL><<<(unsigned)((int64_t)a.B * a.Hkv * ((a.T + 127) / 128)), 256, 0, s>>>(a);
}

template <class E>
static void launch_type(const AttnArgs& a, const Plan& p, hipStream_t s) {
    if (a.D == 64) launch_all<E, 64, true>(a, p, s);
    else if (a.D < 64) launch_all<E, 64, false>(a, p, s);
    else if (a.D == 128) launch_all<E, 128, true>(a, p, s);
    else if (a.D < 128) launch_all<E, 128, false>(a, p, s);
    else if (a.D == 256) launch_all<E, 256, true>(a, p, s);
    else launch_all<E, 256, false>(a, p, s);
}

}  // namespace otpu

using namespace otpu;

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int check_sizes(const char* who, int B, int Lq, int Hq, int Hkv, int D, int P, int T) {
    if (B < 0 || Lq < 0 || P < 0 || T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv)
        return otpu_fail(OTPU_EINVAL, "%s: B %d, Lq %d, %d heads on %d, P %d, T %d", who, B, Lq, Hq, Hkv, P, T);
    if (D < 8 || D > 256 || D % 8) return otpu_fail(OTPU_EINVAL, "%s: heads of %d (a multiple of 8, at most 256)", who, D);
    if ((int64_t)B * Lq * Hq > (1 << 30) || (int64_t)B * Lq * Hq * D > (1ll << 36))
        return otpu_fail(OTPU_EINVAL, "%s: %lld rows of %d", who, (long long)B * Lq * Hq, D);
    return OTPU_OK;
}

extern "C" int64_t otpu_attn_work_bytes(int B, int Lq, int Hq, int Hkv, int D, int P, int T) {
    if (check_sizes("attn_work_bytes", B, Lq, Hq, Hkv, D, P, T)) return -1;
    return plan(B, Lq, Hq, Hkv, D, P, T).bytes;
}

extern "C" int otpu_attn_shared(const void* q, int64_t qb, int64_t qt, int64_t qh, const void* pk, int64_t pks,
                                int64_t pkh, const void* pv, int64_t pvs, int64_t pvh, int P, const void* k, int64_t kb,
                                int64_t kt, int64_t kh, const void* v, int64_t vb, int64_t vt, int64_t vh,
                                const int32_t* lens, int T, int B, int Lq, int Hq, int Hkv, int D, int dtype, float scale,
                                void* out, int64_t ob, int64_t ot, int64_t oh, float* weights, void* work,
                                int64_t work_bytes, otpu_stream_t stream) {
    if (dtype != OTPU_BF16 && dtype != OTPU_F16) return otpu_fail(OTPU_EFORMAT, "attn_shared: type %d (bf16, fp16)", dtype);
    if (const int rc = check_sizes("attn_shared", B, Lq, Hq, Hkv, D, P, T)) return rc;
    if (!(scale > 0.f) || scale > 1e30f) return otpu_fail(OTPU_EINVAL, "attn_shared: scale %g", (double)scale);
    if (B == 0 || Lq == 0) return OTPU_OK;
    if (!q || !out || !work || (P && (!pk || !pv)) || (T && (!k || !v || !lens)))
        return otpu_fail(OTPU_EINVAL, "attn_shared: a NULL operand");
    const int64_t st[] = {qb, qt, qh, P ? pks : 0, P ? pkh : 0, P ? pvs : 0, P ? pvh : 0, T ? kb : 0, T ? kt : 0,
                          T ? kh : 0, T ? vb : 0, T ? vt : 0, T ? vh : 0, ob, ot, oh};
    for (int64_t x : st)
        if (x % 8) return otpu_fail(OTPU_EALIGN, "attn_shared: a stride of %lld elements (multiples of 8)", (long long)x);
    const int64_t tok[] = {P ? pks : 0, P ? pvs : 0, T ? kt : 0, T ? vt : 0};
    for (int64_t x : tok)
        if (x < 0 || x >= (1 << 22)) return otpu_fail(OTPU_EINVAL, "attn_shared: tokens %lld elements apart", (long long)x);
    if (!al16(q) || !al16(out) || (P && (!al16(pk) || !al16(pv))) || (T && (!al16(k) || !al16(v))) ||
        ((uintptr_t)work & 255) || (T && ((uintptr_t)lens & 3)) || ((uintptr_t)weights & 3))
        return otpu_fail(OTPU_EALIGN, "attn_shared: operands 16-byte aligned, work 256-byte");
    const Plan p = plan(B, Lq, Hq, Hkv, D, P, T);
    if (work_bytes < p.bytes)
        return otpu_fail(OTPU_EINVAL, "attn_shared: work area of %lld bytes, need %lld", (long long)work_bytes,
                         (long long)p.bytes);
    AttnArgs a = {};
    a.q = (const char*)q; a.qb = 2 * qb; a.qt = 2 * qt; a.qh = 2 * qh;
    a.pk = (const char*)pk; a.pks = 2 * pks; a.pkh = 2 * pkh;
    a.pv = (const char*)pv; a.pvs = 2 * pvs; a.pvh = 2 * pvh;
    a.k = (const char*)k; a.kb = 2 * kb; a.kt = 2 * kt; a.kh = 2 * kh;
    a.v = (const char*)v; a.vb = 2 * vb; a.vt = 2 * vt; a.vh = 2 * vh;
    a.lens = lens;
    a.out = (char*)out; a.ob = 2 * ob; a.ot = 2 * ot; a.oh = 2 * oh;
    a.weights = weights;
    a.P = P; a.T = T; a.B = B; a.Lq = Lq; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.D = D;
    a.scale2 = scale * 1.4426950408889634f;
    a.sp = p.sp; a.ss = p.ss;
    const int64_t n = p.sp + p.ss;
    a.po = (float*)work;
    a.pm = a.po + n * p.rows * D;
    a.pl = a.pm + n * p.rows;
    a.lse = a.pl + n * p.rows;
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == OTPU_BF16) launch_type<BF16>(a, p, s);
    else launch_type<F16>(a, p, s);
    return otpu_launch_check("attn_shared");
}
