// Attention for a batch that shares a long prefix: each query sees all P keys of the shared prefix and
// its own sequence's keys up to its own place.  The softmax is split over key segments with a running
// maximum m and sum l of each (o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s), so the prefix is
// multiplied once by the rows of every sequence together and each sequence's cache by its own rows.
//
//   segment_kernel   one segment's share of the keys for a tile of rows: partial o, m, l
//   both_kernel      all keys for a tile of rows, where such tiles fill the CUs
//   combine_kernel   the partials of a row joined and rounded to the output's type; the own tokens'
//                    weights from their scores
//   weights_kernel   the weights where many rows would make the scores large: from the keys again
//
// What bounds it, by sizes (bf16, 16 heads on 8, heads of 128; whole calls, one after another): own keys and a
// prefix under few rows by memory (64 sequences on 1024 own tokens each 52 us, 5.2 TB/s; 16 on 65536 shared
// tokens 61 us, 4.4); many rows by the matrix units at the clock that their power leaves (8 x 512 queries on 8192
// tokens 297 us, 985 TFLOP/s; a library product of 8192^3 reaches 1190); the smallest calls by launches (one
// sequence on 128 shared tokens and up to 64 own: two, 8.5 us).
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
    static constexpr uint16_t INF = 0x7F80;
};
struct F16 {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    typedef _Float16 e;
    static __device__ __forceinline__ v16f mma(v8s a, v8s b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static constexpr uint16_t INF = 0x7C00;
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
    int sp, ss, per_p;                       // splits of the prefix, of the own keys; keys of a prefix split
    uint32_t np, no;                         // workgroups of the prefix, of the own keys
    uint32_t half;                           // own keys: order of the row tiles (find_part), or 0
    int rows_p, rows_o;                      // rows of their tiles: 32 or 128
    bool both;                               // a workgroup's rows against the prefix and their own keys (D <= 128)
    bool whole;                              // a row's only share is its output, nothing to join (D <= 128)
    float* po;                               // partial o [sp + ss][rows][D]
    float* pm;                               // m [sp + ss][rows]
    float* pl;                               // l [sp + ss][rows]
    float* lse;                              // [rows]: log2 of the softmax's sum, or NULL
    float* sc;                               // own scores [B, Hkv, R][tp], or NULL
    int64_t tp;
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// direct-to-LDS load: 16 bytes a lane, lane L's at lds + 16 L
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 : : "v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
// wait until at most N of this wave's loads are outstanding
template <int N>
__device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }
__device__ __forceinline__ void bar() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

__device__ __forceinline__ float swap32_max(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(v), false, false);
    return fmaxf(bitsf(p[0]), bitsf(p[1]));
}
__device__ __forceinline__ float swap32_sum(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(v), false, false);
    return bitsf(p[0]) + bitsf(p[1]);
}

// Two shapes of a workgroup of four waves:
//   rows   128 rows, 32 a wave, against the same keys: KT keys and values a step through LDS, two places each;
//          a step's scores are multiplied among the arithmetic of the step before
//   keys   32 rows (or fewer) against keys that every wave takes 32 at a time for itself, without a barrier:
//          its keys' next load is under way during the softmax and its values' product, its values' during
//          the next scores
// `keys` is bound by the loads of its keys whatever its rows, so 32 or fewer rows take it.
constexpr int NW = 4;
template <int DP_> struct Shape {
    static constexpr int DP = DP_;
    static constexpr int CR = DP / 8;                      // 16-byte chunks a key
    static constexpr int KT = DP <= 128 ? 64 : 32;         // rows: keys a step
    static constexpr int RB = KT * DP * 2;                 // ... their bytes, and their values'
    static constexpr int KB = 32 * DP * 2;                 // keys: a wave's keys' bytes, and its values'
    static constexpr int MERGE = (NW - 1) * 64 * (DP / 2 + 2) * 4;
    static constexpr int ROWS_LDS = 4 * RB, KEYS_LDS = NW * 2 * KB > MERGE + 4 ? NW * 2 * KB : MERGE + 4;
    static constexpr int LDS = ROWS_LDS > KEYS_LDS ? ROWS_LDS : KEYS_LDS;
};

// Chunk c of row r lies in slot c ^ f(r).  LDS serves 256 bytes a cycle from 64 banks.  Keys: the 16 rows
// that 16 lanes read at one c in 16 different slots (rows of 128 bytes: slots of both row parities).
// Values: the 4 rows by 4 chunks that 32 lanes of a transposing read take, likewise.
template <int CR> __device__ __forceinline__ int kswz(int r) { return CR < 16 ? (r >> 1) & 7 : r & 15; }
template <int CR> __device__ __forceinline__ int vswz(int r) { return CR < 16 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); }

// Direct loads of ROWS rows of a segment from row r0 on into LDS at `to`, dealt to W waves of which this is
// number w; rows past `last` (counted from r0) read it instead.
template <int CR, bool FULL, bool VAL, int ROWS, int W>
__device__ __forceinline__ void load_rows(const char* base, int64_t stride, int64_t r0, int last, uint32_t to, int w, int D) {
    constexpr int RPL = 64 / CR, LOADS = ROWS / RPL / W;   // rows a load covers, loads a wave issues
    const int lane = threadIdx.x & 63;
    const uint64_t b64 = (uint64_t)(base + r0 * stride);   // (uniform: into scalar registers)
    const char* const b = (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)b64) |
                                        (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b64 >> 32)) << 32);
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
        const int r = (w * LOADS + u) * RPL + lane / CR;
        const int c = (lane % CR) ^ (VAL ? vswz<CR>(r) : kswz<CR>(r));
        if (FULL || c * 8 < D)
            dma16(b, (uint32_t)min(r, last) * (uint32_t)stride + 16u * c, to + (uint32_t)(w * LOADS + u) * 1024u);
    }
}

// what a wave holds of its 32 rows: lane (r32, hh) the row r32, of o^T the columns 8 r + 4 hh + 0..3 of
// each 32, and half of the keys of l
template <int DP> struct Acc {
    v16f o[DP / 32];
    float m, l;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
        m = -__builtin_inff();
        l = 0.f;
    }
};

// An infinity or NaN among the values of a key that some row does not see would reach that row as
// 0 * inf.  So a step with such keys multiplies the finite values alone (the others are set to zero, which
// the result says), and add_infinite adds the others to the partials of the rows that see them.
template <class E>
__device__ __forceinline__ bool finite_values(char* vs, int pieces) {
    bool found = false;
    constexpr uint32_t EX = E::INF * 0x10001u, LO = (0x8000u - E::INF) * 0x10001u;
#pragma unroll 1
    for (int x = threadIdx.x & 63; x < pieces; x += 64) {
        v4u w = reinterpret_cast<const v4u*>(vs)[x];
        const v4u bad = ((w & EX) + LO) & 0x80008000u;     // bit 15 of each value that is not finite
        if ((bad[0] | bad[1] | bad[2] | bad[3]) != 0) {
            w &= ~((bad >> 15) * 0xFFFFu);
            reinterpret_cast<v4u*>(vs)[x] = w;
            found = true;
        }
    }
    return __any(found);
}

// Places past the segment's last key hold its values again: zeros instead, as an infinity would meet their
// weights of 0.
template <int CR>
__device__ __forceinline__ void clear_tail(char* vs, int from, int rows) {
    for (int x = from * CR + (int)(threadIdx.x & 63); x < rows * CR; x += 64) reinterpret_cast<v4u*>(vs)[x] = v4u{0, 0, 0, 0};
}

// S^T = K Q^T of 32 TT keys at ks (LDS): a lane has its row's scores of keys 8 r + 4 hh + 0..3 of each 32
template <class E, int DP, int TT>
__device__ __forceinline__ void scores(v16f (&s)[TT], const char* ks, const v8s (&qf)[DP / 16]) {
    constexpr int CR = DP / 8;
    const int lane = threadIdx.x & 63, r32 = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
    for (int x = 0; x < DP / 16; ++x) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int kr = t * 32 + r32;
            const v8s kf = *reinterpret_cast<const v8s*>(ks + kr * (DP * 2) + (((2 * x + hh) ^ kswz<CR>(kr)) << 4));
            s[t] = E::mma(kf, qf[x], s[t]);
        }
    }
}

// The running softmax over the scores of the segment's keys from `at` on, in two parts.  raise: scores that
// the row does not see made -inf, m, l and o brought up to the scores' maximum.  lim: the segment's keys that
// this lane's row sees; first: the least of the wave's.
template <int DP, int TT>
__device__ __forceinline__ void raise(Acc<DP>& a, v16f (&s)[TT], int at, int lim, int first, float c2) {
    const int hh = (threadIdx.x >> 5) & 1;
    if (at + 32 * TT > first) {                            // (uniform) keys that a row does not see
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
    // m is raised, and o and l scaled, only where a score passes it by more than 15, and then to 7 under the
    // score: weights of 2^7 to 2^15 for the largest keep fp16's subnormals (an error of 2^-25 whatever the
    // weight) 2^-32 below it, which 2^17 keys of one small weight would show otherwise; to fp32 sums and bf16
    // any m is the same
    if (__any(mt > a.m + 15.f)) {
        const float mn = fmaxf(a.m, mt - 7.f);
        const float al = mn > -__builtin_inff() ? __builtin_amdgcn_exp2f(a.m - mn) : 1.f;
        a.m = mn;
        a.l *= al;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) a.o[t][r] *= al;
    }
}

// The weights, their sum into l, rounded to 16 bits for the product.
template <class E, int DP, int TT>
__device__ __forceinline__ void weigh(Acc<DP>& a, const v16f (&s)[TT], v8s (&p)[2 * TT], float c2) {
    const float mu = a.m > -__builtin_inff() ? a.m : 0.f;  // (a row that has seen no key yet)
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            typename E::v8 w;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][8 * j + e], c2, -mu));
                a.l += x;
                w[e] = (typename E::e)x;
            }
            p[2 * t + j] = __builtin_bit_cast(v8s, w);
        }
}

// o^T += V^T P^T of the values at vs (LDS): p's eight weights are this lane's keys 16j + 4 hh + 0..3 and
// 16j + 8 + 4 hh + 0..3, the order in which the values' transposing reads give them
template <class E, int DP, int TT>
__device__ __forceinline__ void product(Acc<DP>& a, const char* vs, const v8s (&p)[2 * TT]) {
    constexpr int CR = DP / 8;
    typedef __attribute__((address_space(3))) v4s lv4s;
    const int lane = threadIdx.x & 63, hh = lane >> 5;
#pragma unroll
    for (int j = 0; j < 2 * TT; ++j) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
            const int kr = 16 * j + 4 * hh + (lane & 15) / 4;
            const int c = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            const char* const p0 = vs + kr * (DP * 2) + ((c ^ vswz<CR>(kr)) << 4) + 8 * (lane & 1);
            const char* const p1 = vs + (kr + 8) * (DP * 2) + ((c ^ vswz<CR>(kr + 8)) << 4) + 8 * (lane & 1);
            const v4s a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)p0);
            const v4s a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)p1);
            a.o[d] = E::mma(__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), p[j], a.o[d]);
        }
    }
}

// One workgroup's part: keys [key0, key1) of a segment for a tile of rows.
struct Part {
    const char *k, *v;                       // the segment's key 0 of the head
    int64_t ks, vs;                          // byte strides of a token
    int key0, key1, lim;                     // lim: the segment's keys that this lane's row sees
    int least;                               // the least of the workgroup's rows
    int head;                                // of the keys
    const char* q;                           // this lane's row
    bool valid;                              // a row of its own (not the clamped last one)
    int64_t at;                              // its place among the partials: (slot, row)
    float* sc;                               // its scores' row, or NULL
};

// a row (of q, or of k in its place): its columns 16 s + 8 hh + 0..7, an operand of the products
template <int DP, bool FULL>
__device__ __forceinline__ void load_query(v8s (&qf)[DP / 16], const char* q, int D) {
    const int hh = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int c = 2 * s + hh;
        if (FULL || c * 8 < D) qf[s] = *reinterpret_cast<const v8s*>(q + c * 16);
        else qf[s] = v8s{0, 0, 0, 0, 0, 0, 0, 0};
    }
}

// the output's row of a place among the partials of the only segment
__device__ __forceinline__ char* out_row(const AttnArgs& a, int64_t at) {
    const int row = (int)at, bi = row / a.Hq, head = row - bi * a.Hq, b = bi / a.Lq;
    return a.out + b * a.ob + (bi - b * a.Lq) * a.ot + head * a.oh;
}

template <class E, int DP, bool FULL>
__device__ __forceinline__ void store_part(const AttnArgs& a, const Acc<DP>& c, float l, const Part& p) {
    if (!p.valid) return;
    const int hh = (threadIdx.x >> 5) & 1;
    // (4096 queries of 16 heads on their own keys through a join: 118 us, without it 104; heads of 256 have no
    // registers for it)
    if (DP <= 128 && a.whole) {
        char* const out = out_row(a, p.at);
        const float il = l == 0.f ? 0.f : 1.f / l;
        if (a.lse && hh == 0) a.lse[p.at] = c.m + __builtin_log2f(l);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = t * 32 + 8 * r + 4 * hh;
                typename E::v4 z;
#pragma unroll
                for (int j = 0; j < 4; ++j) z[j] = (typename E::e)(c.o[t][4 * r + j] * il);
                if (FULL || d < a.D) *reinterpret_cast<typename E::v4*>(out + 2 * d) = z;
            }
        return;
    }
    // (a sum that is NaN counts in the join, also where no score was a number and raised m)
    if (hh == 0) { a.pm[p.at] = l == l ? c.m : 0.f; a.pl[p.at] = l; }
    float* const po = a.po + p.at * a.D;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = t * 32 + 8 * r + 4 * hh;
            if (FULL || d < a.D)
                *reinterpret_cast<v4f*>(po + d) = v4f{c.o[t][4 * r], c.o[t][4 * r + 1], c.o[t][4 * r + 2], c.o[t][4 * r + 3]};
        }
}

// the values that finite_values took out, from keys of tiles of KT, added to the partials of the wave's rows
// that see them
template <class E, int DP, int KT>
__device__ __forceinline__ void add_infinite(const AttnArgs& a, const Part& p) {
    const int lane = threadIdx.x & 63;
    const int from = p.key0 + max(p.least - p.key0, 0) / KT * KT;
    __threadfence();
    for (int r = 0; r < 32; ++r) {
        if (!__shfl((int)p.valid, r, 64)) continue;
        const int lim = __shfl(p.lim, r, 64);
        const int64_t at = __shfl(p.at, r, 64);
        float* const po = a.po + at * a.D;
        typename E::e* const out = reinterpret_cast<typename E::e*>(out_row(a, at));
        for (int d = lane; d < a.D; d += 64) {
            float add = 0.f;
            for (int t = from; t < lim; ++t) {
                const float x = (float)reinterpret_cast<const typename E::e*>(p.v + (int64_t)t * p.vs)[d];
                if (!(__builtin_fabsf(x) < __builtin_inff())) add += x;
            }
            if (DP <= 128 && add != 0.f && a.whole) out[d] = (typename E::e)((float)out[d] + add);
            else if (add != 0.f) po[d] += add;
        }
    }
}

// whether `x` holds in a wave of the workgroup; at: a word of LDS that no wave needs any more
__device__ __forceinline__ bool any_wave(char* at, bool x) {
    int* const word = reinterpret_cast<int*>(at);
    bar();
    *word = 0;
    bar();
    if (x) *word = 1;
    bar();
    return __builtin_amdgcn_readfirstlane(*word) != 0;
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o, 64));   // (both halves hold the same rows)
    return __builtin_amdgcn_readfirstlane(x);
}

// columns past D: zeros that no load overwrites
__device__ __forceinline__ void clear_lds(char* lds, int bytes) {
    for (int i = threadIdx.x; i < bytes / 16; i += NW * 64) reinterpret_cast<v4u*>(lds)[i] = v4u{0, 0, 0, 0};
    bar();
}

// Two workgroups a CU, a wave of each on a SIMD: the one's products fill the other's arithmetic in part (MFMA
// busy 51 to 56% of the cycles, at 1.9 GHz).  Two groups of waves that alternate at barriers instead, products beside
// softmax: 780 TFLOP/s against 990.  Keys loaded two steps ahead: no change, the loads are not waited for; four
// places of 32 keys in place of two of 64: the same to 10% slower, for the barriers.
// BOTH: the prefix's keys, then the own ones (p's), as one row of steps.
enum { PREFIX, OWN_KEYS, BOTH };
template <class E, int DP, bool FULL, int KIND>
__device__ __forceinline__ void rows_part(const AttnArgs& a, char* lds, const Part& p) {
    using S = Shape<DP>;
    constexpr bool OWN = KIND != PREFIX;
    constexpr int KT = S::KT, CR = S::CR, LOADS = KT / (64 / CR) / NW;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Acc<DP> c;
    c.clear();
    if (!FULL) clear_lds(lds, S::ROWS_LDS);
    v8s qf[DP / 16];
    load_query<DP, FULL>(qf, p.q, a.D);
    const uint32_t lds0 = lds_addr(lds);
    const int before = KIND == BOTH ? (a.P + KT - 1) / KT : 0;   // steps of the prefix in front of the segment's own
    const int n = p.key1 - p.key0, steps = before + (n + KT - 1) / KT;
    auto keys = [&](int i) INL {
        const uint32_t to = lds0 + (uint32_t)((i & 1) * S::RB);
        const bool own = KIND != BOTH || i >= before;
        const int at = own ? p.key0 + (i - before) * KT : i * KT, end = own ? p.key1 : a.P;
        load_rows<CR, FULL, false, KT, NW>(own ? p.k : a.pk + p.head * a.pkh, own ? p.ks : a.pks, at, end - 1 - at, to, wave, a.D);
    };
    auto vals = [&](int i) INL {
        const uint32_t to = lds0 + (uint32_t)((2 + (i & 1)) * S::RB);
        const bool own = KIND != BOTH || i >= before;
        const int at = own ? p.key0 + (i - before) * KT : i * KT, end = own ? p.key1 : a.P;
        load_rows<CR, FULL, true, KT, NW>(own ? p.v : a.pv + p.head * a.pvh, own ? p.vs : a.pvs, at, end - 1 - at, to, wave, a.D);
    };
    keys(0);
    vals(0);
    if (steps > 1) keys(1);
    const int first = wave_min(p.lim), none = -wave_min(-p.lim);
    bool bad = false;
    if (steps > 1) wait_dma<2 * LOADS>();                  // the first keys
    else wait_dma<LOADS>();
    bar();
    v16f s[KT / 32], next[KT / 32];
    v8s w[KT / 16];
    scores<E, DP>(s, lds, qf);
#pragma unroll 2
    for (int i = 0; i < steps; ++i) {
        wait_dma<0>();                                     // its values, the next keys
        bar();
        if (i + 1 < steps) vals(i + 1);
        if (i + 2 < steps) keys(i + 2);
        char* const vs = lds + (2 + (i & 1)) * S::RB;
        const bool own = KIND == OWN_KEYS || (KIND == BOTH && i >= before);
        const int at = KIND == BOTH && !own ? i * KT : p.key0 + (i - before) * KT, end = KIND == BOTH ? a.P : p.key1;
        if (own && at >= none) continue;                   // (uniform over the wave) no row of it sees these keys
        raise(c, s, at, KIND == BOTH && !own ? end : p.lim, KIND == BOTH && !own ? end : first, a.scale2);
        if (own && at + KT > p.least) bad |= finite_values<E>(vs, KT * CR);
        if (!own && at + KT > end) clear_tail<CR>(vs, end - at, KT);
        // the next scores' products among the weights' arithmetic (after the last step of a place's old keys, unused)
        scores<E, DP>(next, lds + ((i + 1) & 1) * S::RB, qf);
        weigh<E>(c, s, w, a.scale2);
        product<E, DP, KT / 32>(c, vs, w);
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) s[t] = next[t];
    }
    store_part<E, DP, FULL>(a, c, swap32_sum(c.l), p);
    if constexpr (OWN)
        if (any_wave(lds, bad)) add_infinite<E, DP, KT>(a, p);
}

// No barrier until the join: a wave's loads are its own, and 64 KB of LDS a workgroup leave two on a CU, 128 KB
// of keys and values under way or in use.
template <class E, int DP, bool FULL, bool OWN>
__device__ __forceinline__ void keys_part(const AttnArgs& a, char* lds, const Part& p) {
    using S = Shape<DP>;
    constexpr int CR = S::CR, LOADS = 32 / (64 / CR);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Acc<DP> c;
    c.clear();
    if (!FULL) clear_lds(lds, S::KEYS_LDS);
    char* const ks = lds + wave * 2 * S::KB;
    char* const vs = ks + S::KB;
    const uint32_t kl = lds_addr(ks), vl = lds_addr(vs);
    const int n = p.key1 - p.key0, tiles = (n + 31) / 32;
    auto keys = [&](int j) INL { load_rows<CR, FULL, false, 32, 1>(p.k, p.ks, p.key0 + 32 * j, n - 1 - 32 * j, kl, 0, a.D); };
    auto vals = [&](int j) INL { load_rows<CR, FULL, true, 32, 1>(p.v, p.vs, p.key0 + 32 * j, n - 1 - 32 * j, vl, 0, a.D); };
    v8s qf[DP / 16];
    load_query<DP, FULL>(qf, p.q, a.D);
    const int first = wave_min(p.lim);
    bool bad = false;
    if (wave < tiles) { keys(wave); vals(wave); }
    for (int j = wave; j < tiles; j += NW) {
        const bool more = j + NW < tiles;
        wait_dma<LOADS>();                                 // the keys are there; the values' loads are younger
        const int at = p.key0 + 32 * j;
        v16f s[1];
        v8s w[2];
        scores<E, DP>(s, ks, qf);
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
        if (more) keys(j + NW);
        if (OWN && p.sc) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<v4f*>(p.sc + at + 8 * r + 4 * (lane >> 5)) =
                    v4f{s[0][4 * r], s[0][4 * r + 1], s[0][4 * r + 2], s[0][4 * r + 3]};
        }
        raise(c, s, at, p.lim, first, a.scale2);
        weigh<E>(c, s, w, a.scale2);
        if (more) wait_dma<LOADS>();                       // (the next keys' loads are younger)
        else wait_dma<0>();
        if (OWN && at + 32 > p.least) bad |= finite_values<E>(vs, 32 * CR);
        if (!OWN && at + 32 > p.key1) clear_tail<CR>(vs, p.key1 - at, 32);
        product<E, DP, 1>(c, vs, w);
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
        if (more) vals(j + NW);
    }
    float l = swap32_sum(c.l);
    // the waves' shares joined through LDS
    constexpr int ST = DP / 2 + 2;
    float* const x = reinterpret_cast<float*>(lds);
    bar();
    if (wave > 0) {
        float* const y = x + (wave - 1) * ST * 64 + lane;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) y[(t * 16 + r) * 64] = c.o[t][r];
        y[(DP / 2) * 64] = c.m;
        y[(DP / 2 + 1) * 64] = l;
    }
    bar();
    const bool any_bad = OWN && any_wave(lds + S::MERGE, bad);
    if (wave > 0) return;
    for (int w = 0; w < NW - 1 && w + 1 < tiles; ++w) {
        const float* const y = x + w * ST * 64 + lane;
        const float m1 = y[(DP / 2) * 64], mn = fmaxf(c.m, m1);
        const float e0 = c.m > -__builtin_inff() ? __builtin_amdgcn_exp2f(c.m - mn) : 0.f;
        const float e1 = m1 > -__builtin_inff() ? __builtin_amdgcn_exp2f(m1 - mn) : 0.f;
        l = l * e0 + y[(DP / 2 + 1) * 64] * e1;
        c.m = mn;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) {
#pragma unroll
            for (int r = 0; r < 16; ++r) c.o[t][r] = c.o[t][r] * e0 + y[(t * 16 + r) * 64] * e1;
        }
    }
    store_part<E, DP, FULL>(a, c, l, p);
    if constexpr (OWN)
        if (any_bad) add_infinite<E, DP, 32>(a, p);
}

// The workgroups of the prefix, then those of the own keys.  Prefix: (head, row tile, split), the heads over
// the XCDs and a split's row tiles next to each other, so that one L2 serves them the same keys.  (Both
// kinds in turn, for the products of the one beside the loads of the other, takes that sharing from the
// row tiles: 256 sequences on 131072 tokens 743 us, one kind after the other 526.)  Own: (head, row tile,
// sequence, split), without a prefix a sequence's last rows first: they see the most keys (16384 queries on
// their own 1153 -> 1038 us, 4096 104 -> 96, 64 x 512 no difference; behind a prefix no gain, and heads of 256 lose 2%).  Where a prompt's row tiles all have
// their places at once and some CUs two, the first on the CUs (`half` a head) go from those of most keys
// down and the second from the least up, so that each CU has the same work: 8 x 512 queries on their own keys
// 27 -> 23 us, 4 x 1024 40 -> 32, 4096 96 -> 94.
// The part of workgroup x of its kind; `wrow`: this lane's row in a tile of bm rows; false: no key
__device__ __forceinline__ bool find_part(const AttnArgs& a, bool own, uint32_t x, int bm, int wrow, Part& p) {
    const int R = a.Lq * a.G;
    const int64_t rows = (int64_t)a.B * a.Lq * a.Hq;
    const int h = p.head = x % a.Hkv;
    x /= a.Hkv;
    if (!own) {
        const int M = a.B * R, tiles = (M + bm - 1) / bm;
        const int tile = x % tiles, split = x / tiles;
        const int mrow = tile * bm + wrow, mc = min(mrow, M - 1);
        const int b = mc / R, rem = mc - b * R, i = rem / a.G, head = h * a.G + rem - i * a.G;
        p.key0 = min(split * a.per_p, a.P);
        p.key1 = min(p.key0 + a.per_p, a.P);
        p.lim = p.least = p.key1;
        p.k = a.pk + h * a.pkh; p.ks = a.pks;
        p.v = a.pv + h * a.pvh; p.vs = a.pvs;
        p.q = a.q + b * a.qb + i * a.qt + head * a.qh;
        p.valid = mrow < M;
        p.at = split * rows + ((int64_t)b * a.Lq + i) * a.Hq + head;
        p.sc = nullptr;
    } else {
        const int tiles = (R + bm - 1) / bm;
        int tile = x % tiles, b = x / tiles % a.B;
        if (!a.np) tile = tiles - 1 - tile;
        const int split = x / tiles / a.B;
        if (a.half) {
            const uint32_t k = x < a.half ? x : (uint32_t)tiles * a.B - 1 - (x - a.half);
            tile = tiles - 1 - (int)(k / a.B);
            b = k % a.B;
        }
        const int mrow = tile * bm + wrow, mc = min(mrow, R - 1);
        const int i = mc / a.G, g = mc - i * a.G, head = h * a.G + g;
        const int len = min(max(a.lens[b], 0), a.T);
        const int seen = max(len - a.Lq + (min((tile + 1) * bm, R) - 1) / a.G + 1, 0);   // by the tile's last row
        const int per = ((seen + a.ss - 1) / a.ss + 31) & ~31;
        p.key0 = min(split * per, seen);
        p.key1 = min(p.key0 + per, seen);
        p.lim = min(len - a.Lq + i + 1, p.key1);
        p.least = min(len - a.Lq + tile * bm / a.G + 1, p.key1);
        p.k = a.k + b * a.kb + h * a.kh; p.ks = a.kt;
        p.v = a.v + b * a.vb + h * a.vh; p.vs = a.vt;
        p.q = a.q + b * a.qb + i * a.qt + head * a.qh;
        p.valid = mrow < R;
        p.at = (a.sp + split) * rows + ((int64_t)b * a.Lq + i) * a.Hq + head;
        p.sc = a.sc && p.valid ? a.sc + (((int64_t)b * a.Hkv + h) * R + mc) * a.tp : nullptr;
    }
    if (p.key1 > p.key0 || a.both) return true;            // (uniform over the workgroup)
    if (p.valid && (threadIdx.x & 63) < 32) {
        if (a.whole) {
            char* const out = out_row(a, p.at);
            for (int d = 0; d < a.D; d += 8) *reinterpret_cast<v4u*>(out + 2 * d) = v4u{0, 0, 0, 0};
        } else {
            a.pm[p.at] = -__builtin_inff();
            a.pl[p.at] = 0.f;
        }
    }
    return false;
}

template <class E, int DP, bool FULL>
__global__ __launch_bounds__(NW * 64, DP <= 128 ? 2 : 1) void segment_kernel(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[Shape<DP>::LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool own = blockIdx.x >= a.np, keys = (own ? a.rows_o : a.rows_p) == 32;
    Part p;
    if (!find_part(a, own, own ? blockIdx.x - a.np : blockIdx.x, keys ? 32 : 32 * NW, (keys ? 0 : wave * 32) + (lane & 31), p))
        return;
    if (!own) {
        if (keys) keys_part<E, DP, FULL, false>(a, lds, p);
        else rows_part<E, DP, FULL, PREFIX>(a, lds, p);
    } else {
        if (keys) keys_part<E, DP, FULL, true>(a, lds, p);
        else rows_part<E, DP, FULL, OWN_KEYS>(a, lds, p);
    }
}

// A sequence's tile of 128 rows against the prefix and its own keys (a kernel of its own: in segment_kernel its
// addresses would not stay in scalar registers).  16 x 256 queries on 1024 shared tokens and their own, 16 heads
// on 8 of 128: 77 -> 51 us; 4 x 2048 on 2048 276 -> 229, 8 x 512 on 8192 and up to 1024 own tokens 318 -> 297.
template <class E, int DP, bool FULL>
__global__ __launch_bounds__(NW * 64, 2) void both_kernel(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[Shape<DP>::ROWS_LDS];
    Part p;
    find_part(a, true, blockIdx.x, 32 * NW, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32 + (threadIdx.x & 31), p);
    rows_part<E, DP, FULL, BOTH>(a, lds, p);
}

// The partials of a row joined: GP threads take every GP-th partial of four columns, their sums meet in
// LDS.  The first nw workgroups add the own tokens' weights from the scores: 1024 tokens of a (sequence,
// head) each, the rows' sums joined again.
constexpr int WT = 1024;
template <class E, int GP>
__global__ __launch_bounds__(256) void combine_kernel(AttnArgs a, int nw) {
    __shared__ float sm[256], sl[256];
    __shared__ v4f so[256];
    const int64_t rows = (int64_t)a.B * a.Lq * a.Hq;
    const int n = a.sp + a.ss, tid = threadIdx.x;
    if ((int)blockIdx.x < nw) {
        const int R = a.Lq * a.G, nt = (a.T + WT - 1) / WT;
        const int x = blockIdx.x, bh = x / nt, t0 = x % nt * WT;
        const int b = bh / a.Hkv, h = bh - b * a.Hkv;
        const int len = min(max(a.lens[b], 0), a.T);
        if (t0 >= len) return;
        const int t = t0 + 4 * tid;
        const float* const sc = a.sc + (int64_t)bh * R * a.tp + min(t, (int)a.tp - 4);
        v4f s[8];                                          // eight rows' scores, on their way during the sums
        auto load = [&](int r0) INL {
#pragma unroll
            for (int u = 0; u < 8; ++u) s[u] = *reinterpret_cast<const v4f*>(sc + (int64_t)min(r0 + u, R - 1) * a.tp);
        };
        load(0);
        // (R <= 32) a row's lse: 8 threads over its partials
        {
            const int r = min(tid >> 3, R - 1), i = r / a.G;
            const int64_t row = ((int64_t)b * a.Lq + i) * a.Hq + h * a.G + r - i * a.G;
            float m = -__builtin_inff(), l = 0.f;
            for (int k0 = tid & 7; k0 < n; k0 += 32) {
                float ms[4], ls[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t at = min(k0 + 8 * u, n - 1) * rows + row;
                    ms[u] = a.pm[at];
                    ls[u] = a.pl[at];
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float mn = fmaxf(m, ms[u]);
                    if (k0 + 8 * u < n && mn > -__builtin_inff()) {
                        l = l * __builtin_amdgcn_exp2f(m - mn) + ls[u] * __builtin_amdgcn_exp2f(ms[u] - mn);
                        m = mn;
                    }
                }
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                const float m1 = __shfl_xor(m, o, 64), l1 = __shfl_xor(l, o, 64), mn = fmaxf(m, m1);
                if (mn > -__builtin_inff()) l = l * __builtin_amdgcn_exp2f(m - mn) + l1 * __builtin_amdgcn_exp2f(m1 - mn);
                m = mn;
            }
            if ((tid & 7) == 0) sm[tid >> 3] = m + __builtin_log2f(l);
        }
        __syncthreads();
        if (t >= len) return;
        v4f w = {0.f, 0.f, 0.f, 0.f};
        for (int r0 = 0; r0 < R; r0 += 8) {
            if (r0) load(r0);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int see = r0 + u < R ? len - a.Lq + (r0 + u) / a.G : -1;   // the row's own token
                const float lse = sm[min(r0 + u, R - 1)];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (t + j <= see) w[j] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j], a.scale2, -lse));
            }
        }
        float* const out = a.weights + (int64_t)bh * a.T + t;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (t + j < len) out[j] += w[j];
        return;
    }
    const int per = a.D / 4, rpb = 256 / (per * GP);       // rows a workgroup
    const int rl = tid / (per * GP), y = tid - rl * per * GP, g = y / per, d = (y - g * per) * 4;
    // rows of one head of the keys, on the XCD whose L2 its partials were written through
    const int x = blockIdx.x - nw, hk = x % a.Hkv, R = a.Lq * a.G;
    const int64_t mr = (int64_t)(x / a.Hkv) * rpb + rl;    // (b, i, g)
    const bool ok = rl < rpb && mr < (int64_t)a.B * R;
    const int64_t bi = mr / a.G;
    const int head = hk * a.G + (int)(mr - bi * a.G);
    const int64_t row = bi * a.Hq + head;
    float m = -__builtin_inff(), l = 0.f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
    if (ok) {
        constexpr int U = 4;                               // partials whose loads go out together
        for (int s0 = g; s0 < n; s0 += U * GP) {
            float ms[U], ls[U];
            v4f os[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * GP;
                ms[u] = -__builtin_inff();
                ls[u] = 0.f;
                if (s < n) {
                    ms[u] = a.pm[s * rows + row];
                    ls[u] = a.pl[s * rows + row];
                    os[u] = *reinterpret_cast<const v4f*>(a.po + (s * rows + row) * a.D + d);
                }
            }
            float mn = m;
#pragma unroll
            for (int u = 0; u < U; ++u) mn = fmaxf(mn, ms[u]);
            if (mn == -__builtin_inff()) continue;
            const float e = __builtin_amdgcn_exp2f(m - mn);
            l *= e;
            o *= e;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (ms[u] > -__builtin_inff()) {           // (a share without a key has no o)
                    const float w = __builtin_amdgcn_exp2f(ms[u] - mn);
                    l += w * ls[u];
                    o += w * os[u];
                }
            m = mn;
        }
    }
    if constexpr (GP > 1) {
        sm[tid] = m;
        sl[tid] = l;
        so[tid] = o;
        __syncthreads();
        if (!ok || g > 0) return;
#pragma unroll
        for (int k = 1; k < GP; ++k) {
            const float m1 = sm[tid + k * per];
            if (m1 == -__builtin_inff()) continue;
            const float mn = fmaxf(m, m1), e0 = __builtin_amdgcn_exp2f(m - mn), e1 = __builtin_amdgcn_exp2f(m1 - mn);
            l = l * e0 + sl[tid + k * per] * e1;
            o = o * e0 + so[tid + k * per] * e1;
            m = mn;
        }
    }
    if (!ok) return;
    const float il = l == 0.f ? 0.f : 1.f / l;
    typename E::v4 z;
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = (typename E::e)(o[j] * il);
    const int64_t b = bi / a.Lq;
    const int i = (int)(bi - b * a.Lq);
    *reinterpret_cast<typename E::v4*>(a.out + b * a.ob + i * a.ot + head * a.oh + d * 2) = z;
    if (a.lse && d == 0) a.lse[row] = m + __builtin_log2f(l);
}

// Own key weights where R > 32 rows see a (sequence, head)'s keys (up to 32 their scores are kept: at 32 half of the
// keys' bytes for heads of 128, all of them for 64, 8 times them for 8): a workgroup takes 32 keys of a (sequence, head), its waves the rows in tiles of 32 by turns.  As in `scores` a lane has one row
// and 16 of the keys, so that the row's lse is its own and the sums over row tiles stay in registers; lanes and
// waves are summed once at the end, in one order, and nothing is atomic.  (82 x 13 queries, 15 heads on 3 of 128, on
// up to 786 own tokens 24 us.  128 keys a workgroup, each wave all rows for its own 32, read the queries a quarter as
// often with fewer waves a SIMD: the call 56 us against 58, 16 x 64 queries on 2048 tokens 103 against 118, but 8 x 512
// on up to 1024 102 against 90.)
template <class E, int DP, bool FULL>
__global__ __launch_bounds__(NW * 64) void weights_kernel(AttnArgs a) {
    constexpr int KS = DP / 16;
    __shared__ float part[NW][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hh = lane >> 5;
    const int R = a.Lq * a.G;
    const int h = blockIdx.x % a.Hkv;
    const int x = blockIdx.x / a.Hkv;
    const int nt = (a.T + 31) / 32;
    const int b = x / nt, t0 = (x % nt) * 32;
    const int len = min(max(a.lens[b], 0), a.T), own = len - a.Lq;
    if (t0 >= len) return;                                 // (uniform over the workgroup)
    const char* const krow = a.k + b * a.kb + h * a.kh + (int64_t)min(t0 + r32, len - 1) * a.kt;
    v8s kf[KS];
    load_query<DP, FULL>(kf, krow, a.D);
    float sum[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.f;
    // rows of tokens before own + t0 see none of the keys
    for (int m0 = (max(t0 - own, 0) * a.G & ~31) + 32 * wave; m0 < R; m0 += 32 * NW) {
        const int mc = min(m0 + r32, R - 1), i = mc / a.G, head = h * a.G + mc - i * a.G;
        const float lse = a.lse[((int64_t)b * a.Lq + i) * a.Hq + head];
        v8s qf[KS];
        load_query<DP, FULL>(qf, a.q + b * a.qb + i * a.qt + head * a.qh, a.D);
        v16f s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int u = 0; u < KS; ++u) s = E::mma(kf[u], qf[u], s);
        const int see = m0 + r32 < R ? own + i : -1;       // the row's own token
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (t0 + 8 * (r / 4) + 4 * hh + r % 4 <= see) sum[r] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.scale2, -lse));
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float v = sum[r];                                  // over the 32 rows: DPP within 16 lanes, then their pair
        v += bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(v), 0xB1, 0xF, 0xF, false));
        v += bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(v), 0x4E, 0xF, 0xF, false));
        v += bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(v), 0x141, 0xF, 0xF, false));
        v += bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(v), 0x140, 0xF, 0xF, false));
        const auto p = __builtin_amdgcn_permlane16_swap(fbits(v), fbits(v), false, false);
        v = bitsf(p[0]) + bitsf(p[1]);
        if (r32 == 0) part[wave][8 * (r / 4) + 4 * hh + r % 4] = v;
    }
    __syncthreads();
    if (threadIdx.x < 32 && t0 + (int)threadIdx.x < len) {
        float v = part[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += part[w][threadIdx.x];
        a.weights[((int64_t)b * a.Hkv + h) * a.T + t0 + threadIdx.x] += v;
    }
}

// ---- the host's side --------------------------------------------------------------------------

struct Plan {
    int rows_p, rows_o;                      // rows of a tile: prefix, own
    int sp, ss, per_p;                       // splits; keys of a prefix split
    int64_t np, no;                          // workgroups
    int64_t rows, tp;
    bool both;                               // one segment of the prefix and the own keys
    bool whole;                              // one share a row, stored as its output
    bool scores;                             // own scores kept for the weights
    int64_t po, pm, pl, lse, sc, bytes;      // the work area's parts, in floats; its size
};

// weights: the call asks for them.  any: the parts that some call of these sizes uses.
static Plan plan(int B, int Lq, int Hq, int Hkv, int D, int P, int T, bool weights, bool any = false) {
    Plan p = {};
    const int R = Lq * (Hq / Hkv);
    const int64_t M = (int64_t)B * R, slots = 2 * (int64_t)otpu_cu_count();
    p.rows = (int64_t)B * Lq * Hq;
    // (own keys of up to 64 rows: two tiles of 32 read them from the L2; 16 x 24 queries, 4 heads on 2, on 200 own
    // tokens 9.2 us, a tile of 128 12.8.  A prefix: no difference.)
    p.rows_p = M <= 32 ? 32 : 32 * NW;
    p.rows_o = R <= 64 ? 32 : 32 * NW;
    const int64_t gp = (int64_t)Hkv * ((M + p.rows_p - 1) / p.rows_p);
    const int64_t go = (int64_t)B * Hkv * ((R + p.rows_o - 1) / p.rows_o);
    // Splits: as many as fill the places of the CUs, of `least` keys or more.  (Two places a CU, also for the copy of
    // 256 columns, which has one: 64 sequences on 16384 tokens and up to 1024 own, heads of 256, 121 us, counted as one
    // 136; 16 on 65536 125 against 110.)
    auto splits = [&](int64_t groups, int64_t keys, int64_t least) {
        if (keys <= 0 || groups <= 0) return (int64_t)0;
        const int64_t s = (slots + groups - 1) / groups, most = (keys + least - 1) / least;
        return s > most ? most : s;
    };
    p.ss = (int)splits(go, T, 256);
    p.no = go * p.ss;
    int64_t s = splits(gp, P, p.rows_p == 32 ? 128 : 64);
    if (p.rows_p > 32 && s > 1) {
        // A tile of 128 rows writes 64 KB of partials a split, read once more, where another split saves
        // each workgroup steps: the sum is least near sqrt(P / (2 groups)) (64 sequences on 4096 tokens, 8
        // groups: 8, 16 and 32 splits 19.0, 15.7 and 16.7 us; on 16384 16, 32 and 64 29.8, 25.4 and 29.8).
        // Half of that beside own keys that fill the CUs: there the steps' latency does not count (64
        // sequences on 16384, up to 1024 own tokens: 32 splits 65 us, 16 62, 8 71).
        const int64_t r = (int64_t)__builtin_ceil(__builtin_sqrt((double)P / (2.0 * (double)gp)));
        if (r < s) s = p.no >= slots / 2 ? (r + 1) / 2 : r;
    }
    p.sp = (int)s;
    p.per_p = p.sp ? ((P + p.sp - 1) / p.sp + 31) & ~31 : 0;
    p.np = gp * p.sp;
    // Tiles of a sequence's rows that fill the places take the prefix and their own keys in one: no partials, no
    // join.  Where sequences leave little of their last tiles free (1 in 20 rows at most).
    p.both = D <= 128 && p.sp == 1 && p.ss == 1 && p.rows_o == 128 && 20 * 128 * (go / Hkv) <= 21 * M;
    if (p.both) {
        p.sp = 0;
        p.np = 0;
    }
    p.scores = weights && T && R <= 32;
    p.whole = p.both || (D <= 128 && p.sp + p.ss == 1 && !p.scores);
    p.tp = (T + 31) & ~31;
    const int64_t n = p.whole && !any ? 0 : p.sp + p.ss;   // partials
    auto part = [&](int64_t floats) {
        const int64_t at = p.bytes / 4;
        p.bytes += (4 * floats + 255) & ~(int64_t)255;
        return at;
    };
    p.po = part(n * p.rows * D);
    p.pm = part(n * p.rows);
    p.pl = part(n * p.rows);
    p.lse = part(any || (weights && T && !p.scores) ? p.rows : 0);
    p.sc = part(p.scores || (any && R <= 32) ? (int64_t)B * Hkv * R * p.tp : 0);
    return p;
}

template <class E, int GP>
static void launch_combine(const AttnArgs& a, const Plan& p, hipStream_t s) {
    const int rpb = 256 / (a.D / 4 * GP);
    const int nrows = a.Hkv * (int)(((int64_t)a.B * a.Lq * a.G + rpb - 1) / rpb);
    const int nw = a.sc ? a.B * a.Hkv * ((a.T + WT - 1) / WT) : 0;
    combine_kernel<E, GP><<<nrows + nw, 256, 0, s>>>(a, nw);
}

template <class E, int DP, bool FULL>
static void launch_all(const AttnArgs& a, const Plan& p, hipStream_t s) {
    if constexpr (DP <= 128)
        if (a.both) both_kernel<E, DP, FULL><<<(unsigned)p.no, NW * 64, 0, s>>>(a);
    if (!a.both && p.np + p.no) segment_kernel<E, DP, FULL><<<(unsigned)(p.np + p.no), NW * 64, 0, s>>>(a);
    // threads a partial's row: by how many partials there are (at most 256 in all: D / 4 columns' threads)
    const int n = p.sp + p.ss;
    if (a.whole) {}
    else if (n > 8) launch_combine<E, 4>(a, p, s);
    else if (n > 2) launch_combine<E, 2>(a, p, s);
    else launch_combine<E, 1>(a, p, s);
    if (a.weights && a.T && !a.sc)
        weights_kernel<E, DP, FULL><<<(unsigned)((int64_t)a.B * a.Hkv * ((a.T + 31) / 32)), NW * 64, 0, s>>>(a);
}

template <class E>
static void launch_type(const AttnArgs& a, const Plan& p, hipStream_t s) {
    if (a.D == 64) launch_all<E, 64, true>(a, p, s);
    else if (a.D < 64) launch_all<E, 64, false>(a, p, s);
    else if (a.D == 128) launch_all<E, 128, true>(a, p, s);
    else if (a.D < 128) launch_all<E, 128, false>(a, p, s);
    else launch_all<E, 256, false>(a, p, s);              // (256 too: the copy for whole rows spills registers)
}

}  // namespace otpu

using namespace otpu;

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int check_sizes(const char* who, int B, int Lq, int Hq, int Hkv, int D, int P, int T) {
    if (B < 0 || Lq < 0 || P < 0 || P > (1 << 30) || T < 0 || T > (1 << 30) || Hq < 1 || Hkv < 1 || Hq % Hkv)
        return otpu_fail(OTPU_EINVAL, "%s: B %d, Lq %d, %d heads on %d, P %d, T %d", who, B, Lq, Hq, Hkv, P, T);
    if (D < 8 || D > 256 || D % 8) return otpu_fail(OTPU_EINVAL, "%s: heads of %d (a multiple of 8, at most 256)", who, D);
    // (a launch holds fewer than 2^32 threads)
    const int64_t rows = (int64_t)B * Lq * Hq;
    if (rows > (1 << 23) || (int64_t)B * Hkv * ((T + 31) / 32) >= (1 << 24))
        return otpu_fail(OTPU_EINVAL, "%s: %lld rows (at most 2^23), %d x %d caches of %d tokens (below 2^24 pieces of 32)", who,
                         (long long)rows, B, Hkv, T);
    return OTPU_OK;
}

extern "C" int64_t otpu_attn_work_bytes(int B, int Lq, int Hq, int Hkv, int D, int P, int T) {
    if (check_sizes("attn_work_bytes", B, Lq, Hq, Hkv, D, P, T)) return -1;
    return plan(B, Lq, Hq, Hkv, D, P, T, false, true).bytes;
}

extern "C" int64_t otpu_attn_call_bytes(int B, int Lq, int Hq, int Hkv, int D, int P, int T, int weights) {
    if (check_sizes("attn_call_bytes", B, Lq, Hq, Hkv, D, P, T)) return -1;
    return plan(B, Lq, Hq, Hkv, D, P, T, weights != 0).bytes;
}

extern "C" int otpu_attn_shared(const otpu_attn_args* args, otpu_stream_t stream) {
    if (!args || args->bytes != (int64_t)sizeof(otpu_attn_args))
        return otpu_fail(OTPU_EINVAL, "attn_shared: the arguments' size is not this header's %d", (int)sizeof(otpu_attn_args));
    const auto [bytes, q, qb, qt, qh, pk, pks, pkh, pv, pvs, pvh, k, kb, kt, kh, v, vb, vt, vh, lens, out, ob, ot, oh, weights,
                work, work_bytes, B, Lq, Hq, Hkv, D, P, T, dtype, scale] = *args;
    if (dtype != OTPU_BF16 && dtype != OTPU_F16) return otpu_fail(OTPU_EFORMAT, "attn_shared: type %d (bf16, fp16)", dtype);
    if (const int rc = check_sizes("attn_shared", B, Lq, Hq, Hkv, D, P, T)) return rc;
    // (0 in fp32 would make NaN of the keys that a row does not see)
    const float scale2 = (float)(scale * 1.4426950408889634);
    if (!(scale2 > 0.f) || scale > 1e30) return otpu_fail(OTPU_EINVAL, "attn_shared: scale %g", scale);
    if (B == 0 || Lq == 0) return OTPU_OK;
    const Plan p = plan(B, Lq, Hq, Hkv, D, P, T, weights != nullptr);
    if (!q || !out || (!work && (p.bytes || work_bytes)) || (P && (!pk || !pv)) || (T && (!k || !v || !lens)))
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
    if (work_bytes != p.bytes) {
        const int64_t any = plan(B, Lq, Hq, Hkv, D, P, T, false, true).bytes;
        if (work_bytes < any)
            return otpu_fail(OTPU_EINVAL, "attn_shared: work area of %lld bytes, need %lld, or this call's %lld", (long long)work_bytes,
                             (long long)any, (long long)p.bytes);
    }
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
    a.scale2 = scale2;
    a.sp = p.sp; a.ss = p.ss; a.per_p = p.per_p;
    a.np = (uint32_t)p.np; a.no = (uint32_t)p.no;
    a.rows_p = p.rows_p; a.rows_o = p.rows_o;
    float* const f = (float*)work;
    a.po = f + p.po; a.pm = f + p.pm; a.pl = f + p.pl;
    a.tp = p.tp;
    if (weights && T) {
        if (p.scores) a.sc = f + p.sc;
        else a.lse = f + p.lse;
    }
    a.both = p.both;
    a.whole = p.whole;
    const int cus = otpu_cu_count();
    if (!p.np && p.ss == 1 && Lq > 1 && p.no > cus && p.no <= 2 * (int64_t)cus) a.half = (uint32_t)(cus / Hkv);
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == OTPU_BF16) launch_type<BF16>(a, p, s);
    else launch_type<F16>(a, p, s);
    return otpu_launch_check("attn_shared");
}
