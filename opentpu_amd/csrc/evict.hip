// Eviction from a key/value cache by accumulated attention weight.  Of a (sequence, head)'s n slots the
// `budget` slots stay that come first by (recent, weight, slot): the newest positions always, then the
// largest weights, the lower slot where weights are equal.  The j-th slot below the budget that goes takes
// over the j-th slot at or past it that stays: attention does not ask for an order of slots, so only the
// holes are filled, sources and destinations are disjoint and every move is independent.
//
//   evict_select_kernel   a workgroup a (sequence, head): the threshold by radix selection (11, 11 and 10
//                         bits), the holes and their sources, the slots' weights and positions; up to 64
//                         rows of k and v
//   evict_move_kernel     more rows of k and v, and the slots that are free
//
// The moves are bound by memory (64 x 8 caches of 2048 slots cut to 1000: 268 MB read and written, 65 us after a
// selection of 15, 4.1 TB/s; a copy reaches 5.1).  The selection is a chain of a few trips to memory, three
// passes over keys in registers with three barriers each, and a scan: 8 us for 256 caches of 1024 slots with
// the launch, 27 for caches of 32768, where one workgroup's instructions bound it.
#include "otpu_common.h"

namespace otpu {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int EW = 1024;                     // threads of a selecting workgroup
constexpr int BINS = 2048;
// Moves that the selecting workgroup makes itself, with the free slots' clearing: a launch less, whatever the slots.
// 256 caches of 16-bit rows of 64 cut to 64 slots, of 1024: 9.4 us, moved and cleared by the second kernel 11.9; of
// 32768 slots 36.4 and 41.0; 8 caches of 32768 22.9 and 24.3.
constexpr int HERE = 64;

struct EvictArgs {
    char* k; int64_t kb, kt, kh;             // byte strides of sequence, slot, head
    char* v; int64_t vb, vt, vh;
    int row;                                 // bytes of a row (of one head)
    const float* w;                          // [B, H, T]
    const int32_t* pos;
    const int32_t* lens;
    int B, T, H, budget, recent;
    float* wn; int32_t* pn; int32_t* ln;     // the new ones (may be the old ones)
    int* count;                              // [B H] moves
    int2* moves;                             // [B H][most] (to, from)
    int most;
    bool here;                               // few moves: the selecting workgroup makes them
};

// weights in the order of the selection: NaN above infinity, -0 with +0
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xFFC00000u;
    const uint32_t u = fbits(w + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// inclusive sums over 16 lanes of a row, and over the wave (DPP row_shr 1, 2, 4, 8, row_bcast 15 and 31)
__device__ __forceinline__ int row_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    return x + __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
}
__device__ __forceinline__ int wave_scan(int x) {
    x = row_scan(x);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
}

// exclusive sum of v over the workgroup's threads, in thread order; total: the whole sum.  tmp: EW / 64
// words that the next call does not use.  Every lane of every wave takes part.
static_assert(EW / 64 == 16, "the waves' sums in a row of 16 lanes");
__device__ __forceinline__ int block_scan(int v, int* tmp, int& total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = wave_scan(v);
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    const int y = row_scan(tmp[lane & 15]);
    total = __builtin_amdgcn_readlane(y, 15);
    return (wave ? __builtin_amdgcn_readlane(y, wave - 1) : 0) + x - v;
}

// rows of k and v from slot m.y to slot m.x, `c` pieces of 16 bytes each: threads in groups of c (or all of
// them for one row), several rows' loads out at once
template <int THREADS, int U>
__device__ __forceinline__ void move_rows(const EvictArgs& a, char* k, char* v, const int2* mv, int n, int first, int step) {
    const int c = a.row / 16, per = c < THREADS ? THREADS / c : 1;      // rows at once
    const int g = threadIdx.x / (c < THREADS ? c : THREADS), x0 = threadIdx.x - g * c;
    if (g >= per) return;
    for (int j0 = first * per + g; j0 < n; j0 += U * step * per) {
        int2 m[U];
#pragma unroll
        for (int u = 0; u < U; ++u) m[u] = mv[min(j0 + u * step * per, n - 1)];
        for (int x = x0; x < c; x += THREADS) {
            v4u kk[U], vv[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                kk[u] = *reinterpret_cast<const v4u*>(k + m[u].y * a.kt + 16 * x);
                vv[u] = *reinterpret_cast<const v4u*>(v + m[u].y * a.vt + 16 * x);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j0 + u * step * per < n) {
                    *reinterpret_cast<v4u*>(k + m[u].x * a.kt + 16 * x) = kk[u];
                    *reinterpret_cast<v4u*>(v + m[u].x * a.vt + 16 * x) = vv[u];
                }
        }
    }
}

// KPT keys a thread in registers, slots in turn over the threads; a cache of more than KPT * 1024 slots in
// such chunks, its keys read again for each pass over them.
template <int KPT>
__global__ __launch_bounds__(EW, KPT <= 2 ? 8 : 4) void evict_select_kernel(EvictArgs a) {
    constexpr int WV = EW / 64;
    // four counts a digit, by lane: weights lie in few digits, and one address takes one lane at a time
    __shared__ __attribute__((aligned(16))) int hist[4 * BINS];
    __shared__ int2 few[HERE];               // few moves
    __shared__ int tmp[2][WV];
    __shared__ uint64_t stay_bits[KPT * WV], tie_bits[KPT * WV];
    __shared__ uint32_t digit;
    __shared__ int above, equal;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bh = blockIdx.x, b = bh / a.H;
    const int n = min(max(a.lens[b], 0), a.T), left = min(n, a.budget);
    const float* const w = a.w + (int64_t)bh * a.T;
    const int32_t* const pos = a.pos + (int64_t)bh * a.T;
    float* const wn = a.wn + (int64_t)bh * a.T;
    int32_t* const pn = a.pn + (int64_t)bh * a.T;
    const bool new_w = wn != w, new_p = pn != pos;   // not in place
    if (tid == 0 && bh % a.H == 0 && a.ln != a.lens) a.ln[b] = left;

    if (n <= a.budget || a.budget == 0) {    // every slot stays, or none
        for (int t = tid; t < (a.here ? a.T : left); t += EW) {
            wn[t] = t < left ? w[t] : 0.f;
            pn[t] = t < left ? pos[t] : -1;
        }
        if (tid == 0) a.count[bh] = 0;
        return;
    }
    for (int i = tid; i < BINS; i += EW) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
    const int chunks = (n + EW * KPT - 1) / (EW * KPT);
    uint32_t key[KPT];
    int32_t newest = INT32_MIN;              // the newest position
    int32_t ps[KPT];
    const uint32_t utid = tid;               // (uniform addresses and this offset: few registers)
    auto load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int t0 = (c * KPT + i) * EW;
            ps[i] = INT32_MIN;
            key[i] = 0;
            if (t0 + tid < n) {
                ps[i] = (pos + t0)[utid];
                key[i] = fbits((w + t0)[utid]);
            }
        }
    };
    for (int c = 0; c < chunks; ++c) {
        load(c);
#pragma unroll
        for (int i = 0; i < KPT; ++i) newest = max(newest, ps[i]);
    }
    const uint32_t top = wave_max_dpp((uint32_t)newest ^ 0x80000000u, 64);
    if (lane == 0) tmp[0][wave] = (int)top;
    __syncthreads();
    newest = (int32_t)(wave_max_dpp((uint32_t)tmp[0][lane & 15], 16) ^ 0x80000000u);
    // positions from `old` on stay (none of them where recent is 0)
    const int32_t old = (int32_t)max((int64_t)newest - a.recent + 1, (int64_t)INT32_MIN);
    // key 0: no slot (a weight's key is at least that of -inf).  fill: what new arrays hold but for the
    // holes, while it is at hand
    auto keys = [&](int c, bool fill) __attribute__((always_inline)) {
        if (chunks > 1) load(c);
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int t0 = (c * KPT + i) * EW, t = t0 + tid;
            const uint32_t k = a.recent > 0 && ps[i] >= old ? 0xFFFFFFFFu : weight_key(bitsf(key[i]));
            if (fill && t < left) {
                if (new_w) (wn + t0)[utid] = bitsf(key[i]);
                if (new_p) (pn + t0)[utid] = ps[i];
            }
            key[i] = t < n ? k : 0u;
        }
    };
    if (chunks == 1) keys(0, true);

    // the key of the left-th slot, and how many of the slots with that key stay
    uint32_t prefix = 0, mask = 0;
    int need = left, same = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
        const uint32_t dm = pass == 2 ? 0x3FFu : 0x7FFu;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) keys(c, pass == 0);
#pragma unroll
            for (int i = 0; i < KPT; ++i)      // (key 0 is below every slot's: never chosen)
                if ((key[i] & mask) == prefix) atomicAdd(&hist[4 * ((key[i] >> shift) & dm) + (lane & 3)], 1);
        }
        __syncthreads();
        // from the largest digit down: thread i sums digits 2047 - 2i and 2046 - 2i
        int4* const h4 = reinterpret_cast<int4*>(hist) + (BINS - 2 - 2 * tid);
        const int4 lo = h4[0], hi = h4[1];
        h4[0] = h4[1] = make_int4(0, 0, 0, 0);
        const int c0 = hi.x + hi.y + hi.z + hi.w, c1 = lo.x + lo.y + lo.z + lo.w;
        int total;
        const int before = block_scan(c0 + c1, tmp[1 - (pass & 1)], total);
        if (before < need && before + c0 + c1 >= need) {
            const bool first = before + c0 >= need;
            digit = (uint32_t)(first ? BINS - 1 - 2 * tid : BINS - 2 - 2 * tid);
            above = first ? before : before + c0;
            equal = first ? c0 : c1;
        }
        __syncthreads();
        prefix |= digit << shift;
        mask |= dm << shift;
        need -= above;
        same = equal;
        if (same == need) break;              // (uniform) all of this digit's slots stay: no ties
    }

    // In slot order: which of the equal keys stay, the holes and the sources.  A wave's slots at one place are
    // 64 in a row, so the ballots of a comparison, place after place and wave after wave, are its bits in slot
    // order, and a thread goes on with 32 of them.
    int2* const mv = a.here ? few : a.moves + (int64_t)bh * a.most;
    int ties = 0, holes = 0, extras = 0, total;
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) keys(c, false);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const uint64_t above_it = __ballot(key[i] > prefix || (same == need && key[i] >= prefix));
            if (lane == 0) stay_bits[i * WV + wave] = above_it;
        }
        if (same != need) {
#pragma unroll
            for (int i = 0; i < KPT; ++i) {
                const uint64_t tie = __ballot(key[i] == prefix);
                if (lane == 0) tie_bits[i * WV + wave] = tie;
            }
        }
        __syncthreads();
        const bool mine = tid < KPT * 32;
        uint32_t stay = mine ? reinterpret_cast<const uint32_t*>(stay_bits)[tid] : 0u;
        if (same != need) {
            uint32_t tie = mine ? reinterpret_cast<const uint32_t*>(tie_bits)[tid] : 0u;
            int room = need - ties - block_scan(__builtin_popcount(tie), tmp[0], total);
            ties += total;
            for (; tie && room > 0; --room, tie &= tie - 1) stay |= tie & -tie;
            __syncthreads();
        }
        const int t0 = (c * KPT * 32 + tid) * 32;            // this thread's first slot
        const uint32_t low = !mine || t0 >= left ? 0u : (left - t0 >= 32 ? ~0u : (1u << (left - t0)) - 1);
        uint32_t hole = low & ~stay, extra = mine ? stay & ~low : 0u;
        const uint32_t at = (uint32_t)block_scan(__builtin_popcount(hole) | __builtin_popcount(extra) << 16, tmp[1], total);
        for (int j = holes + (int)(at & 0xFFFF); hole; ++j, hole &= hole - 1) mv[j].x = t0 + __builtin_ctz(hole);
        for (int j = extras + (int)(at >> 16); extra; ++j, extra &= extra - 1) mv[j].y = t0 + __builtin_ctz(extra);
        holes += total & 0xFFFF;
        extras += (int)((uint32_t)total >> 16);
    }
    __syncthreads();
    for (int j = tid; j < holes; j += EW) {
        const int2 m = mv[j];
        wn[m.x] = w[m.y];
        pn[m.x] = pos[m.y];
    }
    if (a.here) move_rows<EW, 1>(a, a.k + b * a.kb + (bh - b * a.H) * a.kh, a.v + b * a.vb + (bh - b * a.H) * a.vh, mv, holes, 0, 1);
    if (a.here) {
        __syncthreads();                      // the sources are read, in place too
        for (int t = left + tid; t < a.T; t += EW) { wn[t] = 0.f; pn[t] = -1; }
    }
    if (tid == 0) a.count[bh] = holes;
}

// the lengths, when no workgroup reads the old ones any more
__device__ __forceinline__ void store_lens(const EvictArgs& a) {
    for (int b = threadIdx.x; b < a.B; b += 256) a.ln[b] = min(min(max(a.lens[b], 0), a.T), a.budget);
}
__global__ __launch_bounds__(256) void evict_lens_kernel(EvictArgs a) { store_lens(a); }

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H;
    if (bh == 0 && blockIdx.y == 0 && a.ln == a.lens) store_lens(a);
    // the slots past the new length (the same from the old length and the new one).  Here, where there is a second
    // launch: the selection need not wait for its one workgroup's stores (32 caches of 32768 slots cut to 4096 46 -> 44 us)
    const int left = min(min(max(a.lens[b], 0), a.T), a.budget);
    for (int64_t t = left + (int)(blockIdx.y * 256 + threadIdx.x); t < a.T; t += 256 * (int64_t)gridDim.y) {
        a.wn[(int64_t)bh * a.T + t] = 0.f;
        a.pn[(int64_t)bh * a.T + t] = -1;
    }
    move_rows<256, 4>(a, a.k + b * a.kb + h * a.kh, a.v + b * a.vb + h * a.vh, a.moves + (int64_t)bh * a.most, a.count[bh],
                   blockIdx.y, gridDim.y);
}

static void launch_select(const EvictArgs& a, hipStream_t s) {
    const unsigned grid = (unsigned)(a.B * a.H);
    const int per = (a.T + EW - 1) / EW;
    if (per <= 1) evict_select_kernel<1><<<grid, EW, 0, s>>>(a);
    else if (per <= 2) evict_select_kernel<2><<<grid, EW, 0, s>>>(a);
    else if (per <= 4) evict_select_kernel<4><<<grid, EW, 0, s>>>(a);
    else if (per <= 8) evict_select_kernel<8><<<grid, EW, 0, s>>>(a);
    else if (per <= 16) evict_select_kernel<16><<<grid, EW, 0, s>>>(a);
    else evict_select_kernel<32><<<grid, EW, 0, s>>>(a);
}

}  // namespace otpu

using namespace otpu;

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// the most slots that a (sequence, head) can move
static int most_moves(int T, int budget) { return T <= budget ? 0 : (T - budget < budget ? T - budget : budget); }

extern "C" int64_t otpu_kv_evict_work_bytes(int B, int T, int H, int budget) {
    if (B < 0 || T < 0 || H < 1 || budget < 0) {
        otpu_fail(OTPU_EINVAL, "kv_evict_work_bytes: B %d, T %d, H %d, budget %d", B, T, H, budget);
        return -1;
    }
    const int64_t n = (int64_t)B * H;
    return ((4 * n + 255) & ~(int64_t)255) + 8 * n * most_moves(T, budget) + 256;
}

extern "C" int otpu_kv_evict(const otpu_evict_args* args, otpu_stream_t stream) {
    if (!args || args->bytes != (int64_t)sizeof(otpu_evict_args))
        return otpu_fail(OTPU_EINVAL, "kv_evict: the arguments' size is not this header's %d", (int)sizeof(otpu_evict_args));
    const auto [bytes, k, kb, kt, kh, v, vb, vt, vh, weights, pos, lens, weights_out, pos_out, lens_out, work, work_bytes, B, T, H,
                row_bytes, budget, recent] = *args;
    if (B < 0 || T < 0 || T > (1 << 30) || H < 1 || budget < 0 || recent < 0 || (int64_t)B * H >= (1 << 22))
        return otpu_fail(OTPU_EINVAL, "kv_evict: B %d, T %d, H %d, budget %d, recent %d", B, T, H, budget, recent);
    if (row_bytes < 16 || row_bytes % 16 || row_bytes > (1 << 20))
        return otpu_fail(OTPU_EINVAL, "kv_evict: rows of %d bytes (a multiple of 16)", row_bytes);
    if (B == 0) return OTPU_OK;
    if (!lens || !lens_out || !work || (T && (!k || !v || !weights || !pos || !weights_out || !pos_out)))
        return otpu_fail(OTPU_EINVAL, "kv_evict: a NULL operand");
    const int64_t st[] = {kb, kt, kh, vb, vt, vh};
    for (int64_t x : st)
        if (x % 16) return otpu_fail(OTPU_EALIGN, "kv_evict: a stride of %lld bytes (multiples of 16)", (long long)x);
    if (!al16(k) || !al16(v) || ((uintptr_t)work & 255))
        return otpu_fail(OTPU_EALIGN, "kv_evict: k and v 16-byte aligned, work 256-byte");
    const int64_t need = otpu_kv_evict_work_bytes(B, T, H, budget);
    if (work_bytes < need)
        return otpu_fail(OTPU_EINVAL, "kv_evict: work area of %lld bytes, need %lld", (long long)work_bytes, (long long)need);
    EvictArgs a = {};
    a.k = (char*)k; a.kb = kb; a.kt = kt; a.kh = kh;
    a.v = (char*)v; a.vb = vb; a.vt = vt; a.vh = vh;
    a.row = row_bytes; a.w = weights; a.pos = pos; a.lens = lens;
    a.B = B; a.T = T; a.H = H; a.budget = budget; a.recent = recent;
    a.wn = weights_out; a.pn = pos_out; a.ln = lens_out;
    a.most = most_moves(T, budget);
    a.count = (int*)work;
    a.moves = (int2*)((char*)work + ((4 * (int64_t)B * H + 255) & ~(int64_t)255));
    const hipStream_t s = (hipStream_t)stream;
    a.here = a.most <= HERE;
    if (T) launch_select(a, s);
    if (T && !a.here) {
        const int c = row_bytes / 16, per = c < 256 ? 256 / c : 1;
        const int64_t pieces = (a.most + per - 1) / per;
        const int64_t want = (8 * (int64_t)otpu_cu_count() + B * H - 1) / ((int64_t)B * H);
        evict_move_kernel<<<dim3((unsigned)(B * H), (unsigned)(pieces < want ? pieces : want)), 256, 0, s>>>(a);
    } else if (lens_out == lens || !T) {
        evict_lens_kernel<<<1, 256, 0, s>>>(a);
    }
    return otpu_launch_check("kv_evict");
}
