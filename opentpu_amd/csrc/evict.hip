// Eviction from a key/value cache by accumulated attention weight.  Of a (sequence, head)'s n slots the
// `budget` slots stay that come first by (recent, weight, slot): the newest positions always, then the
// largest weights, the lower slot where weights are equal.  The j-th slot below the budget that goes takes
// over the j-th slot at or past it that stays: attention does not ask for an order of slots, so only the
// holes are filled, sources and destinations are disjoint and every move is independent.
//
//   evict_select_kernel   a workgroup a (sequence, head): the threshold by radix selection (11, 11 and 10
//                         bits), the holes and their sources, the slots' weights and positions
//   evict_move_kernel     the rows of k and v, 16 bytes a lane
#include "otpu_common.h"

namespace otpu {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int EW = 1024;                     // threads of a selecting workgroup
constexpr int BINS = 2048;

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
};

// weights in the order of the selection: NaN above infinity, -0 with +0
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xFFC00000u;
    const uint32_t u = fbits(w + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// exclusive sum of v over the workgroup's threads, in thread order; total: the whole sum
__device__ __forceinline__ int block_scan(int v, int* tmp, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < EW / 64; ++i) {
        const int t = tmp[i];
        before += i < wave ? t : 0;
        all += t;
    }
    __syncthreads();
    total = all;
    return before + x - v;
}

__global__ __launch_bounds__(EW) void evict_select_kernel(EvictArgs a) {
    __shared__ int hist[BINS];
    __shared__ int tmp[EW / 64];
    __shared__ uint32_t digit;
    __shared__ int above;
    const int tid = threadIdx.x;
    const int bh = blockIdx.x, b = bh / a.H;
    const int n = min(max(a.lens[b], 0), a.T), left = min(n, a.budget);
    const float* const w = a.w + (int64_t)bh * a.T;
    const int32_t* const pos = a.pos + (int64_t)bh * a.T;
    float* const wn = a.wn + (int64_t)bh * a.T;
    int32_t* const pn = a.pn + (int64_t)bh * a.T;

    if (n <= a.budget || a.budget == 0) {    // every slot stays, or none
        for (int t = tid; t < a.T; t += EW) {
            wn[t] = t < left ? w[t] : 0.f;
            pn[t] = t < left ? pos[t] : -1;
        }
        if (tid == 0) a.count[bh] = 0;
        return;
    }
    // the newest position
    int64_t newest = INT32_MIN;
    for (int t = tid; t < n; t += EW) newest = max(newest, (int64_t)pos[t]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) newest = max(newest, (int64_t)__shfl_xor((int)newest, o, 64));
    if ((tid & 63) == 0) tmp[tid >> 6] = (int)newest;
    __syncthreads();
    for (int i = 0; i < EW / 64; ++i) newest = max(newest, (int64_t)tmp[i]);
    __syncthreads();
    const int64_t old = newest - a.recent;   // positions past it stay
    auto key = [&](int t) __attribute__((always_inline)) {
        return (int64_t)pos[t] > old ? 0xFFFFFFFFu : weight_key(w[t]);
    };

    // the key of the left-th slot, and how many of the slots with that key stay
    uint32_t prefix = 0, mask = 0;
    int need = left;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < BINS; i += EW) hist[i] = 0;
        __syncthreads();
        for (int t = tid; t < n; t += EW) {
            const uint32_t x = key(t);
            if ((x & mask) == prefix) atomicAdd(&hist[(x >> shift) & ((1u << bits) - 1)], 1);
        }
        __syncthreads();
        // from the largest digit down: thread i sums digits 2047 - 2i and 2046 - 2i
        const int c0 = hist[BINS - 1 - 2 * tid], c1 = hist[BINS - 2 - 2 * tid];
        int total;
        const int before = block_scan(c0 + c1, tmp, total);
        if (before < need && before + c0 + c1 >= need) {
            const bool first = before + c0 >= need;
            digit = (uint32_t)(first ? BINS - 1 - 2 * tid : BINS - 2 - 2 * tid);
            above = first ? before : before + c0;
        }
        __syncthreads();
        prefix |= digit << shift;
        mask |= ((1u << bits) - 1) << shift;
        need -= above;
        __syncthreads();
    }

    // in slot order: which of the equal keys stay, the holes and the sources
    int2* const mv = a.moves + (int64_t)bh * a.most;
    int ties = 0, holes = 0, extras = 0;
    for (int t0 = 0; t0 < n; t0 += EW) {
        const int t = t0 + tid;
        const uint32_t x = t < n ? key(t) : 0u;
        const bool tie = t < n && x == prefix;
        int total;
        const int before = block_scan(tie ? 1 : 0, tmp, total);
        const bool stays = t < n && (x > prefix || (tie && ties + before < need));
        ties += total;
        const bool hole = t < left && !stays, extra = t >= left && stays;
        int tot;
        const int at = block_scan((hole ? 1 : 0) | (extra ? 1 << 16 : 0), tmp, tot);
        if (hole) mv[holes + (at & 0xFFFF)].x = t;
        if (extra) mv[extras + (at >> 16)].y = t;
        holes += tot & 0xFFFF;
        extras += tot >> 16;
        if (t < left && stays && wn != w) { wn[t] = w[t]; pn[t] = pos[t]; }
    }
    __threadfence_block();
    __syncthreads();
    for (int j = tid; j < holes; j += EW) {
        const int2 m = mv[j];
        wn[m.x] = w[m.y];
        pn[m.x] = pos[m.y];
    }
    __syncthreads();
    for (int t = left + tid; t < a.T; t += EW) { wn[t] = 0.f; pn[t] = -1; }
    if (tid == 0) a.count[bh] = holes;
}

__global__ __launch_bounds__(256) void evict_lens_kernel(const int32_t* lens, int32_t* ln, int B, int T, int budget) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < B) ln[b] = min(min(max(lens[b], 0), T), budget);
}

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H;
    const int n = a.count[bh], c = a.row / 16;
    const int2* const mv = a.moves + (int64_t)bh * a.most;
    char* const k = a.k + b * a.kb + h * a.kh;
    char* const v = a.v + b * a.vb + h * a.vh;
    for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < (int64_t)n * c; i += (int64_t)gridDim.y * 256) {
        const int j = (int)(i / c), x = (int)(i - (int64_t)j * c) * 16;
        const int2 m = mv[j];
        const v4u kk = *reinterpret_cast<const v4u*>(k + m.y * a.kt + x);
        const v4u vv = *reinterpret_cast<const v4u*>(v + m.y * a.vt + x);
        *reinterpret_cast<v4u*>(k + m.x * a.kt + x) = kk;
        *reinterpret_cast<v4u*>(v + m.x * a.vt + x) = vv;
    }
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

extern "C" int otpu_kv_evict(void* k, int64_t kb, int64_t kt, int64_t kh, void* v, int64_t vb, int64_t vt, int64_t vh,
                             int row_bytes, const float* weights, const int32_t* pos, const int32_t* lens, int B, int T,
                             int H, int budget, int recent, float* weights_out, int32_t* pos_out, int32_t* lens_out,
                             void* work, int64_t work_bytes, otpu_stream_t stream) {
    if (B < 0 || T < 0 || H < 1 || budget < 0 || recent < 0 || (int64_t)B * H > (1 << 24))
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
    if (T) evict_select_kernel<<<(unsigned)(B * H), EW, 0, s>>>(a);
    if (a.most) {
        const int64_t pieces = ((int64_t)a.most * (row_bytes / 16) + 255) / 256;
        const int64_t want = (8 * (int64_t)otpu_cu_count() + B * H - 1) / ((int64_t)B * H);
        evict_move_kernel<<<dim3((unsigned)(B * H), (unsigned)(pieces < want ? pieces : want)), 256, 0, s>>>(a);
    }
    evict_lens_kernel<<<(B + 255) / 256, 256, 0, s>>>(lens, lens_out, B, T, budget);
    return otpu_launch_check("kv_evict");
}
