// Attention over sequences with capped scores, a bias of distance and masks
// by document, causal and prefix (bl_masked_attention), for head_dim 64.
//
// A row's mask is an interval of its own sequence in every form: row i sees
// the keys [0, visible(i)) of it, visible(i) = length, i + 1, or
// max(i + 1, prefix). So no mask is stored or read: a tile of keys needs one
// comparison against the row's bound, and tiles past every row's bound are
// never loaded.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "host.h"

namespace bl {
namespace masked {

constexpr int HD = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
    int batch, tokens;
    int heads, kv_heads, group;  // group = heads / kv_heads
    int last_rows;
    float scale, cap;
    int mask;
    const uint16_t* qkv;
    long long row;      // elements between rows of qkv
    void* out;
    long long out_row;
    int out_dtype;
    const int* offsets;
    const int* lengths;
    const int* prefix;
    const float* slopes;
    const float* pos;
    long long pos_row;
    int pos_axes;
    int splits;         // CTAs of a cluster that share the keys
    int chunks;         // query chunks (or tiles) a sequence has at most
    Status* status;
};

// A sequence's rows, whatever the offsets and lengths hold: clamped to the
// buffer, so no index below can leave it.
struct Span {
    long long begin;  // first row
    int len;          // rows
    int prefix;       // keys every row sees (BL_MASK_PREFIX)
    int first;        // first query row
};
__device__ __forceinline__ Span span_of(const Params& p, int s) {
    Span q;
    if (p.offsets != nullptr) {
        const int b = min(max(p.offsets[s], 0), p.tokens);
        q.begin = b;
        q.len = min(max(p.offsets[s + 1], b), p.tokens) - b;
    } else {
        q.begin = static_cast<long long>(s) * p.tokens;
        q.len = p.lengths != nullptr ? min(max(p.lengths[s], 0), p.tokens) : p.tokens;
    }
    q.prefix = p.mask == BL_MASK_PREFIX ? min(max(p.prefix[s], 0), q.len) : 0;
    q.first = p.last_rows > 0 ? max(q.len - p.last_rows, 0) : 0;
    return q;
}
// How many of its sequence's keys row i sees.
__device__ __forceinline__ int visible(const Params& p, const Span& q, int i) {
    return p.mask == BL_MASK_NONE ? q.len : max(i + 1, q.prefix);
}

__device__ __forceinline__ float2 unpack2(uint32_t w, bool bf16) {
    if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ void unpack8(const uint4& v, bool bf16, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = unpack2(w[i], bf16);
        f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
}

// cap tanh(s / cap) as cap - 2 cap / (1 + e^(2 s / cap)): an absolute error of
// a few 2^-23 cap, which is what an exponent needs.
__device__ __forceinline__ float capped(float s, float cap, float two_log2e_over_cap) {
    return cap - __fdividef(2.0f * cap, 1.0f + ex2(s * two_log2e_over_cap));
}

// ------------------------------------------------------------------ few rows
//
// One CTA computes R query rows of one K/V head (rows and heads of its group
// alike) over one split of the keys. Eight lanes hold one key's 64 values, 8
// each, so a warp reads four keys with one 16-byte load a lane and a score is
// eight products a lane and three shuffles. Every group of eight lanes keeps
// its own running maximum, sum and output over the keys it has seen; they are
// merged once at the end: lanes, warps, then the cluster's CTAs.
constexpr int kWarps = 8;
constexpr int kUnroll = 4;  // key quads a warp has in flight

template <int R>
__global__ void __launch_bounds__(32 * kWarps) rows_kernel(const Params p, int bf16) {
    pdl_trigger();
    pdl_wait();
    __shared__ float part_o[kWarps][R][HD];
    __shared__ float2 part_ml[kWarps][R];
    __shared__ float cta_o[R][HD];
    __shared__ float2 cta_ml[R];
    const int warp = warp_id(), lane = lane_id();
    const int split = blockIdx.x % p.splits;
    const int unit = blockIdx.x / p.splits;
    const int chunk = unit % p.chunks;
    const Span q = span_of(p, unit / p.chunks);
    const int nrows = q.len - q.first;
    const int kvh = blockIdx.y;
    const int c0 = chunk * R;
    if (c0 >= nrows * p.group) return;  // the whole cluster leaves

    const int g = lane >> 3, d = (lane & 7) * 8;
    float qv[R][8], acc[R][8], m[R], l[R], slope[R], qp[R][3];
    int row[R], seen[R], most = 0;
    for (int r = 0; r < R; ++r) {
        const int c = min(c0 + r, nrows * p.group - 1);
        const int head = kvh * p.group + c % p.group;
        row[r] = q.first + c / p.group;
        seen[r] = visible(p, q, row[r]);
        most = max(most, seen[r]);
        const uint4 v = *reinterpret_cast<const uint4*>(p.qkv + (q.begin + row[r]) * p.row +
                                                        head * HD + d);
        unpack8(v, bf16 != 0, qv[r]);
        for (int i = 0; i < 8; ++i) qv[r][i] *= p.scale, acc[r][i] = 0.0f;
        m[r] = -INFINITY, l[r] = 0.0f;
        slope[r] = p.slopes != nullptr ? p.slopes[head] : 0.0f;
        for (int a = 0; a < 3; ++a)
            qp[r][a] = p.pos != nullptr && a < p.pos_axes
                           ? p.pos[(q.begin + row[r]) * p.pos_row + a] : 0.0f;
    }
    const float cap_in = p.cap > 0.0f ? 2.0f * kLog2e / p.cap : 0.0f;
    const int per = ((most + p.splits - 1) / p.splits + 15) / 16 * 16;
    const int k0 = min(split * per, most), k1 = min(k0 + per, most);
    const uint16_t* kbase = p.qkv + q.begin * p.row + (p.heads + kvh) * HD + d;
    const uint16_t* vbase = kbase + p.kv_heads * HD;

    for (int base = k0 + 4 * kUnroll * warp; base < k1; base += 4 * kUnroll * kWarps) {
        uint4 kr[kUnroll], vr[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int key = base + 4 * u + g;
            kr[u] = vr[u] = make_uint4(0, 0, 0, 0);
            if (key < k1) {
                kr[u] = *reinterpret_cast<const uint4*>(kbase + key * p.row);
                vr[u] = *reinterpret_cast<const uint4*>(vbase + key * p.row);
            }
        }
        float s[R][kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float kf[8];
            unpack8(kr[u], bf16 != 0, kf);
            const int key = base + 4 * u + g;
            float kp[3] = {0.0f, 0.0f, 0.0f};
            if (p.pos != nullptr && key < k1)
                for (int a = 0; a < p.pos_axes; ++a) kp[a] = p.pos[(q.begin + key) * p.pos_row + a];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float t = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) t = fmaf(qv[r][i], kf[i], t);
                t += __shfl_xor_sync(0xFFFFFFFFu, t, 1);
                t += __shfl_xor_sync(0xFFFFFFFFu, t, 2);
                t += __shfl_xor_sync(0xFFFFFFFFu, t, 4);
                if (p.cap > 0.0f) t = capped(t, p.cap, cap_in);
                if (p.slopes != nullptr) {
                    float far;
                    if (p.pos != nullptr) {
                        const float x = qp[r][0] - kp[0], y = qp[r][1] - kp[1], z = qp[r][2] - kp[2];
                        far = sqrtf(fmaf(x, x, fmaf(y, y, z * z)));
                    } else {
                        far = fabsf(static_cast<float>(row[r] - key));
                    }
                    t = fmaf(-slope[r], far, t);
                }
                s[r][u] = key < min(k1, seen[r]) ? t * kLog2e : -INFINITY;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = m[r];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) top = fmaxf(top, s[r][u]);
            const float ref = top == -INFINITY ? 0.0f : top;
            const float shrink = ex2(m[r] - ref);
            m[r] = top;
            l[r] *= shrink;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[r][i] *= shrink;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) s[r][u] = ex2(s[r][u] - ref), l[r] += s[r][u];
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float vf[8];
            unpack8(vr[u], false, vf);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[r][i] = fmaf(s[r][u], vf[i], acc[r][i]);
        }
    }

    // lanes of one key group -> warp
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float top = fmaxf(fmaxf(m[r], __shfl_xor_sync(0xFFFFFFFFu, m[r], 8)),
                                __shfl_xor_sync(0xFFFFFFFFu, fmaxf(m[r], __shfl_xor_sync(
                                    0xFFFFFFFFu, m[r], 8)), 16));
        const float w = ex2(m[r] - (top == -INFINITY ? 0.0f : top));
        l[r] *= w;
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 8);
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            acc[r][i] *= w;
            acc[r][i] += __shfl_xor_sync(0xFFFFFFFFu, acc[r][i], 8);
            acc[r][i] += __shfl_xor_sync(0xFFFFFFFFu, acc[r][i], 16);
        }
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) part_o[warp][r][d + i] = acc[r][i];
            if (lane == 0) part_ml[warp][r] = make_float2(top, l[r]);
        }
    }
    __syncthreads();
    // warps -> CTA
    for (int t = threadIdx.x; t < R * HD; t += 32 * kWarps) {
        const int r = t / HD, e = t % HD;
        float top = -INFINITY, o = 0.0f, sum = 0.0f;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_ml[w][r].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(part_ml[w][r].x - ref);
            o = fmaf(f, part_o[w][r][e], o);
            sum = fmaf(f, part_ml[w][r].y, sum);
        }
        cta_o[r][e] = o;
        if (e == 0) cta_ml[r] = make_float2(top, sum);
    }
    __syncthreads();
    if (p.splits > 1) {
        fence_cluster();
        cluster_sync();
    }
    // CTAs -> row, by the cluster's first CTA
    if (split == 0) {
        for (int t = threadIdx.x; t < R * HD; t += 32 * kWarps) {
            const int r = t / HD, e = t % HD;
            const int c = c0 + r;
            if (c >= nrows * p.group) continue;
            float top = -INFINITY, o = 0.0f, sum = 0.0f;
            for (int k = 0; k < p.splits; ++k)
                top = fmaxf(top, dsmem_ld2(dsmem_addr(smem_u32(&cta_ml[r]), k)).x);
            const float ref = top == -INFINITY ? 0.0f : top;
            for (int k = 0; k < p.splits; ++k) {
                const float2 ml = dsmem_ld2(dsmem_addr(smem_u32(&cta_ml[r]), k));
                const float f = ex2(ml.x - ref);
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v)
                             : "r"(dsmem_addr(smem_u32(&cta_o[r][e]), k)));
                o = fmaf(f, v, o);
                sum = fmaf(f, ml.y, sum);
            }
            o = sum == 0.0f ? 0.0f : o / sum;
            const long long at = (q.begin + q.first + c / p.group) * p.out_row +
                                 (kvh * p.group + c % p.group) * HD + e;
            if (p.out_dtype == BL_F32) static_cast<float*>(p.out)[at] = o;
            else if (p.out_dtype == BL_F16) static_cast<__half*>(p.out)[at] = __float2half_rn(o);
            else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(o);
        }
    }
    if (p.splits > 1) {
        __syncwarp();
        cluster_sync();  // no CTA leaves while its partials are read
    }
}

// ------------------------------------------------------------------ tiles
//
// One CTA computes 128 query rows of one head over a range of 64-key tiles on
// the tensor cores; two CTAs share an SM, with half the TMEM each. The
// exponentials bound it (one a score at 16 a clock and SM, against a quarter
// of that time for its products), so the rest is there to keep that unit fed.
// Every query row has two softmax threads, one for the even key tiles and one
// for the odd, so four softmax warps a scheduler cover one another's waits;
// S has three TMEM buffers, so the scores of the next tile are there before a
// thread asks for them. Both add to one O, whose reference exponent R (the
// lagging running maximum) they hand to each other: R(i) follows from R(i - 1)
// and the maximum of tile i, known long before tile i's exponentials are done.
// Warps:
//   0      finds the CTA's sequence among the packed ones, then the TMA
//          producer: the Q tile once, then K and V tiles into a ring.
//   1      MMA issuer: S = Q K^T (M 128, N 64, K 64) into TMEM, O += P V (P
//          from TMEM, f16, over the S it came from); S(i + 3) follows PV(i),
//          whose buffer it takes.
//   2..5   softmax of the even key tiles, one thread a query row (TMEM lane),
//   6..9   of the odd ones.
// A thread reads its 64 scores from TMEM twice, 32 at a time, for the maximum
// and for the exponentials (a 32-column load takes 17 clocks of a warp
// scheduler's TMEM port, 32 exponentials 256), which leaves it within the 96
// registers that ten warps and two CTAs allow.
// Tiles start at their sequence's first row, so a key tile holds keys of one
// sequence, and past its end only rows that no query sees: their scores are
// replaced by -inf and their V rows zeroed in shared memory before the
// product, since 0 * NaN from another sequence's rows would reach O.
constexpr int BM = 128;
constexpr int BN = 64;
constexpr int STAGES = 5;  // K/V ring
constexpr int SBUFS = 3;
constexpr int kTileThreads = 320;  // two CTAs of 96 registers a thread
constexpr int kSoftmaxWarp0 = 2;
constexpr uint32_t kQBytes = BM * HD * 2;
constexpr uint32_t kKvBytes = BN * HD * 2;
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kColO = SBUFS * BN;
static_assert(kColO + HD <= kTmemCols, "TMEM columns");
// The running maximum may trail the true one by this much (log2 units) before
// O is rescaled: P stays below 2^8, well inside f16.
constexpr float kRescaleThreshold = 8.0f;

struct TileTail {
    uint64_t q_full;
    uint64_t kv_full[STAGES];
    uint64_t kv_empty[STAGES];
    // by S buffer (tile i: i % SBUFS). S(i) complete means that S(i - 1) and
    // PV(i - 3) are, so each parity names one phase wherever it is waited for.
    uint64_t s_full[SBUFS];
    uint64_t p_full[SBUFS];
    uint64_t o_done[SBUFS];  // PV(i) is complete
    uint64_t ref_full[2][4]; // R of the stream's tile is written, by TMEM quarter
    uint64_t o_final;
    uint64_t odd_done;       // the odd stream's sums are written
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
    // this CTA's work, found once by warp 0
    Span span;
    int q0, rows;   // first query row within the sequence, rows of the tile (0: no work)
    int t0, n;      // its key tiles
    float ref[2][BM];      // R after the stream's last tile
    float odd_sum[BM];
    float kpos[8][3][BN];  // each softmax warp's copy of a key tile's positions
};
constexpr size_t kTileSmem = 1024 + kQBytes + 2 * STAGES * kKvBytes + sizeof(TileTail);
static_assert(2 * (kTileSmem + 1024) <= 233472, "two CTAs an SM");

// The sequence (its rows, without the prefix) and tile of tile `index` of the
// packed batch: a warp walks the offsets 256 sequences at a time, eight a lane,
// so a chunk costs one round trip to memory. Returns the sequence, -1 behind
// the last tile.
__device__ __forceinline__ int find_tile(const Params& p, int index, int& begin, int& len,
                                         int& tile) {
    const int lane = lane_id();
    int total = 0;
    for (int base = 0; base < p.batch; base += 256) {
        const int first = base + 8 * lane;
        int at[9];
#pragma unroll
        for (int i = 0; i < 9; ++i) at[i] = p.offsets[min(first + i, p.batch)];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 9; ++i) at[i] = min(max(at[i], 0), p.tokens);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + i < p.batch) mine += (max(at[i + 1] - at[i], 0) + BM - 1) / BM;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= o) upto += u;
        }
        const unsigned past = __ballot_sync(0xFFFFFFFFu, total + upto > index);
        if (past != 0) {
            const int owner = __ffs(past) - 1;
            int left = index - total - (upto - mine), s = 0, b = 0, n = 0;
            bool found = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int rows = first + i < p.batch ? max(at[i + 1] - at[i], 0) : 0;
                const int count = (rows + BM - 1) / BM;
                if (!found && left < count) found = true, s = first + i, b = at[i], n = rows;
                if (!found) left -= count;
            }
            begin = __shfl_sync(0xFFFFFFFFu, b, owner);
            len = __shfl_sync(0xFFFFFFFFu, n, owner);
            tile = __shfl_sync(0xFFFFFFFFu, left, owner);
            return __shfl_sync(0xFFFFFFFFu, found ? s : -1, owner);
        }
        total += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return -1;
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float sqrt_approx(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void store4(void* out, long long at, int dt, const float4& v) {
    if (dt == BL_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = v;
    } else {
        const uint2 w = dt == BL_F16 ? make_uint2(pack_f16x2(v.x, v.y), pack_f16x2(v.z, v.w))
                                     : make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = w;
    }
}
__device__ __forceinline__ void store8(void* out, long long at, int dt, const float* v) {
    if (dt == BL_F32) {
        store4(out, at, dt, make_float4(v[0], v[1], v[2], v[3]));
        store4(out, at + 4, dt, make_float4(v[4], v[5], v[6], v[7]));
    } else {
        const uint4 w = dt == BL_F16
            ? make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]),
                         pack_f16x2(v[6], v[7]))
            : make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                         pack_bf16x2(v[6], v[7]));
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = w;
    }
}

enum { BIAS_NONE = 0, BIAS_INDEX = 1, BIAS_PLANE = 2, BIAS_SPACE = 3 };

template <bool kCap, int kBias>
__global__ void __launch_bounds__(kTileThreads, 2)
    tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv,
                const __grid_constant__ Params p, int bf16) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* sQ = smem;
    uint8_t* sK = smem + kQBytes;  // stage s at + s * kKvBytes
    uint8_t* sV = sK + STAGES * kKvBytes;
    TileTail* tail = reinterpret_cast<TileTail*>(sV + STAGES * kKvBytes);
    volatile int* abort = &tail->abort;
    const int warp = warp_id(), lane = lane_id();
    const int head = blockIdx.y, kvh = head / p.group;
    constexpr unsigned kFull = 0xFFFFFFFFu;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&tail->q_full), 1);
        for (int t = 0; t < STAGES; ++t) {
            mbar_init(smem_u32(&tail->kv_full[t]), 1);
            mbar_init(smem_u32(&tail->kv_empty[t]), 1);
        }
        for (int t = 0; t < SBUFS; ++t) {
            mbar_init(smem_u32(&tail->s_full[t]), 1);
            mbar_init(smem_u32(&tail->p_full[t]), 4);  // one arrival a warp
            mbar_init(smem_u32(&tail->o_done[t]), 1);
        }
        for (int t = 0; t < 8; ++t) mbar_init(smem_u32(&tail->ref_full[t >> 2][t & 3]), 1);
        mbar_init(smem_u32(&tail->o_final), 1);
        mbar_init(smem_u32(&tail->odd_done), 4);
        mbar_init(smem_u32(&tail->drain), 1);
        tail->abort = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_kv);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tail->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    pdl_trigger();
    pdl_wait();
    if (warp == 0) {
        __syncwarp();
        const int unit = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.splits));
        const unsigned split = blockIdx.x - static_cast<unsigned>(unit) * p.splits;
        Span q{};
        int tile = 0, rows = 0, q0 = 0, first = 0, count = 0;
        if (p.chunks > 0) {
            q = span_of(p, unit / p.chunks);
            tile = unit % p.chunks;
        } else {
            int begin = 0;
            const int seq = find_tile(p, unit, begin, q.len, tile);
            q.begin = begin;
            if (seq < 0) q.len = 0;
            else if (p.mask == BL_MASK_PREFIX) q.prefix = min(max(p.prefix[seq], 0), q.len);
        }
        const int tiles = (q.len - q.first + BM - 1) / BM;
        if (tile >= 0 && tile < tiles) {
            // with a causal mask the last rows see most: they start first
            if (p.mask != BL_MASK_NONE) tile = tiles - 1 - tile;
            q0 = q.first + tile * BM;
            rows = min(q.len - q0, BM);
            // below 2^25 tiles and at most 8 splits: 32 bits hold the products
            const unsigned nt = (visible(p, q, q0 + rows - 1) + BN - 1) / BN;
            first = static_cast<int>(nt * split / p.splits);
            count = static_cast<int>(nt * (split + 1) / p.splits) - first;
        }
        if (lane == 0) {
            tail->span = q;
            tail->q0 = q0, tail->rows = rows, tail->t0 = first, tail->n = count;
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tail->tmem_base;
    if (tail->rows == 0) {  // no such tile (the same for every CTA of a cluster)
        if (warp == 1) tmem_dealloc(tmem, kTmemCols);
        return;
    }
    const int t0 = tail->t0, n = tail->n;

    // One lane waits and the vote hands its outcome to the warp, unless the
    // barrier is past that phase already.
    const bool elected = elect_one();
    auto wait_warp = [&](uint64_t* bar, int parity, uint32_t code, uint32_t where) -> bool {
        if (__all_sync(kFull, mbar_try_wait(smem_u32(bar), parity))) return true;
        bool r = true;
        if (elected) r = mbar_wait(smem_u32(bar), parity, abort, p.status, code, where);
        return __all_sync(kFull, r);
    };
    if (warp == 0) {
        // ------------------------------------------------------ producer
        const int row0 = static_cast<int>(tail->span.begin);
        if (elected && n > 0) {
            mbar_arrive_expect_tx(smem_u32(&tail->q_full), kQBytes);
            tma_load_2d(smem_u32(sQ), &tm_q, head * HD, row0 + tail->q0, smem_u32(&tail->q_full));
        }
        int loaded = 0;
        for (int s = 0, phase = 1; loaded < n; ++loaded) {
            if (loaded >= STAGES && !wait_warp(&tail->kv_empty[s], phase, ST_TIMEOUT_TMA, loaded))
                break;
            if (elected) {
                const uint32_t bar = smem_u32(&tail->kv_full[s]);
                const int y = row0 + (t0 + loaded) * BN;
                mbar_arrive_expect_tx(bar, 2 * kKvBytes);
                tma_load_2d(smem_u32(sK + s * kKvBytes), &tm_kv, (p.heads + kvh) * HD, y, bar);
                tma_load_2d(smem_u32(sV + s * kKvBytes), &tm_kv, (p.heads + p.kv_heads + kvh) * HD,
                            y, bar);
            }
            __syncwarp();
            if (++s == STAGES) s = 0, phase ^= 1;
        }
        if (elected && n > 0 && *abort) {
            // unwinding: every copy in flight lands before the CTA ends
            mbar_wait(smem_u32(&tail->q_full), 0, nullptr, p.status, ST_TIMEOUT_DRAIN, 0);
            for (int s = 0; s < STAGES && s < loaded; ++s)
                mbar_wait(smem_u32(&tail->kv_full[s]), ((loaded - s - 1) / STAGES) & 1, nullptr,
                          p.status, ST_TIMEOUT_DRAIN, s);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------ MMA issuer
        const uint32_t idesc_s = idesc_f16(BM, BN, bf16, bf16, 0, 0);
        const uint32_t idesc_o = idesc_f16(BM, HD, 0, 0, 0, 1);
        const uint64_t dq = sdesc_sw128(smem_u32(sQ), 16, 1024);
        const uint64_t dk = sdesc_sw128(smem_u32(sK), 16, 1024);
        // V rows are keys with the 64 columns contiguous: the MN-major B
        // operand, one swizzle atom wide, groups of 8 keys 1024 bytes apart
        const uint64_t dv = sdesc_sw128(smem_u32(sV), kKvBytes, 1024);
        constexpr uint64_t kStep = kKvBytes >> 4;
        const int end = tail->span.len;
        // ring places, stepped as the loop goes: S runs SBUFS tiles ahead of PV
        int sb = 0, st = 0, st_phase = 0;  // of the next S: TMEM buffer, stage
        int pb = 0, p_phase = 0, pt = 0;   // of the next PV
        auto wait_tile = [&](int i) -> bool {
            if (!wait_warp(&tail->kv_full[st], st_phase, ST_TIMEOUT_MMA, i)) return false;
            const int valid = end - (t0 + i) * BN;
            if (valid < BN) {
                // the sequence ends inside this tile: its V rows past the
                // end belong to no key (a whole 128-byte row each, so the
                // swizzle does not matter)
                uint8_t* v = sV + st * kKvBytes;
                for (int r = valid + (lane >> 3); r < BN; r += 4)
                    *reinterpret_cast<uint4*>(v + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
            }
            return true;
        };
        auto issue_s = [&]() {
            const uint64_t b = dk + st * kStep;
            const uint32_t dst = tmem + BN * sb;
            if (elected) {
                mma_ss(dst, dq, b, idesc_s, 0u);
#pragma unroll
                for (int k = 1; k < HD / 16; ++k) mma_ss(dst, dq + 2 * k, b + 2 * k, idesc_s, 1u);
                mma_commit(smem_u32(&tail->s_full[sb]));
            }
            __syncwarp();
            if (++sb == SBUFS) sb = 0;
            if (++st == STAGES) st = 0, st_phase ^= 1;
        };
        auto issue_pv = [&](int i) {
            const uint64_t b = dv + pt * kStep;
            const uint32_t a = tmem + BN * pb, o = tmem + kColO;
            if (elected) {
                mma_ts(o, a, b, idesc_o, i > 0 ? 1u : 0u);
#pragma unroll
                for (int k = 1; k < BN / 16; ++k) mma_ts(o, a + k * 8, b + 128 * k, idesc_o, 1u);
                mma_commit(smem_u32(&tail->o_done[pb]));
                if (i + STAGES < n) mma_commit(smem_u32(&tail->kv_empty[pt]));
                if (i == n - 1) mma_commit(smem_u32(&tail->o_final));
            }
            __syncwarp();
            if (++pb == SBUFS) pb = 0, p_phase ^= 1;
            if (++pt == STAGES) pt = 0;
        };
        bool ok = n == 0 || wait_warp(&tail->q_full, 0, ST_TIMEOUT_MMA, 0xFFFF);
        for (int i = 0; i < SBUFS && i < n && ok; ++i) {
            ok = wait_tile(i);
            tc_fence_after();
            if (ok) issue_s();
        }
        for (int i = 0; i < n && ok; ++i) {
            // what S(i + 3) needs first: between P(i) and it stand only MMAs
            const bool more = i + SBUFS < n;
            if (more) ok = wait_tile(i + SBUFS);
            ok = ok && wait_warp(&tail->p_full[pb], p_phase, ST_TIMEOUT_MMA, 0x10000 | i);
            if (!ok) break;
            tc_fence_after();
            issue_pv(i);
            if (more) issue_s();
        }
        if (!ok) {
            // unwinding: what was issued completes before TMEM is released
            if (elected) {
                mma_commit(smem_u32(&tail->drain));
                mbar_wait(smem_u32(&tail->drain), 0, nullptr, p.status, ST_TIMEOUT_DRAIN, 0xD);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------ softmax
        const int sub = warp & 3;
        const int odd = (warp - kSoftmaxWarp0) >> 2;  // the stream
        const int row = sub * 32 + lane;
        const uint32_t t_lane = tmem + (static_cast<uint32_t>(sub * 32) << 16);
        const uint32_t o_col = t_lane + kColO;
        const Span q = tail->span;
        const int at = tail->q0 + row;  // this row within the sequence
        const bool live = row < tail->rows;
        const int seen = live ? visible(p, q, at) : 0;
        constexpr bool kPlain = !kCap && kBias == BIAS_NONE;
        // kPlain keeps raw scores and scales them in the exponent's FMA; the
        // other forms turn each score into log2 units first
        const float c = kPlain ? p.scale * kLog2e : 1.0f;
        const float in = kCap ? 2.0f * p.scale / p.cap * kLog2e : p.scale * kLog2e;
        const float cap2 = p.cap * kLog2e;
        const float slope2 = kBias != BIAS_NONE ? p.slopes[head] * kLog2e : 0.0f;
        float qp[3] = {0.0f, 0.0f, 0.0f};
        if (kBias >= BIAS_PLANE) {
#pragma unroll
            for (int a = 0; a < 3; ++a)
                if (live && a < p.pos_axes) qp[a] = p.pos[(q.begin + at) * p.pos_row + a];
        }
        const float(*kpos)[BN] = tail->kpos[warp - kSoftmaxWarp0];
        float m_used = -INFINITY, l = 0.0f;  // R as this thread last knew it; l is relative to it
        bool ok = true;
        // tile i: S buffer `buf` = i % SBUFS, whose use it is the phase of
        int buf = odd, phase = 0;
        for (int i = odd; i < n; i += 2) {
            const int k0 = (t0 + i) * BN;
            if (kBias >= BIAS_PLANE) {
                __syncwarp();  // every lane is done with the last tile's copy
                constexpr int kAxes = kBias == BIAS_SPACE ? 3 : 2;
#pragma unroll
                for (int a = 0; a < kAxes; ++a)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = k0 + lane + 32 * e;
                        tail->kpos[warp - kSoftmaxWarp0][a][lane + 32 * e] =
                            key < q.len && a < p.pos_axes ? p.pos[(q.begin + key) * p.pos_row + a]
                                                          : 0.0f;
                    }
                __syncwarp();
            }
            const uint32_t s_col = t_lane + BN * buf;
            ok = wait_warp(&tail->s_full[buf], phase, ST_TIMEOUT_SOFTMAX, i);
            if (!ok) break;
            tc_fence_after();
            const int valid = seen - k0;
            // some row of the warp sees less than the whole tile
            const bool cut = __any_sync(kFull, valid < BN);
            const float rel = static_cast<float>(at - k0);
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t s[32];
                tmem_ld32(s_col + 32 * h, s);
                tmem_wait_ld();
                if (!kPlain) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int k = 32 * h + e;
                        float t = __uint_as_float(s[e]) * in;
                        if (kCap) t = fmaf(rcp_approx(1.0f + ex2(t)), -2.0f * cap2, cap2);
                        if (kBias == BIAS_INDEX)
                            t = fmaf(-slope2, fabsf(rel - static_cast<float>(k)), t);
                        if (kBias >= BIAS_PLANE) {
                            const float x = qp[0] - kpos[0][k], y = qp[1] - kpos[1][k];
                            float d2 = fmaf(x, x, y * y);
                            if (kBias == BIAS_SPACE) {
                                const float z = qp[2] - kpos[2][k];
                                d2 = fmaf(z, z, d2);
                            }
                            t = fmaf(-slope2, sqrt_approx(d2), t);
                        }
                        s[e] = __float_as_uint(t);
                    }
                }
                if (cut) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * h + e >= valid) s[e] = __float_as_uint(-INFINITY);
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mx[j] = fmax3(mx[j], __uint_as_float(s[e + 2 * j]),
                                      __uint_as_float(s[e + 2 * j + 1]));
                if (!kPlain) tmem_st32(s_col + 32 * h, s);
            }
            if (!kPlain) tmem_wait_st();
            const float m_row = fmax3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
            // R(i) from R(i - 1), the other stream's, and this tile's maximum
            float prev = -INFINITY;
            if (i > 0) {
                ok = wait_warp(&tail->ref_full[odd ^ 1][sub], ((i - 1) >> 1) & 1, ST_TIMEOUT_SOFTMAX,
                               0x10000 | i);
                if (!ok) break;
                prev = tail->ref[odd ^ 1][row];
            }
            const float m_new = fmaxf(prev, m_row * c);
            const bool need = m_new > prev + kRescaleThreshold;
            const float now = need ? m_new : prev;
            tail->ref[odd][row] = now;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&tail->ref_full[odd][sub]));
            // raised here or by the other stream: rare after the first tiles
            const bool raised = __any_sync(kFull, now != m_used);
            if (raised) l *= now != m_used ? ex2(m_used - now) : 1.0f;
            m_used = now;
            if (raised && i > 0 && __any_sync(kFull, need)) {
                ok = wait_warp(&tail->o_done[(i - 1) % SBUFS], ((i - 1) / SBUFS) & 1,
                               ST_TIMEOUT_SOFTMAX, 0x20000 | i);
                if (!ok) break;
                tc_fence_after();
                const float alpha = need ? ex2(prev - now) : 1.0f;
#pragma unroll
                for (int h = 0; h < HD / 16; ++h) {
                    uint32_t o[16];
                    tmem_ld16(o_col + 16 * h, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                    tmem_st16(o_col + 16 * h, o);
                }
                tmem_wait_st();
            }
            // a row that has seen no key yet (another split's, or none) has no
            // maximum: its exponents are taken against 0
            const float nm = m_used == -INFINITY ? 0.0f : -m_used;
            const unsigned long long nm2 = f2pack(nm, nm), c2 = f2pack(c, c);
            unsigned long long acc[2] = {f2pack(0.0f, 0.0f), f2pack(0.0f, 0.0f)};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t s[32];
                tmem_ld32(s_col + 32 * h, s);
                tmem_wait_ld();
                if (kPlain && cut) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * h + e >= valid) s[e] = __float_as_uint(-INFINITY);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float x0, x1;
                    f2unpack(ffma2(f2pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])),
                                   c2, nm2), x0, x1);
                    x0 = ex2(x0), x1 = ex2(x1);
                    acc[e & 1] = fadd2(acc[e & 1], f2pack(x0, x1));
                    s[e] = pack_f16x2(x0, x1);
                }
                // P's columns [16 h, 16 h + 16) lie over scores already read
                tmem_st16(s_col + 16 * h, s);
            }
            float sa, sb;
            f2unpack(fadd2(acc[0], acc[1]), sa, sb);
            l += sa + sb;
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&tail->p_full[buf]));
            buf += 2;
            if (buf >= SBUFS) buf -= SBUFS, phase ^= 1;
        }
        if (odd) {
            tail->odd_sum[row] = l;
            tail->ref[1][row] = m_used;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&tail->odd_done));
        } else {
            ok = ok && wait_warp(&tail->odd_done, 0, ST_TIMEOUT_SOFTMAX, 0x30000);
            if (ok && n > 0) ok = wait_warp(&tail->o_final, 0, ST_TIMEOUT_SOFTMAX, 0x40000);
            tc_fence_after();
            // O is relative to the last R, the larger of the two
            const float other = ok ? tail->ref[1][row] : -INFINITY;
            const float top = ok ? fmaxf(m_used, other) : -INFINITY;
            const float ref = top == -INFINITY ? 0.0f : top;
            const float sum = ok ? ex2(m_used - ref) * l + ex2(other - ref) * tail->odd_sum[row] : 0.0f;
            const float w = p.splits == 1 ? 1.0f / sum : 1.0f;
            const long long to = (q.begin + at) * p.out_row + head * HD;
            float4* po = reinterpret_cast<float4*>(sK);
#pragma unroll
            for (int h = 0; h < HD / 16; ++h) {
                uint32_t a[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) a[k] = 0;
                if (ok && n > 0) tmem_ld16(o_col + 16 * h, a);
                tmem_wait_ld();
                float v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = w * __uint_as_float(a[k]);
                if (p.splits == 1) {
                    if (ok && live) {
                        store8(p.out, to + 16 * h, p.out_dtype, v);
                        store8(p.out, to + 16 * h + 8, p.out_dtype, v + 8);
                    }
                } else {
                    // the split's O of each row into the K ring, free by now
                    // (the last PV is complete, so every copy has landed and
                    // been read); a row's vectors rotated so that a warp's
                    // stores spread over the banks
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        po[row * 16 + ((4 * h + k) ^ (row & 15))] =
                            make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                }
            }
            if (p.splits > 1) reinterpret_cast<float2*>(sV)[row] = make_float2(top, sum);
        }
    }
    if (p.splits > 1) {
        // The cluster's CTAs share out the tile's rows; each adds every
        // split's part of its rows in rank order (the same bits in every run).
        __syncwarp();
        fence_cluster();
        cluster_sync();
        const int me = static_cast<int>(cluster_rank());
        const int r0 = BM * me / p.splits, r1 = min(BM * (me + 1) / p.splits, tail->rows);
        const long long to = (tail->span.begin + tail->q0) * p.out_row + head * HD;
        // (the loop's bound is the warp's, so that the warp reaches the cluster
        // barrier after it as one)
        for (int w0 = r0 * 16 + 32 * warp; w0 < r1 * 16; w0 += kTileThreads) {
            const int i = min(w0 + lane, r1 * 16 - 1);  // the last lanes repeat a store
            const int row = i >> 4, k = i & 15;
            const uint32_t at_ml = smem_u32(sV) + row * 8;
            const uint32_t at_o = smem_u32(sK) + (row * 16 + (k ^ (row & 15))) * 16;
            float2 ml[8];
            float4 o[8];
#pragma unroll
            for (int s = 0; s < 8; ++s)  // every load on its way before the first use
                if (s < p.splits) {
                    ml[s] = dsmem_ld2(dsmem_addr(at_ml, s));
                    o[s] = dsmem_ld4(dsmem_addr(at_o, s));
                }
            float top = -INFINITY;
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < p.splits) top = fmaxf(top, ml[s].x);
            const float ref = top == -INFINITY ? 0.0f : top;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float sum = 0.0f;
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < p.splits) {
                    const float w = ex2(ml[s].x - ref);
                    sum = fmaf(w, ml[s].y, sum);
                    a.x = fmaf(w, o[s].x, a.x), a.y = fmaf(w, o[s].y, a.y);
                    a.z = fmaf(w, o[s].z, a.z), a.w = fmaf(w, o[s].w, a.w);
                }
            const float inv = 1.0f / sum;
            store4(p.out, to + row * p.out_row + 4 * k, p.out_dtype,
                   make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
        }
        __syncwarp();
        cluster_sync();  // no CTA leaves while its part is read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

int validate(const bl_masked_attention_args& a) {
    if (a.head_dim != HD)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: head_dim %u (only 64)", a.head_dim);
    if (a.batch == 0 || a.tokens == 0 || a.heads == 0)
        return fail(BL_ERR_INVALID, "masked attention: zero dimension");
    const uint32_t kv = a.kv_heads ? a.kv_heads : a.heads;
    if (a.heads % kv != 0)
        return fail(BL_ERR_INVALID, "masked attention: %u heads over %u K/V heads", a.heads, kv);
    if (a.heads > 65535 || kv > 65535)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: %u heads", a.heads);
    if (a.offsets != nullptr && a.lengths != nullptr)
        return fail(BL_ERR_INVALID, "masked attention: offsets (packed) and lengths (padded)");
    const uint64_t rows = a.offsets != nullptr ? a.tokens : 1ull * a.batch * a.tokens;
    if (a.tokens > 0x7FFFFFFFu || a.batch > 0x7FFF0000u || rows > 0x7FFFFFFFull)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: %u sequences of %u rows", a.batch, a.tokens);
    if (a.qk_dtype != BL_F16 && a.qk_dtype != BL_BF16)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: Q/K dtype %d (f16 or bf16)", a.qk_dtype);
    if (a.v_dtype != BL_F16)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: V dtype %d (f16 only)", a.v_dtype);
    if (a.out_dtype != BL_F32 && a.out_dtype != BL_F16 && a.out_dtype != BL_BF16)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: out dtype %d", a.out_dtype);
    if (!(a.scale > 0.0f) || !std::isfinite(a.scale))
        return fail(BL_ERR_INVALID, "masked attention: scale must be finite and positive");
    if (!(a.cap >= 0.0f) || !std::isfinite(a.cap))
        return fail(BL_ERR_INVALID, "masked attention: cap must be finite, 0 for none");
    if (a.mask < BL_MASK_NONE || a.mask > BL_MASK_PREFIX)
        return fail(BL_ERR_INVALID, "masked attention: mask %d", a.mask);
    if ((a.mask == BL_MASK_PREFIX) != (a.prefix != nullptr))
        return fail(BL_ERR_INVALID, "masked attention: prefix lengths go with the prefix mask alone");
    if (a.positions != nullptr && a.slopes == nullptr)
        return fail(BL_ERR_INVALID, "masked attention: positions without slopes");
    if (a.positions != nullptr && (a.pos_axes < 1 || a.pos_axes > 3))
        return fail(BL_ERR_INVALID, "masked attention: %u position axes (1 to 3)", a.pos_axes);
    if (a.positions != nullptr && a.pos_row_stride != 0 && a.pos_row_stride < a.pos_axes)
        return fail(BL_ERR_INVALID, "masked attention: a position row is shorter than its axes");
    if (a.key_splits > 8)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: %u key splits (at most 8)", a.key_splits);
    if (a.qkv == nullptr || a.out == nullptr)
        return fail(BL_ERR_INVALID, "masked attention: null pointer");
    const uint64_t width = (1ull * a.heads + 2ull * kv) * HD, ow = 1ull * a.heads * HD;
    const uint64_t row = a.qkv_row_stride ? a.qkv_row_stride : width;
    const uint64_t orow = a.out_row_stride ? a.out_row_stride : ow;
    if (row < width || row % 8 != 0 || row >= (1ull << 31) ||
        (reinterpret_cast<uintptr_t>(a.qkv) & 15u))
        return fail(BL_ERR_INVALID, "masked attention: qkv row stride %llu or alignment",
                    (unsigned long long)row);
    if (orow < ow || (orow * dtype_size(a.out_dtype)) % 16 != 0 || orow >= (1ull << 40) ||
        (reinterpret_cast<uintptr_t>(a.out) & 15u))
        return fail(BL_ERR_INVALID, "masked attention: output stride or alignment");
    for (const void* q : {static_cast<const void*>(a.offsets), static_cast<const void*>(a.lengths),
                          static_cast<const void*>(a.prefix), static_cast<const void*>(a.slopes),
                          static_cast<const void*>(a.positions)})
        if (reinterpret_cast<uintptr_t>(q) & 3u)
            return fail(BL_ERR_INVALID, "masked attention: a table is not 4-byte aligned");
    return BL_OK;
}

Params params_of(const bl_masked_attention_args& a) {
    Params p{};
    const uint32_t kv = a.kv_heads ? a.kv_heads : a.heads;
    p.batch = static_cast<int>(a.batch), p.tokens = static_cast<int>(a.tokens);
    p.heads = static_cast<int>(a.heads), p.kv_heads = static_cast<int>(kv);
    p.group = static_cast<int>(a.heads / kv);
    p.last_rows = static_cast<int>(std::min(a.last_rows, a.tokens));
    p.scale = a.scale, p.cap = a.cap, p.mask = a.mask;
    p.qkv = static_cast<const uint16_t*>(a.qkv);
    p.row = static_cast<long long>(a.qkv_row_stride ? a.qkv_row_stride
                                                    : (1ull * a.heads + 2ull * kv) * HD);
    p.out = a.out, p.out_dtype = a.out_dtype;
    p.out_row = static_cast<long long>(a.out_row_stride ? a.out_row_stride : 1ull * a.heads * HD);
    p.offsets = a.offsets, p.lengths = a.lengths, p.prefix = a.prefix;
    p.slopes = a.slopes, p.pos = a.positions;
    p.pos_row = static_cast<long long>(a.pos_row_stride ? a.pos_row_stride : a.pos_axes);
    p.pos_axes = static_cast<int>(a.pos_axes);
    p.status = status_ptr();
    return p;
}

int prepare_rows(const bl_masked_attention_args& a, Launch* out) {
    Params p = params_of(a);
    const uint64_t rows = p.last_rows > 0 ? p.last_rows : p.tokens;
    const uint64_t combos = rows * p.group;
    const int r = combos <= 1 ? 1 : combos <= 2 ? 2 : 4;
    p.chunks = static_cast<int>((combos + r - 1) / r);
    const uint64_t units = 1ull * p.chunks * a.batch;
    const uint64_t ctas = units * p.kv_heads;
    p.splits = a.key_splits ? static_cast<int>(a.key_splits)
                            : static_cast<int>(std::max<uint64_t>(
                                  1, std::min<uint64_t>({8, 296 / ctas, (a.tokens + 255ull) / 256})));
    if (units * p.splits > 0x7FFFFFFFull)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: grid too large");
    auto kern = r == 1 ? rows_kernel<1> : r == 2 ? rows_kernel<2> : rows_kernel<4>;
    const dim3 grid(static_cast<unsigned>(units * p.splits), p.kv_heads);
    const int bf16 = a.qk_dtype == BL_BF16;
    out->op = BL_OP_MASKED_ATTENTION;
    out->run = [=](cudaStream_t s) {
        return p.splits > 1 ? launch_k_cluster(kern, grid, dim3(32 * kWarps), dim3(p.splits, 1, 1),
                                               0, s, p, bf16)
                            : launch_k(kern, grid, dim3(32 * kWarps), 0, s, p, bf16);
    };
    return BL_OK;
}

int prepare_tiles(const bl_masked_attention_args& a, Launch* out) {
    Params p = params_of(a);
    // Tiles: a packed batch has at most one short tile a sequence beside its
    // whole ones; the kernel finds which exist (chunks = 0). Otherwise every
    // sequence has as many as its longest form.
    const bool packed = a.offsets != nullptr && p.last_rows == 0;
    const uint64_t per_seq = ((p.last_rows > 0 ? p.last_rows : p.tokens) + BM - 1ull) / BM;
    const uint64_t units = packed ? p.tokens / BM + std::min<uint64_t>(a.batch, a.tokens)
                                  : per_seq * a.batch;
    p.chunks = packed ? 0 : static_cast<int>(per_seq);
    // Split the keys while that many CTAs still run at once (two an SM) and
    // each keeps 256 keys of an average sequence.
    const uint64_t keys = a.offsets != nullptr ? a.tokens / a.batch : a.tokens;
    p.splits = a.key_splits ? static_cast<int>(a.key_splits)
                            : static_cast<int>(std::max<uint64_t>(
                                  1, std::min<uint64_t>({8, 296 / (units * p.heads), keys / 256})));
    if (units * p.splits > 0x7FFFFFFFull)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: grid too large");
    const uint64_t rows = a.offsets != nullptr ? a.tokens : 1ull * a.batch * a.tokens;
    CUtensorMap tm_q, tm_kv;
    const uint64_t dims[2] = {static_cast<uint64_t>(p.heads + 2 * p.kv_heads) * HD, rows};
    const uint32_t qbox[2] = {HD, BM}, kbox[2] = {HD, BN};
    int rc = make_tmap_16bit_2d(&tm_q, a.qkv, dims, static_cast<uint64_t>(p.row) * 2, qbox);
    if (rc == BL_OK)
        rc = make_tmap_16bit_2d(&tm_kv, a.qkv, dims, static_cast<uint64_t>(p.row) * 2, kbox);
    if (rc != BL_OK) return rc;
    using Kern = void (*)(const CUtensorMap, const CUtensorMap, const Params, int);
    static const Kern kerns[2][4] = {
        {tile_kernel<false, BIAS_NONE>, tile_kernel<false, BIAS_INDEX>,
         tile_kernel<false, BIAS_PLANE>, tile_kernel<false, BIAS_SPACE>},
        {tile_kernel<true, BIAS_NONE>, tile_kernel<true, BIAS_INDEX>,
         tile_kernel<true, BIAS_PLANE>, tile_kernel<true, BIAS_SPACE>}};
    const int bias = p.slopes == nullptr ? BIAS_NONE
                     : p.pos == nullptr  ? BIAS_INDEX
                     : p.pos_axes <= 2   ? BIAS_PLANE
                                         : BIAS_SPACE;
    const Kern kern = kerns[p.cap > 0.0f ? 1 : 0][bias];
    BL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(kTileSmem)));
    const dim3 grid(static_cast<unsigned>(units * p.splits), p.heads);
    const int bf16 = a.qk_dtype == BL_BF16;
    out->op = BL_OP_MASKED_ATTENTION;
    out->run = [=](cudaStream_t s) {
        return p.splits > 1 ? launch_k_cluster(kern, grid, dim3(kTileThreads), dim3(p.splits, 1, 1),
                                               kTileSmem, s, tm_q, tm_kv, p, bf16)
                            : launch_k(kern, grid, dim3(kTileThreads), kTileSmem, s, tm_q, tm_kv, p,
                                       bf16);
    };
    return BL_OK;
}

}  // namespace masked

int prepare_masked_attention(const bl_masked_attention_args& a, Launch* out) {
    const int rc = masked::validate(a);
    if (rc != BL_OK) return rc;
    // The last rows of a stream: while a K/V head's query rows are few, the
    // tensor cores' 128-row tile would be nearly empty and the keys' bytes
    // are what counts.
    const uint32_t kv = a.kv_heads ? a.kv_heads : a.heads;
    const uint64_t combos = 1ull * std::min(a.last_rows, a.tokens) * (a.heads / kv);
    return a.last_rows > 0 && combos <= 4 ? masked::prepare_rows(a, out)
                                          : masked::prepare_tiles(a, out);
}

}  // namespace bl

extern "C" int bl_masked_attention(const bl_masked_attention_args* args, void* stream) {
    if (args == nullptr) return bl::fail(BL_ERR_INVALID, "masked attention: null args");
    return bl::guarded("masked attention", [&] {
        bl::Launch l;
        const int rc = bl::prepare_masked_attention(*args, &l);
        return rc != BL_OK ? rc : bl::enqueue(l, static_cast<cudaStream_t>(stream));
    });
}
