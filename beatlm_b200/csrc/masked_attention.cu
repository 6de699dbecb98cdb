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
#include <limits>
#include <type_traits>

#include "host.h"

namespace bl {
namespace masked {

constexpr int HD = 64;
constexpr unsigned kSms = 148;
constexpr float kLog2e = 1.4426950408889634f;

// What capping a score needs, made once on the host.
struct Capping {
    float unit;   // raw score -> u = s / cap
    float c[4];   // the coefficients of tanh's series for raw scores, in log2 units
    float twice;  // raw score -> 2 u in log2 units
    float cap2;   // cap in log2 units
};

struct Params {
    int batch, tokens;
    int heads, kv_heads, group;  // group = heads / kv_heads
    int last_rows;
    float scale, cap;
    Capping capping;
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
    int chunks;         // query tiles a sequence has at most
    int ragged;         // the sequences' lengths are in device memory
    int mixed;          // a cluster splits the keys of long tiles alone
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

// Scores are kept in log2 units.
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

__device__ __forceinline__ unsigned long long both(float v) { return f2pack(v, v); }

// cap tanh(s / cap) of raw scores, in log2 units. Up to |u| = |s / cap| =
// kSmallTanh by the odd series through u^7 on the FMA units (the first term
// left out is below 4 10^-7 of the value there), as s times a cubic in s^2.
// Beyond it as cap - 2 cap / (1 + e^(2 u)), from two approximate functions: an
// absolute error of a few 2^-23 cap, so a few 2^-21 of the value, for any cap;
// it goes to +-cap at the ends without a branch. Where the whole tile of a warp
// is below the limit (`small`) the series alone spares the unit that the
// exponentials need two of its three functions a score: 8 images of up to 1600
// rows, 16 heads, distances on the grid, take 147 us with scores below a quarter
// of their cap and 228 to 241 with scores that pass it.
constexpr float kSmallTanh = 0.25f;
__device__ __forceinline__ float capped_far(float s, const Capping& k) {
    return fmaf(rcp_approx(1.0f + ex2(s * k.twice)), -2.0f * k.cap2, k.cap2);
}
__device__ __forceinline__ unsigned long long capped_small2(unsigned long long s, const Capping& k) {
    const unsigned long long z = fmul2(s, s);
    unsigned long long c = ffma2(z, both(k.c[3]), both(k.c[2]));
    c = ffma2(z, c, both(k.c[1]));
    c = ffma2(z, c, both(k.c[0]));
    return fmul2(s, c);
}
template <bool kSmall>
__device__ __forceinline__ unsigned long long capped2(unsigned long long s, const Capping& k) {
    const unsigned long long near = capped_small2(s, k);
    if (kSmall) return near;
    float a, b, x, y;
    f2unpack(s, a, b);
    f2unpack(near, x, y);
    return f2pack(fabsf(a * k.unit) > kSmallTanh ? capped_far(a, k) : x,
                  fabsf(b * k.unit) > kSmallTanh ? capped_far(b, k) : y);
}
__device__ __forceinline__ float capped(float s, const Capping& k) {
    float x, y;
    f2unpack(capped2<false>(both(s), k), x, y);
    return x;
}

// ------------------------------------------------------------------ few rows
//
// The newest rows of a stream: up to 16 query rows of one K/V head (rows and
// heads of its group alike), for which the keys' bytes are what counts. Each of
// a CTA's four warps walks its own 32-key tiles of one split of the keys, one
// tile ahead of the one it works on (8 KB each, in a shared-memory ring of the
// warp's own, so no barrier between warps). 16 rows are the smallest tile of the
// warp-level tensor instruction (m16n8k16), which takes S = Q K^T and O += P V
// of 16 keys in 16 instructions, so the arithmetic stays below the bytes: on the
// FMA units one row alone cost 400 instructions for 16 keys. Scores, maxima,
// sums and O are f32, P is rounded to f16 for the product (it is at most 1: the
// running maximum is exact here), which costs 2^-11 of each at most. Warps are
// merged once at the end; the CTAs of a cluster send their rows' parts into the
// first one's shared memory and leave, and that adds them in rank order.
// 16 streams of up to 8192 rows, 16 heads over 8 K/V heads (160 MB): 31.2 us,
// 79% of a copy's rate (on the FMA units 86.5), whether the scores reach their
// cap or not; with positions, which are loaded a key at a time where they are
// used, 52.6 us for two axes and 57.4 for three. Three stages take a fifth
// longer (fewer CTAs an SM), 16-key tiles with four 15%.
constexpr int kRowWarps = 4;
constexpr int kRowTile = 32;    // keys of a tile
constexpr int kRowStages = 2;
constexpr int kMaxRows = 16;    // query rows of a CTA
constexpr int kRowTileBytes = 2 * kRowTile * HD * 2;  // K, then V
constexpr size_t kRowRing = kRowWarps * kRowStages * kRowTileBytes;
constexpr int kPartFloats = HD + 2;  // a row's O, maximum and sum from another split
static_assert(kRowStages * kRowTileBytes >= kMaxRows * HD * 4, "a warp's O over its ring");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    // past the split's keys nothing is read and zeros are written
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(real ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (kBf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
                     "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
                     "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool kBf16>
__global__ void __launch_bounds__(32 * kRowWarps) rows_kernel(const __grid_constant__ Params p) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float2 part_ml[kRowWarps][kMaxRows];
    __shared__ uint64_t parts_full;
    float* parts = reinterpret_cast<float*>(ring + kRowRing);  // [split][row][kPartFloats]
    constexpr unsigned kFull = 0xFFFFFFFFu;
    const int warp = warp_id(), lane = lane_id();
    // The heads of the same keys start side by side: their 128-byte parts of
    // a packed row are neighbours, so memory pages are read while they are open.
    const unsigned work = blockIdx.x / static_cast<unsigned>(p.splits);
    const int split = static_cast<int>(blockIdx.x - work * p.splits);
    int seq = static_cast<int>(work / static_cast<unsigned>(p.kv_heads));
    const int kvh = static_cast<int>(work - static_cast<unsigned>(seq) * p.kv_heads);
    // the longest streams first: their CTAs are not the last to start
    if (p.ragged && p.batch <= 32) {
        const int len = span_of(p, min(lane, p.batch - 1)).len;
        int longer = lane < p.batch ? 0 : p.batch;
        for (int j = 0; j < p.batch; ++j) {
            const int other = __shfl_sync(kFull, len, j);
            longer += other > len || (other == len && j < lane);
        }
        seq = __ffs(__ballot_sync(kFull, longer == seq && lane < p.batch)) - 1;
    }
    const Span q = span_of(p, seq);
    const int rows = (q.len - q.first) * p.group;  // at most kMaxRows
    if (rows == 0) return;  // the whole cluster leaves
    if (p.splits > 1) {
        if (threadIdx.x == 0) {
            mbar_init(smem_u32(&parts_full), p.splits - 1);
            fence_barrier_init();
        }
        __syncwarp();
        cluster_arrive();  // waited for before the parts are sent
    }

    const int most = visible(p, q, q.len - 1);  // of the last row
    const int least = visible(p, q, q.first);   // of the first
    const int tiles = (most + kRowTile - 1) / kRowTile;
    const int first = static_cast<int>(static_cast<unsigned>(tiles) * split / p.splits);
    const int last = static_cast<int>(static_cast<unsigned>(tiles) * (split + 1) / p.splits);

    // A lane copies one 16-byte part of every fourth key of a tile. A key row is
    // 128 bytes: its eight parts are rotated by the row, so that the matrix
    // loads meet no bank twice; (4 i + r) & 7 is r or r ^ 4.
    const int lr = lane >> 3, lp = lane & 7;
    const uint16_t* src = p.qkv + (q.begin + (first + warp) * kRowTile + lr) * p.row +
                          (p.heads + kvh) * HD + lp * 8;
    const long long to_v = static_cast<long long>(p.kv_heads) * HD, four = 4 * p.row;
    const uint32_t mine = smem_u32(ring) + warp * kRowStages * kRowTileBytes;
    const uint32_t at0 = lr * 128 + ((lp ^ lr) << 4), at1 = lr * 128 + ((lp ^ lr ^ 4) << 4);
    auto fetch = [&](int tile, int stage) {
        if (tile < last) {
            const uint32_t dst = mine + stage * kRowTileBytes;
            const int left = most - tile * kRowTile - lr;  // this lane's keys before the end
#pragma unroll
            for (int i = 0; i < kRowTile / 4; ++i) {
                const uint32_t at = dst + i * 512 + (i % 2 == 0 ? at0 : at1);
                const bool real = 4 * i < left;
                const uint16_t* from = real ? src + i * four : p.qkv;
                cp_async16(at, from, real);
                cp_async16(at + kRowTile * 128, real ? from + to_v : p.qkv, real);
            }
            src += kRowWarps * kRowTile / 4 * four;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < kRowStages - 1; ++i) fetch(first + warp + i * kRowWarps, i);

    // This thread's two query rows (of the 16: g and g + 8), as the products'
    // accumulators hold them; a row past the last repeats it and is not stored.
    const int g = lane >> 2, quad = lane & 3;
    int row[2], seen[2];
    float slope[2], qp[2][3];
    uint32_t qa[HD / 16][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int c = min(g + 8 * r, rows - 1);
        const int head = kvh * p.group + c % p.group;
        row[r] = q.first + c / p.group;
        seen[r] = visible(p, q, row[r]);
        slope[r] = p.slopes != nullptr ? p.slopes[head] * kLog2e : 0.0f;
        const uint16_t* src = p.qkv + (q.begin + row[r]) * p.row + head * HD + 2 * quad;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            qa[k][r] = *reinterpret_cast<const uint32_t*>(src + 16 * k);
            qa[k][r + 2] = *reinterpret_cast<const uint32_t*>(src + 16 * k + 8);
        }
#pragma unroll
        for (int a = 0; a < 3; ++a)
            qp[r][a] = p.pos != nullptr && a < p.pos_axes
                           ? p.pos[(q.begin + row[r]) * p.pos_row + a] : 0.0f;
    }
    float o[HD / 8][4];
#pragma unroll
    for (int d = 0; d < HD / 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const bool capped_scores = p.cap > 0.0f;
    const float in = p.scale * kLog2e;
    const Capping& cap = p.capping;

    int stage = 0;
    for (int tile = first + warp; tile < last; tile += kRowWarps) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 2) : "memory");
        __syncwarp();
        // the stage read last time is free: every lane is past it
        fetch(tile + (kRowStages - 1) * kRowWarps, (stage + kRowStages - 1) % kRowStages);
        const uint32_t sk = mine + stage * kRowTileBytes, sv = sk + kRowTile * 128;
        stage = (stage + 1) % kRowStages;
        const int base = tile * kRowTile;
        // s[t][2 r + e]: query row g + 8 r, key base + 8 t + 2 quad + e
        constexpr int T = kRowTile / 8;
        float s[T][4];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
            for (int t = 0; t < T; t += 2) {
                // eight keys, then eight, by the two halves of 16 columns
                uint32_t b[4];
                const int key = 8 * t + (lane >> 4) * 8 + (lane & 7);
                const int part = 2 * k + ((lane >> 3) & 1);
                ldmatrix4(sk + key * 128 + ((part ^ (key & 7)) << 4), b);
                mma16<kBf16>(s[t], qa[k], b[0], b[1]);
                mma16<kBf16>(s[t + 1], qa[k], b[2], b[3]);
            }
        auto each = [&](auto&& f) {  // f(score, its row of the two, its key - base - 2 quad)
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] = f(s[t][e], e >> 1, 8 * t + (e & 1));
        };
        if (capped_scores) {
            float far = 0.0f;
            each([&](float x, int, int) { far = fmaxf(far, fabsf(x)); return x; });
            auto cap_all = [&](auto small) {
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int e = 0; e < 4; e += 2)
                        f2unpack(capped2<decltype(small)::value>(f2pack(s[t][e], s[t][e + 1]), cap),
                                 s[t][e], s[t][e + 1]);
            };
            if (__any_sync(kFull, far * cap.unit > kSmallTanh)) cap_all(std::false_type{});
            else cap_all(std::true_type{});
        } else {
            each([&](float x, int, int) { return x * in; });
        }
        const int own = base + 2 * quad;  // this lane's first key
        if (p.slopes != nullptr) {
            if (p.pos == nullptr) {
                const float rel[2] = {static_cast<float>(row[0] - own), static_cast<float>(row[1] - own)};
                each([&](float x, int r, int k) {
                    return fmaf(-slope[r], fabsf(rel[r] - static_cast<float>(k)), x);
                });
            } else {
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = min(own + 8 * t + e, most - 1);
                        float d2[2] = {0.0f, 0.0f};
                        for (int a = 0; a < p.pos_axes; ++a) {
                            const float kp = p.pos[(q.begin + key) * p.pos_row + a];
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float d = (a == 0 ? qp[r][0] : a == 1 ? qp[r][1] : qp[r][2]) - kp;
                                d2[r] = fmaf(d, d, d2[r]);
                            }
                        }
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            s[t][2 * r + e] = fmaf(-slope[r], sqrt_approx(d2[r]), s[t][2 * r + e]);
                    }
            }
        }
        if (base + kRowTile > least)  // some row sees less than the whole tile
            each([&](float x, int r, int k) { return own + k < seen[r] ? x : -INFINITY; });
        float top[2] = {-INFINITY, -INFINITY};
        each([&](float x, int r, int) { top[r] = fmaxf(top[r], x); return x; });
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(kFull, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(kFull, top[r], 2));
            top[r] = fmaxf(top[r], m[r]);
        }
        if (__any_sync(kFull, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float shrink = ex2(m[r] - (top[r] == -INFINITY ? 0.0f : top[r]));
                m[r] = top[r];
                l[r] *= shrink;
#pragma unroll
                for (int d = 0; d < HD / 8; ++d) o[d][2 * r] *= shrink, o[d][2 * r + 1] *= shrink;
            }
        }
        // (no key seen yet: against 0)
        const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
        each([&](float x, int r, int) {
            const float v = ex2(x - ref[r]);
            l[r] += v;
            return v;
        });
#pragma unroll
        for (int t = 0; t < T; t += 2) {
            const uint32_t pa[4] = {pack_f16x2(s[t][0], s[t][1]), pack_f16x2(s[t][2], s[t][3]),
                                    pack_f16x2(s[t + 1][0], s[t + 1][1]),
                                    pack_f16x2(s[t + 1][2], s[t + 1][3])};
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                // keys 8 t.. and 8 t + 8.. of columns 16 d.., then of the next 8
                uint32_t b[4];
                const int key = 8 * t + (lane & 15), part = 2 * d + (lane >> 4);
                ldmatrix4_trans(sv + key * 128 + ((part ^ (key & 7)) << 4), b);
                mma16<false>(o[2 * d], pa, b[0], b[1]);
                mma16<false>(o[2 * d + 1], pa, b[2], b[3]);
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    // the warp's sums, and its O over its ring
    float* po = reinterpret_cast<float*>(ring + warp * kRowStages * kRowTileBytes);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(kFull, l[r], 1);
        l[r] += __shfl_xor_sync(kFull, l[r], 2);
        if (quad == 0) part_ml[warp][g + 8 * r] = make_float2(m[r], l[r]);
#pragma unroll
        for (int d = 0; d < HD / 8; ++d)
            *reinterpret_cast<float2*>(po + (g + 8 * r) * HD + 8 * d + 2 * quad) =
                make_float2(o[d][2 * r], o[d][2 * r + 1]);
    }
    __syncthreads();
    auto put = [&](int r, int e, float v) {
        const long long at = (q.begin + q.first + r / p.group) * p.out_row +
                             (kvh * p.group + r % p.group) * HD + e;
        if (p.out_dtype == BL_F32) static_cast<float*>(p.out)[at] = v;
        else if (p.out_dtype == BL_F16) static_cast<__half*>(p.out)[at] = __float2half_rn(v);
        else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    };
    if (p.splits > 1) cluster_wait();  // the first CTA is there
    // warps -> CTA, and to the cluster's first one
    for (int t = threadIdx.x; t < rows * HD; t += 32 * kRowWarps) {
        const int r = t / HD, e = t % HD;
        float best = -INFINITY, v = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) best = fmaxf(best, part_ml[w][r].x);
        const float ref = best == -INFINITY ? 0.0f : best;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) {
            const float f = ex2(part_ml[w][r].x - ref);
            v = fmaf(f, reinterpret_cast<const float*>(ring + w * kRowStages * kRowTileBytes)[r * HD + e], v);
            sum = fmaf(f, part_ml[w][r].y, sum);
        }
        if (p.splits == 1) {
            put(r, e, v / sum);
            continue;
        }
        const uint32_t to = dsmem_addr(smem_u32(parts + (split * rows + r) * kPartFloats), 0);
        dsmem_st1(to + 4 * e, v);
        if (e == 0) dsmem_st2(to + 4 * HD, best, sum);
    }
    if (p.splits == 1) return;
    fence_cluster();
    __syncthreads();
    if (split != 0) {
        if (threadIdx.x == 0)
            mbar_arrive_remote(dsmem_addr(smem_u32(&parts_full), 0));
        return;
    }
    if (!mbar_wait_cluster(smem_u32(&parts_full), 0, nullptr, p.status, ST_TIMEOUT_SOFTMAX, 0x50000))
        return;
    for (int t = threadIdx.x; t < rows * HD; t += 32 * kRowWarps) {
        const int r = t / HD, e = t % HD;
        float best = -INFINITY, total = 0.0f, sum = 0.0f;
        for (int k = 0; k < p.splits; ++k)
            best = fmaxf(best, parts[(k * rows + r) * kPartFloats + HD]);
        const float ref = best == -INFINITY ? 0.0f : best;
        for (int k = 0; k < p.splits; ++k) {
            const float* part = parts + (k * rows + r) * kPartFloats;
            const float f = ex2(part[HD] - ref);
            total = fmaf(f, part[e], total);
            sum = fmaf(f, part[HD + 1], sum);
        }
        put(r, e, total / sum);
    }
}

// ------------------------------------------------------------------ tiles
//
// One CTA computes 128 query rows of one head over a range of 64-key tiles on
// the tensor cores; two CTAs share an SM, with half the TMEM each. The
// exponentials bound it (one a score at 16 a clock and SM, against half of that
// time for its products), so the rest is there to keep that unit fed.
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
// registers that ten warps and two CTAs allow. P is rounded to f16, the type of V
// (an instruction takes one type), by 2^-11 of a probability at most or by 2^-25
// of the reference below f16's normal range; its sum is of the f32 values.
// One sequence of 10960 rows, 16 heads: 632 us, 778 TFLOP/s in short runs at
// 1965 MHz (692 in long ones, at the power cap); the exponentials' unit is busy
// for 66% of a step (776 clocks of an SM for 128 x 64 scores, 512 at its rate;
// the rest is the softmax threads' way from S to the running maximum, which the
// four of a scheduler cover in part). Making an eighth to a
// third of the exponentials by a polynomial on the FMA units lengthens that way
// and takes 645 to 670 us. A CTA's start and end cost 9000 clocks beside its steps.
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

// The bias of |i - j| comes out of the tensor cores where it is linear over a
// tile, that is where every key that any row of the CTA sees lies on one side
// of the row: it is then lean (k - rel) for key k of the tile, and one more K
// step of the product S adds (slope / scale) k to every score, with the
// operands below; -lean rel is the row's and goes into its exponents' offset.
// So a linear tile costs the softmax nothing. Both halves of the K step hold
// the same (half of the slope each), so the swizzle does not matter; the slope
// is the sum of three bf16 values (24 bits), the key's number is exact.
struct LeanOperands {
    uint8_t slope[BM * 32];      // A: every row the slope's three parts, twice
    uint8_t key[2][BN * 32];     // B: row k holds k (or -k) three times, twice
};

static_assert((kQBytes + 2 * STAGES * kKvBytes) % 1024 == 0, "the tail starts on a swizzle atom");
struct TileTail {
    union {  // first, so that matrix operands and 16-byte loads are aligned
        LeanOperands lean;
        float kpos[8][3][BN];  // each softmax warp's copy of a key tile's positions, negated
    };
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
    int pivot;      // the one with the nearest keys, of the n; -1: in rising order
    int splits, split;  // CTAs that share the tile's keys, and which of them this is
    float ref[2][BM];      // R after the stream's last tile
    float odd_sum[BM];
};
constexpr size_t kTileSmem = 1024 + kQBytes + 2 * STAGES * kKvBytes + sizeof(TileTail);
static_assert(2 * (kTileSmem + 1024) <= 233472, "two CTAs an SM");

// On which side of all the CTA's rows the keys of the tile at k0 lie that any of
// them sees: 1 before, -1 behind, 0 on both. Under a causal mask, and behind a
// prefix, no row sees a key behind itself.
__device__ __forceinline__ int side_of(const Params& p, int prefix, int q0, int k0) {
    if (k0 + BN - 1 <= q0 || (p.mask != BL_MASK_NONE && k0 >= prefix)) return 1;
    return k0 >= q0 + BM - 1 ? -1 : 0;
}

constexpr int kLongTile = 12;  // key tiles that a tile has at least to be shared

// The sequence of tile `index` of a batch of at most 32, its rows without the
// prefix, and the tile counted from the sequence's end, in the order of the
// tiles' keys, most first: a warp ranks them, one sequence a lane. Without a mask
// a sequence's tiles all have its length; under one, a tile further up has BM
// keys less, so the tiles of one level (whole tiles of rows up to the end of
// this one) are alike, and the level follows from how many tiles lie at or above
// each. With p.mixed a cluster shares the keys of one tile while the tile is
// long, and its CTAs take a tile each of the shorter ones (`parts` 1). What is
// long follows from the mean of the tiles' keys over the CTAs that run at once:
// without a mask half as much again (parts cost a start and a join each, so a
// split pays where the tile alone would outlast the others), under one the mean
// (the tiles below it are many), and where tiles left whole, which start last,
// would outlast them, half of a part of the longest.
// Returns the sequence, -1 behind the last tile.
__device__ __forceinline__ int ranked_tile(const Params& p, int index, Span& q, int& tile,
                                           int& parts, int& part) {
    constexpr unsigned kAll = 0xFFFFFFFFu;
    const int lane = lane_id();
    const Span mine = span_of(p, min(lane, p.batch - 1));
    const int len = lane < p.batch ? mine.len : 0;
    const int tiles = lane < p.batch ? (len - mine.first + BM - 1) / BM : 0;
    const int up = (len + BM - 1) / BM;  // the last tile's level; the others' below
    auto above = [&](int level) {        // tiles at this level or above
        return __reduce_add_sync(kAll, min(max(up - level + 1, 0), tiles));
    };
    if (p.mixed) {
        // key tiles of a head's tiles (longer streams count as 2^16 levels)
        const int most = 2 * min(up, 1 << 16), bound = min(tiles, 1 << 12);
        const int sum = bound * (p.mask == BL_MASK_NONE ? most : max(most - bound + 1, 0));
        const float mean = static_cast<float>(__reduce_add_sync(kAll, sum >> 5)) * 32.0f *
                           static_cast<float>(p.heads) / (2 * kSms);
        const float part_of = 0.5f * static_cast<float>(__reduce_max_sync(kAll, most)) / p.splits;
        const bool wave = gridDim.x <= 2 * kSms * p.splits;  // all tiles whole would be one
        const float from = p.splits > 2               ? part_of
                           : p.mask == BL_MASK_NONE   ? 1.5f * mean
                           : wave && part_of < mean   ? part_of
                                                      : mean;
        const int limit = max(static_cast<int>(from), kLongTile);
        const int shared = p.mask == BL_MASK_NONE
                               ? __reduce_add_sync(kAll, most > limit ? tiles : 0)
                               : above(limit / 2 + 1);
        if (index >= shared) {
            index = shared + (index - shared) * parts + part;
            parts = 1, part = 0;
        }
    }
    bool here;
    if (p.mask == BL_MASK_NONE) {
        int before = 0;  // tiles of the longer sequences
        for (int j = 0; j < p.batch; ++j) {
            const int other = __shfl_sync(kAll, len, j), count = __shfl_sync(kAll, tiles, j);
            if (other > len || (other == len && j < lane)) before += count;
        }
        tile = index - before;
        here = tile >= 0 && tile < tiles;
    } else {
        int lo = 0, hi = __reduce_max_sync(kAll, up);  // above(lo) > index, if any is
        if (above(0) <= index) return -1;
        while (lo < hi) {
            const int mid = lo + (hi - lo + 1) / 2;
            if (above(mid) > index) lo = mid; else hi = mid - 1;
        }
        tile = up - lo;
        const bool has = tile >= 0 && tile < tiles;
        const unsigned level = __ballot_sync(kAll, has);
        const int place = index - above(lo + 1);  // within the level
        here = has && __popc(level & ((1u << lane) - 1)) == place;
    }
    const unsigned found = __ballot_sync(kAll, here);
    if (found == 0) return -1;
    const int owner = __ffs(found) - 1;
    q.begin = __shfl_sync(kAll, mine.begin, owner);
    q.len = __shfl_sync(kAll, len, owner);
    q.first = __shfl_sync(kAll, mine.first, owner);
    tile = __shfl_sync(kAll, tile, owner);
    return owner;
}

// The same for a packed batch of more sequences, all their rows: in the
// sequences' order, which a warp walks 256 at a time, eight a lane, so that a
// chunk costs one round trip to memory.
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

// 32 raw scores capped in place. (A branch around each loop: inside it the two
// forms would both be computed.)
__device__ __forceinline__ void cap32(uint32_t (&s)[32], const Capping& k, bool small) {
    auto put = [&](int e, unsigned long long v) {
        float x, y;
        f2unpack(v, x, y);
        s[2 * e] = __float_as_uint(x), s[2 * e + 1] = __float_as_uint(y);
    };
    if (small) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            put(e, capped2<true>(f2pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), k));
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            put(e, capped2<false>(f2pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), k));
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
    // CTAs in the order of their start: the splits of a unit side by side (a
    // cluster), then the heads of a tile, so that the tiles with most keys (the
    // first units) start first in every head and the last CTAs are short
    unsigned work = blockIdx.x / static_cast<unsigned>(p.splits);
    const int rank = static_cast<int>(blockIdx.x - work * p.splits);
    // (one CTA an SM goes out before any SM gets its second: where all fit at
    // once, the second ones come lightest first, beside the heaviest)
    if (p.splits == 1 && gridDim.x <= 2 * kSms && work >= kSms) work = gridDim.x - 1 - (work - kSms);
    const int unit = static_cast<int>(work / static_cast<unsigned>(p.heads));
    const int head = static_cast<int>(work - static_cast<unsigned>(unit) * p.heads);
    const int kvh = head / p.group;
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
        // Only now may the next kernel's CTAs come beside this one (a trigger
        // counts once a CTA, whoever gives it): before it, one of them could
        // take the columns and wait for this kernel's end.
        pdl_trigger();
    }
    pdl_wait();
    if (warp == 0) {
        __syncwarp();
        Span q{};
        int tile = 0, rows = 0, q0 = 0, first = 0, count = 0, pivot = -1;
        int parts = p.splits, part = rank;
        if (p.batch <= 32 && (p.ragged || p.mixed)) {
            const int seq = ranked_tile(p, unit, q, tile, parts, part);
            if (seq < 0) q.len = 0;
            else if (p.mask == BL_MASK_PREFIX) q.prefix = min(max(p.prefix[seq], 0), q.len);
        } else if (p.chunks > 0) {
            q = span_of(p, unit % p.batch);
            tile = unit / p.batch;
        } else {
            int begin = 0;
            const int seq = find_tile(p, unit, begin, q.len, tile);
            q.begin = begin;
            if (seq < 0) q.len = 0;
            else if (p.mask == BL_MASK_PREFIX) q.prefix = min(max(p.prefix[seq], 0), q.len);
        }
        const int tiles = (q.len - q.first + BM - 1) / BM;
        if (tile >= 0 && tile < tiles) {
            tile = tiles - 1 - tile;  // with a causal mask the last rows see most
            q0 = q.first + tile * BM;
            rows = min(q.len - q0, BM);
            // below 2^25 tiles and at most 8 splits: 32 bits hold the products
            const unsigned nt = (visible(p, q, q0 + rows - 1) + BN - 1) / BN;
            first = static_cast<int>(nt * part / parts);
            count = static_cast<int>(nt * (part + 1) / parts) - first;
            if (kBias != BIAS_NONE)
                pivot = min(max((q0 + rows - 1) / BN - first, -1), count - 1);
        }
        if (lane == 0) {
            tail->span = q;
            tail->q0 = q0, tail->rows = rows, tail->t0 = first, tail->n = count;
            tail->pivot = pivot;
            tail->splits = parts, tail->split = part;
        }
        __syncwarp();
    }
    if (kBias == BIAS_INDEX && !kCap && warp >= kSoftmaxWarp0) {
        // 256 threads, 256 16-byte parts of A and as many of the two B
        const int t = threadIdx.x - 32 * kSoftmaxWarp0;
        const float half = 0.5f * p.slopes[head] / p.scale;
        const float a = __bfloat162float(__float2bfloat16_rn(half));
        const float b = __bfloat162float(__float2bfloat16_rn(half - a));
        reinterpret_cast<uint4*>(tail->lean.slope)[t] =
            make_uint4(pack_bf16x2(a, b), pack_bf16x2(half - a - b, 0.0f), 0, 0);
        const float k = static_cast<float>((t & 127) >> 1), e = t < 128 ? k : -k;
        reinterpret_cast<uint4*>(tail->lean.key)[t] =
            make_uint4(pack_bf16x2(e, e), pack_bf16x2(e, 0.0f), 0, 0);
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tail->tmem_base;
    if (tail->rows == 0) {  // no such tile (for all that would share it)
        if (warp == 1) tmem_dealloc(tmem, kTmemCols);
        return;
    }
    const int t0 = tail->t0, n = tail->n;
    const int splits = tail->splits, part_rows = (BM + splits - 1) / splits;
    // The first key of the i-th tile. With a bias of distance the nearest keys
    // come first, those before them downwards, then those behind: the largest
    // scores are then met at once, and the running maximum that O is relative
    // to stays. (In rising order a slope of 1/2 raised it with every tile:
    // 2800 of a step's 4900 clocks.)
    const int pivot = tail->pivot;
    auto first_key = [&](int i) { return (t0 + (i <= pivot ? pivot - i : i)) * BN; };

    // One lane waits and the vote hands its outcome to the warp, unless the
    // barrier is past that phase already. A vote orders no memory: __syncwarp
    // does, so that what came before the barrier's arrivals (R, sums in shared
    // memory) is there for the lanes that did not wait themselves.
    const bool elected = elect_one();
    auto wait_warp = [&](uint64_t* bar, int parity, uint32_t code, uint32_t where) -> bool {
        if (__all_sync(kFull, mbar_try_wait(smem_u32(bar), parity))) return true;
        bool r = true;
        if (elected) r = mbar_wait(smem_u32(bar), parity, abort, p.status, code, where);
        r = __all_sync(kFull, r);
        __syncwarp();
        return r;
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
                const int y = row0 + first_key(loaded);
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
        const int end = tail->span.len, prefix = tail->span.prefix, q0 = tail->q0;
        const uint32_t idesc_lean = idesc_f16(BM, BN, 1, 1, 0, 0);
        const uint64_t d_slope = sdesc_sw32(smem_u32(tail->lean.slope), 256);
        const uint64_t d_key = sdesc_sw32(smem_u32(tail->lean.key), 256);
        // ring places, stepped as the loop goes: S runs SBUFS tiles ahead of PV
        int sb = 0, st = 0, st_phase = 0;  // of the next S: TMEM buffer, stage
        int pb = 0, p_phase = 0, pt = 0;   // of the next PV
        auto wait_tile = [&](int i) -> bool {
            if (!wait_warp(&tail->kv_full[st], st_phase, ST_TIMEOUT_MMA, i)) return false;
            const int valid = end - first_key(i);
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
        auto issue_s = [&](int i) {
            const int side = kBias == BIAS_INDEX && !kCap ? side_of(p, prefix, q0, first_key(i)) : 0;
            const uint64_t b = dk + st * kStep;
            const uint32_t dst = tmem + BN * sb;
            if (elected) {
                mma_ss(dst, dq, b, idesc_s, 0u);
#pragma unroll
                for (int k = 1; k < HD / 16; ++k) mma_ss(dst, dq + 2 * k, b + 2 * k, idesc_s, 1u);
                if (side != 0)
                    mma_ss(dst, d_slope, d_key + (side < 0 ? sizeof(tail->lean.key[0]) >> 4 : 0),
                           idesc_lean, 1u);
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
            if (ok) issue_s(i);
        }
        for (int i = 0; i < n && ok; ++i) {
            // what S(i + 3) needs first: between P(i) and it stand only MMAs
            const bool more = i + SBUFS < n;
            if (more) ok = wait_tile(i + SBUFS);
            ok = ok && wait_warp(&tail->p_full[pb], p_phase, ST_TIMEOUT_MMA, 0x10000 | i);
            if (!ok) break;
            tc_fence_after();
            issue_pv(i);
            if (more) issue_s(i + SBUFS);
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
        constexpr bool kCapOnly = kCap && kBias == BIAS_NONE;
        // raw scores to log2 units; kPlain does it in the exponent's FMA
        const float in = p.scale * kLog2e;
        const Capping& cap = p.capping;
        const float slope2 = kBias != BIAS_NONE ? p.slopes[head] * kLog2e : 0.0f;
        constexpr int kAxes = kBias == BIAS_SPACE ? 3 : 2;
        unsigned long long qp2[kAxes];  // this row's place, twice
#pragma unroll
        for (int a = 0; a < kAxes; ++a)
            qp2[a] = both(kBias >= BIAS_PLANE && live && a < p.pos_axes
                              ? p.pos[(q.begin + at) * p.pos_row + a] : 0.0f);
        const float(*kpos)[BN] = tail->kpos[warp - kSoftmaxWarp0];
        float m_used = -INFINITY, l = 0.0f;  // R as this thread last knew it; l is relative to it
        bool ok = true;
        // tile i: S buffer `buf` = i % SBUFS, whose use it is the phase of
        int buf = odd, phase = 0;
        // the positions of this lane's two keys of the next tile
        float ahead[kAxes][2];
        auto fetch = [&](int i) {
#pragma unroll
            for (int a = 0; a < kAxes; ++a)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = first_key(i) + lane + 32 * e;
                    ahead[a][e] = i < n && key < q.len && a < p.pos_axes
                                      ? p.pos[(q.begin + key) * p.pos_row + a] : 0.0f;
                }
        };
        if (kBias >= BIAS_PLANE) fetch(odd);
        for (int i = odd; i < n; i += 2) {
            const int k0 = first_key(i);
            if (kBias >= BIAS_PLANE) {
                __syncwarp();  // every lane is done with the last tile's copy
#pragma unroll
                for (int a = 0; a < kAxes; ++a)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        tail->kpos[warp - kSoftmaxWarp0][a][lane + 32 * e] = -ahead[a][e];
                __syncwarp();
                fetch(i + 2);
            }
            const uint32_t s_col = t_lane + BN * buf;
            ok = wait_warp(&tail->s_full[buf], phase, ST_TIMEOUT_SOFTMAX, i);
            if (!ok) break;
            tc_fence_after();
            const int valid = seen - k0;
            // some row of the warp sees less than the whole tile
            const bool cut = __any_sync(kFull, valid < BN);
            const float rel = static_cast<float>(at - k0);
            // a linear bias (side_of): what is left of it is the row's
            const int side = kBias == BIAS_INDEX && !kCap ? side_of(p, q.prefix, tail->q0, k0) : 0;
            const bool linear = side != 0;
            const float lean = linear ? -static_cast<float>(side) * slope2 * rel : 0.0f;
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            float far = 0.0f;  // the largest |score|, for the capping's choice
            bool small = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t s[32];
                tmem_ld32(s_col + 32 * h, s);
                tmem_wait_ld();
                auto pair = [&](int e) {
                    return f2pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
                };
                auto set = [&](int e, unsigned long long v) {
                    float x, y;
                    f2unpack(v, x, y);
                    s[2 * e] = __float_as_uint(x), s[2 * e + 1] = __float_as_uint(y);
                };
                if (kCap) {
                    float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            f[j] = fmax3(f[j], fabsf(__uint_as_float(s[e + 2 * j])),
                                         fabsf(__uint_as_float(s[e + 2 * j + 1])));
                    far = fmax3(fmaxf(far, f[0]), fmaxf(f[1], f[2]), f[3]);
                    small = !__any_sync(kFull, far * cap.unit > kSmallTanh);
                }
                if (kBias != BIAS_NONE && !linear) {
                    const unsigned long long down = both(-slope2);
                    if (kCap) cap32(s, cap, small);
                    auto score = [&](int e) { return kCap ? pair(e) : fmul2(pair(e), both(in)); };
                    if (kBias == BIAS_INDEX) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float k = static_cast<float>(32 * h + 2 * e);
                            set(e, ffma2(down, f2pack(fabsf(rel - k), fabsf(rel - k - 1.0f)), score(e)));
                        }
                    } else {
                        // distances from the keys' places, four keys a load
                        auto root = [](unsigned long long v) {
                            float x, y;
                            f2unpack(v, x, y);
                            return f2pack(sqrt_approx(x), sqrt_approx(y));
                        };
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            unsigned long long d0 = 0, d1 = 0;
#pragma unroll
                            for (int a = 0; a < kAxes; ++a) {
                                const float4 w = *reinterpret_cast<const float4*>(&kpos[a][32 * h + 2 * e]);
                                const unsigned long long x0 = fadd2(qp2[a], f2pack(w.x, w.y));
                                const unsigned long long x1 = fadd2(qp2[a], f2pack(w.z, w.w));
                                d0 = a == 0 ? fmul2(x0, x0) : ffma2(x0, x0, d0);
                                d1 = a == 0 ? fmul2(x1, x1) : ffma2(x1, x1, d1);
                            }
                            set(e, ffma2(down, root(d0), score(e)));
                            set(e + 1, ffma2(down, root(d1), score(e + 1)));
                        }
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
                if (kBias != BIAS_NONE && !linear) tmem_st32(s_col + 32 * h, s);
            }
            if (kBias != BIAS_NONE && !linear) tmem_wait_st();
            float m_row = fmax3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
            if (kPlain) m_row *= in;
            if (linear) m_row = fmaf(m_row, in, lean);
            // (capping keeps the order: the largest capped score is the capped
            // largest)
            if (kCapOnly && m_row != -INFINITY) m_row = capped(m_row, cap);
            // R(i) from R(i - 1), the other stream's, and this tile's maximum
            float prev = -INFINITY;
            if (i > 0) {
                ok = wait_warp(&tail->ref_full[odd ^ 1][sub], ((i - 1) >> 1) & 1, ST_TIMEOUT_SOFTMAX,
                               0x10000 | i);
                if (!ok) break;
                prev = tail->ref[odd ^ 1][row];
            }
            const float m_new = fmaxf(prev, m_row);
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
            const unsigned long long nm2 = both(nm);
            unsigned long long acc[2] = {both(0.0f), both(0.0f)};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t s[32];
                tmem_ld32(s_col + 32 * h, s);
                tmem_wait_ld();
                if (kCapOnly) cap32(s, cap, small);
                // (scores stored back in the first pass are masked already)
                if ((kPlain || kCapOnly || linear) && cut) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * h + e >= valid) s[e] = __float_as_uint(-INFINITY);
                }
                auto finish = [&](int e, unsigned long long x) {
                    float x0, x1;
                    f2unpack(x, x0, x1);
                    x0 = ex2(x0), x1 = ex2(x1);
                    acc[e & 1] = fadd2(acc[e & 1], f2pack(x0, x1));
                    s[e] = pack_f16x2(x0, x1);
                };
                auto pair = [&](int e) {
                    return f2pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
                };
                if (kPlain) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) finish(e, ffma2(pair(e), both(in), nm2));
                } else if (kBias == BIAS_INDEX && linear) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) finish(e, ffma2(pair(e), both(in), both(nm + lean)));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) finish(e, fadd2(pair(e), nm2));
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
            if (splits > 1) {
                // the ring is free here: the last PV is complete, so every copy
                // has landed and been read, and every zero behind the sequence's
                // end is written, which the arrivals release to the CTAs that
                // store over them
                __syncwarp();
                cluster_arrive_release();
                cluster_wait();
                // the row's O, maximum and sum into its owner's ring; its vectors
                // rotated, so that a warp's stores spread over the banks
                const int owner = ((row + 1) * splits - 1) / BM;
                const int slot = tail->split * part_rows + row - BM * owner / splits;
                const uint32_t to = dsmem_addr(smem_u32(sK) + slot * (HD * 4), owner);
                dsmem_st2(dsmem_addr(smem_u32(sV) + slot * 8, owner), top, sum);
#pragma unroll
                for (int h = 0; h < HD / 16; ++h) {
                    uint32_t a[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) a[k] = 0;
                    if (ok && n > 0) tmem_ld16(o_col + 16 * h, a);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        dsmem_st4u(to + 16 * ((4 * h + k) ^ (slot & 15)),
                                   make_uint4(a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3]));
                }
            } else {
                const float w = 1.0f / sum;
                const long long to = (q.begin + at) * p.out_row + head * HD;
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
                    if (ok && live) {
                        store8(p.out, to + 16 * h, p.out_dtype, v);
                        store8(p.out, to + 16 * h + 8, p.out_dtype, v + 8);
                    }
                }
            }
        }
    }
    if (splits > 1) {
        // The cluster's CTAs share out the tile's rows, and each has every
        // split's part of its own sent to it (stores into its shared memory,
        // which nobody waits for but the barrier): it adds them in rank order
        // (the same bits in every run) and no CTA reads another's memory.
        __syncwarp();
        if (warp < kSoftmaxWarp0 || warp >= kSoftmaxWarp0 + 4) {
            cluster_arrive_release();
            cluster_wait();
        }
        __syncwarp();
        cluster_sync();
        const int me = tail->split;
        const int r0 = BM * me / splits, r1 = min(BM * (me + 1) / splits, tail->rows);
        const long long to = (tail->span.begin + tail->q0) * p.out_row + head * HD;
        for (int i = threadIdx.x; i < (r1 - r0) * 16; i += kTileThreads) {
            const int r = i >> 4, k = i & 15;
            const float2* ml = reinterpret_cast<const float2*>(sV) + r;
            float top = -INFINITY;
            for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[s * part_rows].x);
            const float ref = top == -INFINITY ? 0.0f : top;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float sum = 0.0f;
            for (int s = 0; s < splits; ++s) {
                const int slot = s * part_rows + r;
                const float4 o = reinterpret_cast<const float4*>(sK)[slot * 16 + (k ^ (slot & 15))];
                const float w = ex2(ml[s * part_rows].x - ref);
                sum = fmaf(w, ml[s * part_rows].y, sum);
                a.x = fmaf(w, o.x, a.x), a.y = fmaf(w, o.y, a.y);
                a.z = fmaf(w, o.z, a.z), a.w = fmaf(w, o.w, a.w);
            }
            const float inv = 1.0f / sum;
            store4(p.out, to + (r0 + r) * p.out_row + 4 * k, p.out_dtype,
                   make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
        }
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
    if (a.cap > 0.0f && static_cast<double>(a.scale) > 1e6 * a.cap)  // the series' coefficients
        return fail(BL_ERR_UNSUPPORTED, "masked attention: cap below a millionth of the scale");
    // the constants that params_of makes of them
    const double unit = a.cap > 0.0f ? static_cast<double>(a.scale) / a.cap : 0.0;
    if (std::max({a.scale * 1.5, a.cap * 1.5, a.scale * std::pow(unit, 6) * 0.08}) >
        std::numeric_limits<float>::max())
        return fail(BL_ERR_UNSUPPORTED, "masked attention: scale %g, cap %g: constants leave 32 bits",
                    a.scale, a.cap);
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
    // Rows of K and V are read until the last CTA is done, so the output lies
    // apart from qkv's rows: in memory of its own or in columns of one wider row.
    // Q alone may be written over, by its own results in its own places: a CTA
    // (or the cluster that shares its keys) stores a row's after the last use of
    // its Q, which nobody else reads.
    const uintptr_t px = reinterpret_cast<uintptr_t>(a.qkv), po = reinterpret_cast<uintptr_t>(a.out);
    const uint64_t esz = dtype_size(a.out_dtype), xs = row * 2, os = orow * esz;
    if (px < po + (rows - 1) * os + ow * esz && po < px + (rows - 1) * xs + width * 2) {
        const uint64_t d = (px < po ? po - px : xs - (px - po) % xs) % xs;
        const bool over_q = px == po && esz == 2 && (xs == os || rows == 1);
        const bool columns = xs == os && d >= width * 2 && d + ow * esz <= xs;
        if (!over_q && !columns)
            return fail(BL_ERR_INVALID, "masked attention: out overlaps qkv");
    }
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
    if (a.cap > 0.0f) {
        const double unit = static_cast<double>(a.scale) / a.cap, v = unit * unit;
        const double log2e = 1.4426950408889634;
        const double c[4] = {1.0, -v / 3.0, v * v * (2.0 / 15.0), -v * v * v * (17.0 / 315.0)};
        for (int i = 0; i < 4; ++i) p.capping.c[i] = static_cast<float>(a.scale * log2e * c[i]);
        p.capping.unit = static_cast<float>(unit);
        p.capping.twice = static_cast<float>(2.0 * unit * log2e);
        p.capping.cap2 = static_cast<float>(a.cap * log2e);
    }
    p.qkv = static_cast<const uint16_t*>(a.qkv);
    p.row = static_cast<long long>(a.qkv_row_stride ? a.qkv_row_stride
                                                    : (1ull * a.heads + 2ull * kv) * HD);
    p.out = a.out, p.out_dtype = a.out_dtype;
    p.out_row = static_cast<long long>(a.out_row_stride ? a.out_row_stride : 1ull * a.heads * HD);
    p.offsets = a.offsets, p.lengths = a.lengths, p.prefix = a.prefix;
    p.slopes = a.slopes, p.pos = a.positions;
    p.pos_row = static_cast<long long>(a.pos_row_stride ? a.pos_row_stride : a.pos_axes);
    p.pos_axes = static_cast<int>(a.pos_axes);
    p.ragged = a.offsets != nullptr || a.lengths != nullptr;
    p.status = status_ptr();
    return p;
}

int prepare_rows(const bl_masked_attention_args& a, Launch* out) {
    Params p = params_of(a);
    const uint64_t combos = 1ull * p.last_rows * p.group;  // at most kMaxRows
    const uint64_t ctas = 1ull * a.batch * p.kv_heads;
    // Splits: as many as run at once (three CTAs an SM), each with 256 keys at
    // least; where that leaves three or fewer and the streams are long, about 768
    // CTAs, so that lengths that differ, and a wave that is not full, even out.
    // 16 streams of up to 8192 rows, 8 K/V heads: 2 splits 40.5 us, 3 35.9, 4
    // 30.4, 6 31.2, 8 35.7; of 8192 each: 45.8, 48.7, 54.7, 46.6, 49.6; of 2048
    // each: 14.1, 12.6, 16.7, 15.8, 18.9.
    uint64_t splits = std::min<uint64_t>({8, 3 * kSms / ctas, a.tokens / 256});
    if (3 * kSms / ctas <= 3 && a.tokens >= 4096) splits = std::max(splits, (768 + ctas / 2) / ctas);
    p.splits = static_cast<int>(a.key_splits ? a.key_splits : std::max<uint64_t>(1, splits));
    if (ctas * p.splits > 0x7FFFFFFFull)
        return fail(BL_ERR_UNSUPPORTED, "masked attention: grid too large");
    auto kern = a.qk_dtype == BL_BF16 ? rows_kernel<true> : rows_kernel<false>;
    const size_t smem = kRowRing + (p.splits > 1 ? p.splits * combos * kPartFloats * sizeof(float) : 0);
    BL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(kRowRing + 8 * kMaxRows * kPartFloats *
                                                                     sizeof(float))));
    const dim3 grid(static_cast<unsigned>(ctas * p.splits));
    out->op = BL_OP_MASKED_ATTENTION;
    out->run = [=](cudaStream_t s) {
        return p.splits > 1 ? launch_k_cluster(kern, grid, dim3(32 * kRowWarps),
                                               dim3(p.splits, 1, 1), smem, s, p)
                            : launch_k(kern, grid, dim3(32 * kRowWarps), smem, s, p);
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
    // Split the keys while that many CTAs still run at once (two an SM) and each
    // keeps 256 keys of an average sequence. Where a mask, or lengths that only
    // the device knows, make up to two waves of tiles unlike, the long ones alone
    // are split (ranked_tile): by two, or by four where that still runs at once
    // and the streams are long. 7 images up to 1370 rows, 6 heads: 24.9 -> 23.0 us
    // (all of them in halves 29.7); 1800, 1000 and 600 rows 31.9 -> 22.6; 5477
    // rows causal, 6 heads 71.4 -> 47.3 (in halves 46.5); 3 x 1370 causal 23.2 ->
    // 17.8, without a mask 26.2 -> 28.9, which the launch by clusters costs; 1370
    // newest rows of 5480 and 2000 45.7 -> 39.0 (in quarters 37.2). A long wave
    // of like tiles is split in halves (4096 keys: 5477 rows, 5 heads 81.4 ->
    // 63.2; 8 heads, 344 CTAs, 106.6 -> 97.9; 430 would lose).
    const uint64_t keys = a.offsets != nullptr ? a.tokens / a.batch : a.tokens;
    const uint64_t ctas = units * p.heads;
    uint64_t splits = std::max<uint64_t>(1, std::min<uint64_t>({8, 2 * kSms / ctas, keys / 256}));
    const bool unlike = p.mask != BL_MASK_NONE || (p.ragged && a.batch > 1);
    if (a.key_splits == 0 && unlike && a.batch <= 32 && splits <= 2 && ctas <= 600 && keys >= 512) {
        p.mixed = 1;
        splits = splits == 2 && keys >= 1536 ? 4 : 2;
    } else if (splits == 1 && ctas <= 370 && keys >= 4096) {
        splits = 2;
    }
    p.splits = static_cast<int>(a.key_splits ? a.key_splits : splits);
    if (units * p.heads * p.splits > 0x7FFFFFFFull)
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
    const dim3 grid(static_cast<unsigned>(units * p.heads * p.splits));
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
    // The last rows of a stream: while a K/V head's query rows are few, a
    // 128-row tile would be nearly empty and the keys' bytes are what counts.
    const uint32_t kv = a.kv_heads ? a.kv_heads : a.heads;
    const uint64_t combos = 1ull * std::min(a.last_rows, a.tokens) * (a.heads / kv);
    return a.last_rows > 0 && combos <= masked::kMaxRows ? masked::prepare_rows(a, out)
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
