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
    if (p.splits > 1) cluster_sync();  // no CTA leaves while its partials are read
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
    if (a.tokens > 0x7FFFFFFFu || a.batch > 0x7FFFFFFEu || rows > 0x7FFFFFFFull)
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

}  // namespace masked

int prepare_masked_attention(const bl_masked_attention_args& a, Launch* out) {
    const int rc = masked::validate(a);
    return rc != BL_OK ? rc : masked::prepare_rows(a, out);
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
