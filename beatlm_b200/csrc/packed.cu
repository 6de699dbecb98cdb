// The row maps of a packed batch (images and clips of different sizes one
// after the other in one token buffer) and rotary positions with several
// axes on its packed Q and K rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "host.h"

namespace bl {
namespace packed {

// ------------------------------------------------------------------ row maps

// Rows of image i: lead + t h w, 0 where a side is not positive, saturated
// above `cap` (any larger count fills the buffer all the same), so no product
// of three 32-bit sides overflows 64 bits.
__device__ __forceinline__ long long image_rows(const int* g, int lead, long long cap) {
    const long long t = g[0], h = g[1], w = g[2];
    if (t <= 0 || h <= 0 || w <= 0) return 0;
    const long long hw = min(h * w, cap + 1);
    return min(hw * t, cap + 1) + lead;
}

// offsets[i] = rows before image i, clamped to the capacity: one block scans
// the images in chunks of its size with a running total.
__global__ void __launch_bounds__(1024) pack_offsets_kernel(const int* grids, int images, int lead,
                                                            long long cap, int* offsets,
                                                            Status* status) {
    pdl_trigger();
    pdl_wait();
    __shared__ long long warp_sum[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long total = 0;
    if (threadIdx.x == 0) offsets[0] = 0;
    for (int base = 0; base < images; base += 1024) {
        const int i = base + threadIdx.x;
        long long v = i < images ? image_rows(grids + 3ll * i, lead, cap) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xFFFFFFFFu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) warp_sum[warp] = v;
        __syncthreads();
        long long before = total, all = total;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) before += warp_sum[w];
            all += warp_sum[w];
        }
        if (i < images) offsets[i + 1] = static_cast<int>(min(before + v, cap));
        total = all;
        __syncthreads();
    }
    if (threadIdx.x == 0 && total > cap) record_status(status, ST_BAD_ARGS, 0x9A);
}

// The last image of lo .. hi that starts at or before row r, offsets[lo] <= r
// (so images without rows are passed over): place `images` is behind the last.
__device__ __forceinline__ int image_of(const int* offsets, int lo, int hi, int r) {
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (offsets[mid] <= r) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// The same among all by a warp, for one row: 32 places at a time, so 1000
// images take two steps in place of ten.
__device__ __forceinline__ int image_of_warp(const int* offsets, int images, int r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = images;
    while (lo < hi) {
        const int step = (hi - lo) / 32 + 1;
        const bool before = lane == 0 || offsets[min(lo + step * lane, hi)] <= r;
        lo = min(lo + step * (31 - __clz(__ballot_sync(0xFFFFFFFFu, before))), hi);
        hi = min(lo + step - 1, hi);
    }
    return lo;
}

// (2 c + 1 - n) / n from x = 2 c + 1 - n: the correctly rounded quotient from
// the correctly rounded reciprocal (Markstein's correction step).
__device__ __forceinline__ float centre(float x, float n, float inverse) {
    const float q = x * inverse;
    return fmaf(fmaf(-q, n, x), inverse, q);
}
// u / n and its remainder for whole u in [0, 2^22) and n in [1, 2^22]: the whole
// number nearest to u times the reciprocal. The reciprocal's rounding moves u / n
// by at most 2^22 2^-24 / n, so that number is within 1/2 + 1/(4 n) of it: the
// quotient, or one more where the remainder (exact) comes out negative.
__device__ __forceinline__ float divide(float u, float n, float inverse, float& rest) {
    const float magic = 12582912.0f;  // 1.5 2^23: the sum is a whole number
    float q = fmaf(u, inverse, magic) - magic;
    rest = fmaf(-q, n, u);
    if (rest < 0.0f) q -= 1.0f, rest += n;
    return q;
}

// Row r of any image, or behind the last: one by one.
__device__ __forceinline__ void write_row(const int* grids, const int* offsets, int images,
                                          int lead, bool normalized, int at, int r, int* image,
                                          float* pos) {
    if (image != nullptr) image[r] = at < images ? at : -1;
    if (pos == nullptr) return;
    float v[3] = {0.0f, 0.0f, 0.0f};
    const int p = at < images ? r - offsets[at] - lead : -1;
    if (p >= 0) {
        const int* g = grids + 3ll * at;
        const unsigned w = g[2], h = g[1], row = static_cast<unsigned>(p) / w, outer = row / h;
        const int c[3] = {static_cast<int>(outer), static_cast<int>(row - outer * h),
                          static_cast<int>(p - row * w)};
#pragma unroll
        for (int a = 0; a < 3; ++a) {
            const float n = static_cast<float>(g[a]);
            v[a] = normalized ? centre(static_cast<float>(c[a] - (g[a] - 1 - c[a])), n, 1.0f / n)
                              : static_cast<float>(c[a]);
        }
    }
#pragma unroll
    for (int a = 0; a < 3; ++a) pos[3ll * r + a] = v[a];
}

// Rows 4 k .. 4 k + 3 for k = first, first + step, ..: a warp searches the image
// of its first row, a thread goes on from there. Where its four rows are patches
// of one image (and the counts exact in 24 bits) it divides the first one's
// place out with the image's reciprocals and steps it, all in f32, and its
// positions leave as three 16-byte stores. The other groups of four are shared
// out over the warp's lanes, a row each, so that a warp that meets an image's
// end loses one search and one division, not four. (The instructions are what
// bounds it: with integer places, converted a row and axis, a million rows of a
// thousand images took 11.5 us; now 9.6, of which a fill of the maps is 3.1.)
__device__ __forceinline__ void write_rows(const int* grids, const int* offsets, int images,
                                           int lead, bool normalized, int cap, int* image,
                                           float* pos, bool vec, int first, int step) {
    __shared__ int2 left[256];
    const int groups = cap / 4 + (cap % 4 != 0), lane = threadIdx.x & 31;
    int2* rest = left + (threadIdx.x & ~31);
    // the image of row r, at or behind image `at`: mostly the next
    auto advance = [&](int at, int r) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (at < images && r >= offsets[at + 1]) ++at;
        return at < images && r >= offsets[at + 1] ? image_of(offsets, at + 1, images, r) : at;
    };
    for (int k0 = first - lane; k0 < groups; k0 += step) {
        const int k = min(k0 + lane, groups - 1), r = 4 * k;
        const int at = advance(image_of_warp(offsets, images, 4 * k0), r);
        constexpr int kExact = 1 << 22;
        const int p = at < images ? r - offsets[at] - lead : -1;
        int g0 = kExact, g1 = 0, g2 = 0;
        if (vec && static_cast<unsigned>(p) < kExact - 4u && r + 4 <= offsets[at + 1])
            g0 = grids[3ll * at], g1 = grids[3ll * at + 1], g2 = grids[3ll * at + 2];
        const bool alone = (g0 | g1 | g2) >= kExact;
        const unsigned others = __ballot_sync(0xFFFFFFFFu, alone);
        if (!alone) {
            if (image != nullptr) reinterpret_cast<int4*>(image)[k] = make_int4(at, at, at, at);
            if (pos != nullptr) {
                const float n0 = g0, n1 = g1, n2 = g2;
                const float i0 = 1.0f / n0, i1 = 1.0f / n1, i2 = 1.0f / n2;
                float c0, c1, c2, out[12];
                c0 = divide(divide(static_cast<float>(p), n2, i2, c2), n1, i1, c1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    out[3 * i] = normalized ? centre(fmaf(2.0f, c0, 1.0f - n0), n0, i0) : c0;
                    out[3 * i + 1] = normalized ? centre(fmaf(2.0f, c1, 1.0f - n1), n1, i1) : c1;
                    out[3 * i + 2] = normalized ? centre(fmaf(2.0f, c2, 1.0f - n2), n2, i2) : c2;
                    c2 += 1.0f;
                    if (c2 == n2) c2 = 0.0f, c1 += 1.0f;
                    if (c1 == n1) c1 = 0.0f, c0 += 1.0f;
                }
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    reinterpret_cast<float4*>(pos)[3ll * k + e] =
                        make_float4(out[4 * e], out[4 * e + 1], out[4 * e + 2], out[4 * e + 3]);
            }
        }
        if (others != 0) {
            const int count = __popc(others);
            if (alone) rest[__popc(others & ((1u << lane) - 1))] = make_int2(r, at);
            __syncwarp();
            for (int i = lane; i < 4 * count; i += 32) {
                const int row = rest[i >> 2].x + (i & 3);
                if (row < cap)
                    write_row(grids, offsets, images, lead, normalized,
                              advance(rest[i >> 2].y, row), row, image, pos);
            }
            __syncwarp();
        }
    }
}

__global__ void __launch_bounds__(256) pack_rows_kernel(const int* grids, const int* offsets,
                                                        int images, int lead, int normalized,
                                                        int cap, int* image, float* pos, int vec) {
    pdl_trigger();
    pdl_wait();
    write_rows(grids, offsets, images, lead, normalized != 0, cap, image, pos, vec != 0,
               static_cast<int>(blockIdx.x) * 256 + threadIdx.x, gridDim.x * 256);
}

// All of it in one launch for up to kPackImages images: every block copies the
// sizes into its own shared memory and scans them there (12 KB of reads from L2
// a thousand images, 2 us, cheaper than a second launch and its wait) and writes
// its rows; block 0 writes the offsets. Eight images, 2802 rows: 3.4 us.
constexpr int kPackImages = 4096;
__global__ void __launch_bounds__(256) pack_kernel(const int* grids, int images, int lead,
                                                   int normalized, int cap, int* offsets,
                                                   int* image, float* pos, int vec,
                                                   Status* status) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ int sizes[];  // [images][3], then the offsets
    int* at = sizes + 3 * images;
    __shared__ long long warp_sum[8];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
#pragma unroll 4
    for (int i = t; i < 3 * images; i += 256) sizes[i] = grids[i];
    __syncthreads();
    // a thread sums neighbours, then leaves what is before each in its place
    const int each = (images + 255) / 256, first = min(t * each, images);
    const int last = min(first + each, images);
    long long mine = 0;
    for (int i = first; i < last; ++i) {
        at[i] = static_cast<int>(min(image_rows(sizes + 3 * i, lead, cap), cap + 1ll));
        mine += at[i];
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += u;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    long long before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        if (w < warp) before += warp_sum[w];
        total += warp_sum[w];
    }
    for (int i = first; i < last; ++i) {
        const int rows = at[i];
        at[i] = static_cast<int>(min(before, static_cast<long long>(cap)));
        before += rows;
    }
    if (t == 0) at[images] = static_cast<int>(min(total, static_cast<long long>(cap)));
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int i = t; i <= images; i += 256) offsets[i] = at[i];
        if (t == 0 && total > cap) record_status(status, ST_BAD_ARGS, 0x9A);
    }
    if (image != nullptr || pos != nullptr)
        write_rows(sizes, at, images, lead, normalized != 0, cap, image, pos, vec != 0,
                   static_cast<int>(blockIdx.x) * 256 + t, gridDim.x * 256);
}

// ------------------------------------------------------------------ rotary

struct RopeParams {
    long long rows;
    int heads, head_dim, pairs;
    int sections[3];  // pairs of each axis, 0 past the last
    int inverse;
    const void* x;
    long long x_stride;
    void* out;
    long long out_stride;
    const float* pos;
    long long pos_stride;
    // the block's shape: chunks of a head's pairs, head groups, rows, and the
    // heads a thread turns one after the other
    int chunks, groups, tile_rows, per_thread;
    double turn[BL_ROPE_MAX_PAIRS];  // frequency / pi: angles in half turns
};

template <typename T> __device__ __forceinline__ float up(T v);
template <> __device__ __forceinline__ float up(float v) { return v; }
template <> __device__ __forceinline__ float up(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T down(float v);
template <> __device__ __forceinline__ float down(float v) { return v; }
template <> __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Vec {
    T v[kVec];
};

// Values 2 w and 2 w + 1 of a vector, and back: 16-bit types by the word.
template <typename T, int kVec>
__device__ __forceinline__ float2 get2(const Vec<T, kVec>& x, int w) {
    if constexpr (sizeof(T) == 4) {
        return make_float2(x.v[2 * w], x.v[2 * w + 1]);
    } else {
        const uint32_t word = reinterpret_cast<const uint32_t*>(&x)[w];
        if constexpr (std::is_same<T, __nv_bfloat16>::value)
            return make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xFFFF0000u));
        else
            return __half22float2(*reinterpret_cast<const __half2*>(&word));
    }
}
template <typename T, int kVec>
__device__ __forceinline__ void put2(Vec<T, kVec>& x, int w, float lo, float hi) {
    if constexpr (sizeof(T) == 4) {
        x.v[2 * w] = lo, x.v[2 * w + 1] = hi;
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        reinterpret_cast<uint32_t*>(&x)[w] = pack_bf16x2(lo, hi);
    } else {
        reinterpret_cast<uint32_t*>(&x)[w] = pack_f16x2(lo, hi);
    }
}
// The kVec pairs that the vectors a and b of one head hold, turned in place.
template <typename T, int kVec, bool kAdjacent>
__device__ __forceinline__ void turn_pairs(Vec<T, kVec>& a, Vec<T, kVec>& b, const float (&c)[kVec],
                                           const float (&s)[kVec]) {
    if constexpr (kVec == 1) {
        const float f = up(a.v[0]), g = up(b.v[0]);
        a.v[0] = down<T>(f * c[0] - g * s[0]);
        b.v[0] = down<T>(g * c[0] + f * s[0]);
    } else if constexpr (kAdjacent) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            Vec<T, kVec>& x = 2 * e < kVec ? a : b;
            const int w = e % (kVec / 2);
            const float2 f = get2(x, w);
            put2(x, w, f.x * c[e] - f.y * s[e], f.y * c[e] + f.x * s[e]);
        }
    } else {
#pragma unroll
        for (int w = 0; w < kVec / 2; ++w) {
            const float2 f = get2(a, w), g = get2(b, w);
            const float c0 = c[2 * w], c1 = c[2 * w + 1], s0 = s[2 * w], s1 = s[2 * w + 1];
            put2(a, w, f.x * c0 - g.x * s0, f.y * c1 - g.y * s1);
            put2(b, w, g.x * c0 + f.x * s0, g.y * c1 + f.y * s1);
        }
    }
}

// A block turns tiles of rows, each thread kVec neighbouring pairs of several
// heads: two vectors of a head (its halves, an axis's halves, or neighbours),
// so every global access is a whole vector and a warp's cover whole sectors.
// What bounds it is memory: each value read once and written once. The angles
// are few beside the values (one a row and pair, against one pair a head), but
// dear: formed in 64 bits in half turns and reduced to [-1, 1] before the
// 32-bit sincospif, whose results are corrected for the rounding of its argument,
// so that positions of 10^6 and more lose nothing the result could hold. A tile's cosines and sines are made once, into one of two shared
// tables (so one barrier a tile is enough), while the tile's values are on
// their way; a thread keeps the frequency of its pair over all its tiles.
// 60280 rows x 32 heads x 64 in bf16 (494 MB): 75.9 us, the rate of a copy.
// (With one head in flight a thread 95.5 us; with four, whose registers leave
// half as many blocks an SM, 82.1.)
constexpr int kRopeBatch = 2;  // heads a thread has in flight

template <typename T, int kVec, int kPairing>
__global__ void __launch_bounds__(256) rope_kernel(const __grid_constant__ RopeParams p) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ float table[];  // [2][tile_rows][2][pairs]
    using V = Vec<T, kVec>;
    const int t = threadIdx.x;
    // as a maker of angles: pair t % pairs of every step-th row
    const int step = 256 / p.pairs, pair = t % p.pairs, first_row = t / p.pairs;
    const int axis = pair < p.sections[0] ? 0 : pair < p.sections[0] + p.sections[1] ? 1 : 2;
    const double turn = p.turn[pair];
    // as a turner of pairs: chunk, head group, row of the tile
    const int chunk = t % p.chunks, group = t / p.chunks % p.groups;
    const int row = t / (p.chunks * p.groups);
    const int j = chunk * kVec;
    int lo, hi;
    if (kPairing == BL_ROPE_HALF) {
        lo = j, hi = j + p.pairs;
    } else if (kPairing == BL_ROPE_ADJACENT) {
        lo = 2 * j, hi = lo + kVec;
    } else {
        const int s0 = p.sections[0], s1 = s0 + p.sections[1];
        const int start = j < s0 ? 0 : j < s1 ? s0 : s1;
        lo = start + j, hi = lo + (j < s0 ? s0 : j < s1 ? s1 - s0 : p.sections[2]);
    }
    const int table_size = 2 * p.tile_rows * p.pairs;
    const long long tiles = (p.rows + p.tile_rows - 1) / p.tile_rows;
    int buffer = 0;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x, buffer ^= 1) {
        const long long r0 = tile * p.tile_rows;
        const long long r = r0 + row;
        const bool mine = row < p.tile_rows && r < p.rows;
        const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
        T* y = static_cast<T*>(p.out) + r * p.out_stride;
        V a[kRopeBatch], b[kRopeBatch];
        auto load = [&](int base) {
#pragma unroll
            for (int i = 0; i < kRopeBatch; ++i) {
                const int head = group + (base + i) * p.groups;
                if (mine && base + i < p.per_thread && head < p.heads) {
                    a[i] = *reinterpret_cast<const V*>(x + head * p.head_dim + lo);
                    b[i] = *reinterpret_cast<const V*>(x + head * p.head_dim + hi);
                }
            }
        };
        load(0);
        float* cs = table + buffer * table_size;
        for (int k = first_row; k < p.tile_rows && first_row < step; k += step) {
            if (r0 + k >= p.rows) break;
            double h = static_cast<double>(p.pos[(r0 + k) * p.pos_stride + axis]) * turn;
            h -= 2.0 * rint(0.5 * h);
            // the 32-bit angle's functions, turned on by what it left out (below
            // 10^-7 radians, so to first order)
            const float near = static_cast<float>(h);
            const float rest = static_cast<float>((h - near) * 3.14159265358979323846);
            float sn, cn;
            sincospif(near, &sn, &cn);
            const float sine = fmaf(cn, rest, sn);
            cs[2 * k * p.pairs + pair] = fmaf(-sn, rest, cn);
            cs[(2 * k + 1) * p.pairs + pair] = p.inverse ? -sine : sine;
        }
        __syncthreads();
        if (mine) {
            float c[kVec], s[kVec];
            const float* at = cs + 2 * row * p.pairs + j;
#pragma unroll
            for (int e = 0; e < kVec; ++e) c[e] = at[e], s[e] = at[p.pairs + e];
            for (int base = 0; base < p.per_thread; base += kRopeBatch) {
                if (base > 0) load(base);
#pragma unroll
                for (int i = 0; i < kRopeBatch; ++i) {
                    const int head = group + (base + i) * p.groups;
                    if (base + i >= p.per_thread || head >= p.heads) continue;
                    turn_pairs<T, kVec, kPairing == BL_ROPE_ADJACENT>(a[i], b[i], c, s);
                    *reinterpret_cast<V*>(y + head * p.head_dim + lo) = a[i];
                    *reinterpret_cast<V*>(y + head * p.head_dim + hi) = b[i];
                }
            }
        }
        const int rest = p.head_dim - 2 * p.pairs;  // values that do not turn
        if (rest > 0 && p.x != p.out) {
            const int per_row = p.heads * rest;
            const int n = static_cast<int>(min(static_cast<long long>(p.tile_rows), p.rows - r0));
            for (int k = 0; k < n; ++k) {
                const T* from = static_cast<const T*>(p.x) + (r0 + k) * p.x_stride;
                T* to = static_cast<T*>(p.out) + (r0 + k) * p.out_stride;
                for (int i = t; i < per_row; i += 256) {
                    const int e = i / rest * p.head_dim + 2 * p.pairs + i % rest;
                    to[e] = from[e];
                }
            }
        }
    }
}

using RopeKernel = void (*)(const RopeParams);
template <typename T, int kVec>
RopeKernel rope_of(int pairing) {
    return pairing == BL_ROPE_HALF       ? rope_kernel<T, kVec, BL_ROPE_HALF>
           : pairing == BL_ROPE_ADJACENT ? rope_kernel<T, kVec, BL_ROPE_ADJACENT>
                                         : rope_kernel<T, kVec, BL_ROPE_AXIS_HALF>;
}
template <typename T>
RopeKernel rope_of(int pairing, int vec) {
    if constexpr (sizeof(T) == 2)
        if (vec == 8) return rope_of<T, 8>(pairing);
    return vec == 4 ? rope_of<T, 4>(pairing) : vec == 2 ? rope_of<T, 2>(pairing) : rope_of<T, 1>(pairing);
}

}  // namespace packed

int prepare_pack(const bl_pack_args& a, Launch* out) {
    if (a.images == 0 || a.capacity == 0)
        return fail(BL_ERR_INVALID, "pack: no images or no rows");
    if (a.images > 0x7FFFFFFEu || a.capacity > 0x7FFFFFF0u || a.lead > 0x7FFFFFFFu)
        return fail(BL_ERR_UNSUPPORTED, "pack: %u images, %u rows, %u lead rows exceed 32-bit rows",
                    a.images, a.capacity, a.lead);
    if (a.grids == nullptr || a.offsets == nullptr)
        return fail(BL_ERR_INVALID, "pack: null grids or offsets");
    for (const void* q : {static_cast<const void*>(a.grids), static_cast<const void*>(a.offsets),
                          static_cast<const void*>(a.image), static_cast<const void*>(a.positions)})
        if (reinterpret_cast<uintptr_t>(q) & 3u)
            return fail(BL_ERR_INVALID, "pack: a buffer is not 4-byte aligned");
    Status* st = status_ptr();
    const bl_pack_args b = a;
    const int vec = ((reinterpret_cast<uintptr_t>(a.image) | reinterpret_cast<uintptr_t>(a.positions)) & 15u) == 0;
    BL_CUDA_TRY(cudaFuncSetAttribute(packed::pack_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (4 * packed::kPackImages + 1) * sizeof(int)));
    out->op = BL_OP_PACK;
    out->run = [=](cudaStream_t s) {
        const int n = static_cast<int>(b.images), lead = static_cast<int>(b.lead);
        const int cap = static_cast<int>(b.capacity), norm = b.normalized != 0;
        const bool maps = b.image != nullptr || b.positions != nullptr;
        // one thread a group of four rows, at most two blocks an SM (each scans
        // all sizes again: four blocks 9.9 us where two take 9.6)
        const unsigned blocks = static_cast<unsigned>(
            maps ? std::min<uint64_t>((cap + 1023ull) / 1024, 148 * 2) : 1);
        if (n <= packed::kPackImages)
            return launch_k(packed::pack_kernel, dim3(blocks), dim3(256),
                            (4ull * n + 1) * sizeof(int), s, b.grids, n, lead, norm, cap, b.offsets,
                            b.image, b.positions, vec, st);
        cudaError_t e = launch_k(packed::pack_offsets_kernel, dim3(1), dim3(1024), 0, s, b.grids, n,
                                 lead, static_cast<long long>(cap), b.offsets, st);
        if (e != cudaSuccess || !maps) return e;
        return launch_k(packed::pack_rows_kernel, dim3(blocks), dim3(256), 0, s, b.grids, b.offsets,
                        n, lead, norm, cap, b.image, b.positions, vec);
    };
    return BL_OK;
}

namespace {

// Bytes from the first to one past the last element of rows x width values.
uint64_t span_bytes(uint64_t rows, uint64_t stride, uint64_t width, uint64_t esz) {
    return ((rows - 1) * stride + width) * esz;
}

}  // namespace

int prepare_rope(const bl_rope_args& a, Launch* out) {
    using packed::RopeParams;
    if (a.rows == 0 || a.heads == 0 || a.head_dim == 0)
        return fail(BL_ERR_INVALID, "rope: zero dimension");
    if (a.axes < 1 || a.axes > 3) return fail(BL_ERR_INVALID, "rope: %u axes (1 to 3)", a.axes);
    uint64_t pairs = 0;
    for (uint32_t i = 0; i < a.axes; ++i) {
        if (a.sections[i] == 0) return fail(BL_ERR_INVALID, "rope: axis %u has no pairs", i);
        pairs += a.sections[i];
    }
    if (2 * pairs > a.head_dim)
        return fail(BL_ERR_INVALID, "rope: %llu pairs in a head of %u", (unsigned long long)pairs,
                    a.head_dim);
    if (pairs > BL_ROPE_MAX_PAIRS)
        return fail(BL_ERR_UNSUPPORTED, "rope: %llu pairs (at most %d)", (unsigned long long)pairs,
                    (int)BL_ROPE_MAX_PAIRS);
    if (a.pairing < BL_ROPE_HALF || a.pairing > BL_ROPE_AXIS_HALF)
        return fail(BL_ERR_INVALID, "rope: pairing %d", a.pairing);
    if (a.dtype != BL_F32 && a.dtype != BL_F16 && a.dtype != BL_BF16)
        return fail(BL_ERR_INVALID, "rope: dtype %d", a.dtype);
    if (a.freqs == nullptr && !(a.theta > 0.0 && std::isfinite(a.theta)))
        return fail(BL_ERR_INVALID, "rope: theta must be finite and positive");
    if (a.x == nullptr || a.out == nullptr || a.positions == nullptr)
        return fail(BL_ERR_INVALID, "rope: null pointer");
    const uint64_t esz = dtype_size(a.dtype), width = 1ull * a.heads * a.head_dim;
    const uint64_t xs = a.x_row_stride ? a.x_row_stride : width;
    const uint64_t os = a.out_row_stride ? a.out_row_stride : width;
    const uint64_t ps = a.pos_row_stride ? a.pos_row_stride : a.axes;
    if (width > 0x7FFFFFFFu || xs >= (1ull << 40) || os >= (1ull << 40) || ps >= (1ull << 40))
        return fail(BL_ERR_UNSUPPORTED, "rope: rows of %llu values", (unsigned long long)width);
    if (a.rows > 0x7FFFFFFFu) return fail(BL_ERR_UNSUPPORTED, "rope: %u rows", a.rows);
    if (xs < width || os < width || ps < a.axes)
        return fail(BL_ERR_INVALID, "rope: a row stride is shorter than its row");
    const uintptr_t px = reinterpret_cast<uintptr_t>(a.x), po = reinterpret_cast<uintptr_t>(a.out);
    if (px % esz || po % esz || (reinterpret_cast<uintptr_t>(a.positions) & 3u))
        return fail(BL_ERR_INVALID, "rope: a buffer is not aligned to its type");
    // In place, or apart: rows that overlap otherwise would be read after
    // they are written. Columns of one wider row set apart are apart.
    if (px == po) {
        if (xs != os && a.rows > 1)
            return fail(BL_ERR_INVALID, "rope: in place with two row strides");
    } else if (px < po + span_bytes(a.rows, os, width, esz) &&
               po < px + span_bytes(a.rows, xs, width, esz)) {
        const uint64_t d = (px < po ? po - px : px - po) % (xs * esz);
        if (xs != os || d < width * esz || d + width * esz > xs * esz)
            return fail(BL_ERR_INVALID, "rope: x and out overlap without being the same");
    }
    RopeParams p{};
    p.rows = a.rows, p.heads = static_cast<int>(a.heads), p.head_dim = static_cast<int>(a.head_dim);
    p.pairs = static_cast<int>(pairs), p.inverse = a.inverse != 0;
    for (uint32_t i = 0; i < a.axes; ++i) p.sections[i] = static_cast<int>(a.sections[i]);
    p.x = a.x, p.x_stride = static_cast<long long>(xs);
    p.out = a.out, p.out_stride = static_cast<long long>(os);
    p.pos = a.positions, p.pos_stride = static_cast<long long>(ps);
    int j = 0;
    const double log_theta = a.freqs == nullptr ? std::log(a.theta) : 0.0;
    for (uint32_t i = 0; i < a.axes; ++i)
        for (uint32_t k = 0; k < a.sections[i]; ++k, ++j) {
            const double f = a.freqs != nullptr ? a.freqs[j]
                             : std::exp(-log_theta * (a.shared_ladder
                                                          ? static_cast<double>(j) / static_cast<double>(pairs)
                                                          : static_cast<double>(k) / a.sections[i]));
            if (!std::isfinite(f)) return fail(BL_ERR_INVALID, "rope: frequency %d is not finite", j);
            p.turn[j] = f / 3.14159265358979323846;
        }
    // The widest vectors (at most 16 bytes) that every chunk of pairs, head,
    // row and base starts on a multiple of: a power of two that divides them
    // all. 60280 rows x 32 heads x 64 in bf16 take 75.9 us by 16-byte vectors,
    // 98.8 by 8-byte and 144 by 4-byte ones.
    int vec = static_cast<int>(16 / esz);
    auto divides = [&](int v) {
        bool ok = pairs % v == 0 && a.head_dim % v == 0 && xs % v == 0 && os % v == 0 &&
                  px % (v * esz) == 0 && po % (v * esz) == 0;
        if (a.pairing == BL_ROPE_AXIS_HALF)
            for (uint32_t i = 0; i < a.axes; ++i) ok = ok && a.sections[i] % v == 0;
        return ok;
    };
    while (vec > 1 && !divides(vec)) vec /= 2;
    p.chunks = p.pairs / vec;
    // Heads a thread turns: one where a block then has one tile of rows at most
    // (the shortest way through), else kRopeBatch, so that a tile's barrier and
    // its loads' way are paid half as often. 5477 rows x 16 heads x 80 in f32:
    // 13.0 us with one, 9.7 with two.
    const unsigned most_blocks = 148 * 8;
    uint64_t tiles = 0;
    for (int want = 1; want <= packed::kRopeBatch; want *= 2) {
        p.groups = std::max(1, std::min((p.heads + want - 1) / want, 256 / p.chunks));
        p.per_thread = (p.heads + p.groups - 1) / p.groups;
        p.tile_rows = std::max(1, 256 / (p.chunks * p.groups));
        tiles = (a.rows + p.tile_rows - 1ull) / p.tile_rows;
        if (tiles <= most_blocks) break;
    }
    const size_t smem = 4ull * p.tile_rows * p.pairs * sizeof(float);
    const unsigned blocks = static_cast<unsigned>(std::min<uint64_t>(tiles, most_blocks));
    const packed::RopeKernel kern = a.dtype == BL_F32   ? packed::rope_of<float>(a.pairing, vec)
                                    : a.dtype == BL_F16 ? packed::rope_of<__half>(a.pairing, vec)
                                                        : packed::rope_of<__nv_bfloat16>(a.pairing, vec);
    out->op = BL_OP_ROPE;
    out->run = [=](cudaStream_t s) { return launch_k(kern, dim3(blocks), dim3(256), smem, s, p); };
    return BL_OK;
}

}  // namespace bl

extern "C" int bl_pack(const bl_pack_args* args, void* stream) {
    if (args == nullptr) return bl::fail(BL_ERR_INVALID, "pack: null args");
    return bl::guarded("pack", [&] {
        bl::Launch l;
        const int rc = bl::prepare_pack(*args, &l);
        return rc != BL_OK ? rc : bl::enqueue(l, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int bl_rope(const bl_rope_args* args, void* stream) {
    if (args == nullptr) return bl::fail(BL_ERR_INVALID, "rope: null args");
    return bl::guarded("rope", [&] {
        bl::Launch l;
        const int rc = bl::prepare_rope(*args, &l);
        return rc != BL_OK ? rc : bl::enqueue(l, static_cast<cudaStream_t>(stream));
    });
}
