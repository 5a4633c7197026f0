// Rotary positions with several axes (time, height, width, ...): pair i of every head turns by the angle
// positions[axis_i][row] * freq_i,
//   y_a = x_a cos - x_b sin,  y_b = x_b cos + x_a sin,
// with (a, b) = (i, i + pairs) or (2 i, 2 i + 1). The inverse rotation (-angle) is its gradient.
//
// Bound: HBM (each element read once and written once, 6 flops a pair). The angle is taken in 64 bits and only
// its fraction of a turn goes on in 32, so a position of 10^6 keeps its angle; products and the sum are fp32,
// one rounding to bf16 at the end. v_sin_f32 / v_cos_f32 take the angle in turns as it is, off by
// less than 2^-19: a result of nearly 0 is off by that share of its pair, not of itself.
#include "common.h"

namespace {

struct RopeArgs {
    const bf16* x;
    bf16* y;
    const int32_t* pos;
    const double* freqs;
    const int32_t* axes;
    long ldx, ldy, ldp;
    int rows, nheads, hd, pairs, naxes, R;
    float sign;
};

typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_a4 __attribute__((aligned(4)));

__device__ __forceinline__ float2 turn(const RopeArgs& a, int row, int i) {  // (cosine, sine) of pair i of a row
    const int ax = min(max(a.axes[i], 0), a.naxes - 1);
    const double t = (double)a.pos[ax * a.ldp + row] * a.freqs[i] * 0.15915494309189535;
    const float f = (float)(t - __builtin_rint(t));
    return make_float2(__builtin_amdgcn_cosf(f), __builtin_amdgcn_sinf(f) * a.sign);
}
__device__ __forceinline__ float lo(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi(unsigned w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ unsigned pack(float p, float q) {
    return (unsigned)__builtin_bit_cast(unsigned short, f2bf(p)) | (unsigned)__builtin_bit_cast(unsigned short, f2bf(q)) << 16;
}

// One workgroup: R rows through all heads. The rows' cosines and sines go to LDS once (64-bit arithmetic is not
// repeated per head); then threads take the rows' 16-byte chunks in the order they lie in memory, so that stores
// fill whole lines whatever the head dim. A chunk is two groups of four elements; with halves a group's partners are
// a group elsewhere in the head, read again through the cache. U chunks a thread are in flight.
// NT: stores that pass the L2 by: 13.2 against 14.8 us for 31 MB (10 007 rows of 24 heads of 64), as long as a wave
// fills whole lines (without that they took twice as long). Outputs under 16 MB stay in the L2 for the attention.
// Measured: 44 640 rows of 32 heads of 72 (412 MB in and out) 74.9 us, 5.5 TB/s; a large copy reaches 5.2 TB/s.
template <bool ADJ, bool NT>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2 cs[];
    constexpr int U = 2;
    const int tid = threadIdx.x;
    const int row0 = blockIdx.x * a.R, R = min(a.R, a.rows - row0);
    for (int i = tid; i < R * a.pairs; i += 256) {
        const int r = i / a.pairs;
        cs[i] = turn(a, row0 + r, i - r * a.pairs);
    }
    __syncthreads();
    const bf16* x = a.x + (long)row0 * a.ldx;
    bf16* y = a.y + (long)row0 * a.ldy;
    const int C = a.hd >> 3, W = a.nheads * C, n = R * W;
    for (int i0 = tid; i0 < n; i0 += 256 * U) {
        u32x4 own[U];
        u32x2 other[U][2];
        int row[U], at[U];  // the chunk's row, and where it begins in its head
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(i0 + 256 * u, n - 1);
            row[u] = i / W;
            const int ch = i - row[u] * W, h = ch / C;
            at[u] = (ch - h * C) * 8;
            const bf16* xr = x + row[u] * a.ldx;
            own[u] = *reinterpret_cast<const u32x4_a4*>(xr + ch * 8);
            if (!ADJ)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int e = at[u] + 4 * g, p = e < a.pairs ? e + a.pairs : e < 2 * a.pairs ? e - a.pairs : e;
                    other[u][g] = *reinterpret_cast<const u32x2_a4*>(xr + ch * 8 + 4 * g + (p - e));
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u;
            u32x4 out;
            const float2* t = cs + row[u] * a.pairs;
            if (ADJ) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int pair = (at[u] >> 1) + w;
                    const float2 c = t[min(pair, a.pairs - 1)];
                    const float p = lo(own[u][w]), q = hi(own[u][w]);
                    out[w] = pair < a.pairs ? pack(p * c.x - q * c.y, q * c.x + p * c.y) : own[u][w];
                }
            } else {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int e = at[u] + 4 * g;
                    const bool first = e < a.pairs, turns = e < 2 * a.pairs;
                    const float2* tg = t + (first ? e : turns ? e - a.pairs : 0);
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const unsigned o = own[u][2 * g + w], v = other[u][g][w];
                        const float2 c0 = tg[2 * w], c1 = tg[2 * w + 1];
                        const float s0 = first ? -c0.y : c0.y, s1 = first ? -c1.y : c1.y;
                        out[2 * g + w] = turns ? pack(lo(o) * c0.x + lo(v) * s0, hi(o) * c1.x + hi(v) * s1) : o;
                    }
                }
            }
            if (i < n) {
                u32x4_a4* to = reinterpret_cast<u32x4_a4*>(y + row[u] * a.ldy + (long)(i - row[u] * W) * 8);
                if (NT)
                    __builtin_nontemporal_store(out, to);
                else
                    *to = out;
            }
        }
    }
}

// Halves again, a thread taking V elements of a head and their partners, and writing both: in place, where a chunk's
// partners would be another thread's; and where a half is whole lines, which need no second read (16 480 rows of 9
// heads of 256, 152 MB: 25.2 us, 6.0 TB/s, against 40.5 us chunk by chunk; heads of 64 the other way, 20.5 against 23.9).
// In place / out of place: 10 007 rows of 24 heads of 64 11.2 / 12.1 us, 44 640 of 32 of 72 87 / 77, 20 001 of 9 of 128
// 16.9 / 17.3, 16 480 of 9 of 256 25.1 / 24.9.
template <int V, bool NT>
__global__ __launch_bounds__(256) void rope_axes_halves_kernel(RopeArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2 cs[];
    typedef unsigned vec __attribute__((ext_vector_type(V / 2)));
    typedef vec vec_a4 __attribute__((aligned(4)));
    constexpr int U = 2;
    const int tid = threadIdx.x;
    const int row0 = blockIdx.x * a.R, R = min(a.R, a.rows - row0);
    for (int i = tid; i < R * a.pairs; i += 256) {
        const int r = i / a.pairs;
        cs[i] = turn(a, row0 + r, i - r * a.pairs);
    }
    __syncthreads();
    const bf16* x = a.x + (long)row0 * a.ldx;
    bf16* y = a.y + (long)row0 * a.ldy;
    if (a.x != a.y) {  // what does not turn
        const int C = (a.hd - 2 * a.pairs) >> 2, W = a.nheads * C;
        for (int i = tid; i < R * W; i += 256) {
            const int row = i / W, ch = i - row * W, h = ch / C;
            const long at = (long)h * a.hd + 2 * a.pairs + (ch - h * C) * 4;
            *reinterpret_cast<u32x2_a4*>(y + row * a.ldy + at) = *reinterpret_cast<const u32x2_a4*>(x + row * a.ldx + at);
        }
    }
    const int C = a.pairs / V, W = a.nheads * C, n = R * W;
    for (int i0 = tid; i0 < n; i0 += 256 * U) {
        vec p[U], q[U];
        int e[U], t[U];
        long at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(i0 + 256 * u, n - 1);
            const int row = i / W, ch = i - row * W, h = ch / C;
            e[u] = (ch - h * C) * V;
            t[u] = row * a.pairs + e[u];
            at[u] = row * a.ldy + (long)h * a.hd + e[u];
            const bf16* from = x + row * a.ldx + (long)h * a.hd + e[u];
            p[u] = *reinterpret_cast<const vec_a4*>(from);
            q[u] = *reinterpret_cast<const vec_a4*>(from + a.pairs);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + 256 * u >= n) break;
            vec vp, vq;
#pragma unroll
            for (int w = 0; w < V / 2; ++w) {
                const float2 c0 = cs[t[u] + 2 * w], c1 = cs[t[u] + 2 * w + 1];
                vp[w] = pack(lo(p[u][w]) * c0.x - lo(q[u][w]) * c0.y, hi(p[u][w]) * c1.x - hi(q[u][w]) * c1.y);
                vq[w] = pack(lo(q[u][w]) * c0.x + lo(p[u][w]) * c0.y, hi(q[u][w]) * c1.x + hi(p[u][w]) * c1.y);
            }
            if (NT) {
                __builtin_nontemporal_store(vp, reinterpret_cast<vec_a4*>(y + at[u]));
                __builtin_nontemporal_store(vq, reinterpret_cast<vec_a4*>(y + at[u] + a.pairs));
            } else {
                *reinterpret_cast<vec_a4*>(y + at[u]) = vp;
                *reinterpret_cast<vec_a4*>(y + at[u] + a.pairs) = vq;
            }
        }
    }
}

// Any sizes and alignment: one thread an element pair through all heads, or an element behind the pairs. HBM again:
// 16 480 rows of 9 heads of 254 (151 MB) 33 us in halves, 30 us adjacent.
template <bool ADJ>
__global__ __launch_bounds__(256) void rope_axes_any_kernel(RopeArgs a) {
    const int per = a.hd - a.pairs;
    const long gid = (long)blockIdx.x * 256 + threadIdx.x;
    if (gid >= (long)a.rows * per) return;
    const int row = (int)(gid / per), i = (int)(gid % per);
    const bf16* x = a.x + row * a.ldx;
    bf16* y = a.y + row * a.ldy;
    if (i >= a.pairs) {
        if (a.x != a.y)
            for (int h = 0; h < a.nheads; ++h) y[(long)h * a.hd + a.pairs + i] = x[(long)h * a.hd + a.pairs + i];
        return;
    }
    const float2 c = turn(a, row, i);
    const int ea = ADJ ? 2 * i : i, eb = ADJ ? 2 * i + 1 : i + a.pairs;
    for (int h = 0; h < a.nheads; ++h) {
        const float p = bf2f(x[(long)h * a.hd + ea]), q = bf2f(x[(long)h * a.hd + eb]);
        y[(long)h * a.hd + ea] = f2bf(p * c.x - q * c.y);
        y[(long)h * a.hd + eb] = f2bf(q * c.x + p * c.y);
    }
}

}  // namespace

extern "C" int mme_rope_axes(const void* x, long ldx, void* y, long ldy, int rows, int nheads, int hd, int pairs,
                             const int32_t* positions, long ld_pos, int naxes, const double* freqs, const int32_t* axes,
                             int adjacent, int inverse, void* stream) {
    MME_REQUIRE(rows >= 0 && nheads > 0 && nheads <= 65535 && naxes > 0, "mme_rope_axes: bad shape");
    MME_REQUIRE(pairs > 0 && hd > 0 && 2L * pairs <= hd, "mme_rope_axes: %d pairs do not fit a head of %d", pairs, hd);
    MME_REQUIRE((long)nheads * hd < (1L << 24), "mme_rope_axes: rows of %ld elements", (long)nheads * hd);
    MME_REQUIRE(ldx >= (long)nheads * hd && ldy >= (long)nheads * hd && ld_pos >= 0, "mme_rope_axes: bad leading dims");
    if (rows == 0) return MME_OK;
    MME_REQUIRE(x && y && positions && freqs && axes, "mme_rope_axes: null pointer");
    MME_REQUIRE(x != y || ldx == ldy, "mme_rope_axes: in place with two leading dims");
    MME_REQUIRE(((uintptr_t)x & 1) == 0 && ((uintptr_t)y & 1) == 0 && ((uintptr_t)positions & 3) == 0 &&
                    ((uintptr_t)axes & 3) == 0 && ((uintptr_t)freqs & 7) == 0,
                "mme_rope_axes: misaligned pointer");
    MME_REQUIRE(x == y || !mme_rows_overlap(x, ldx, rows, (long)nheads * hd, y, ldy, rows, (long)nheads * hd),
                "mme_rope_axes: x and y overlap");
    RopeArgs a{(const bf16*)x, (bf16*)y, positions, freqs, axes, ldx, ldy, ld_pos, rows, nheads, hd, pairs, naxes, 0,
               inverse ? -1.0f : 1.0f};
    hipStream_t s = as_stream(stream);
    const bool chunks = hd % 8 == 0 && pairs % 4 == 0 && ldx % 2 == 0 && ldy % 2 == 0 &&
                        (((uintptr_t)x | (uintptr_t)y) & 3) == 0 && pairs <= 1024;
    if (!chunks) {
        const long blocks = ((long)rows * (hd - pairs) + 255) / 256;
        MME_REQUIRE(blocks < (1L << 24), "mme_rope_axes: too many rows");  // a launch has under 2^32 threads
        if (adjacent)
            hipLaunchKernelGGL(rope_axes_any_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL(rope_axes_any_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, s, a);
        return mme_check_launch("mme_rope_axes");
    }
    // rows a workgroup: enough for four chunks a thread, but workgroups for all CUs first, and 16 KB of LDS at most
    const long row_bytes = 2L * nheads * hd;
    long R = 16384 / row_bytes + 1;
    if (R > (rows + 1023L) / 1024) R = (rows + 1023L) / 1024;
    if (R > 2048 / pairs) R = 2048 / pairs;
    MME_REQUIRE((rows + R - 1) / R < (1L << 24), "mme_rope_axes: too many rows");
    a.R = (int)R;
    const dim3 grid((unsigned)((rows + R - 1) / R));
    const size_t shared = (size_t)R * pairs * sizeof(float2);
    const bool nt = rows * row_bytes > (16L << 20);
    if (adjacent && nt)
        hipLaunchKernelGGL((rope_axes_kernel<true, true>), grid, dim3(256), shared, s, a);
    else if (adjacent)
        hipLaunchKernelGGL((rope_axes_kernel<true, false>), grid, dim3(256), shared, s, a);
    else if (pairs % 64 == 0 && nt)
        hipLaunchKernelGGL((rope_axes_halves_kernel<8, true>), grid, dim3(256), shared, s, a);
    else if (pairs % 64 == 0 || (x == y && pairs % 8 == 0))
        hipLaunchKernelGGL((rope_axes_halves_kernel<8, false>), grid, dim3(256), shared, s, a);
    else if (x == y)
        hipLaunchKernelGGL((rope_axes_halves_kernel<4, false>), grid, dim3(256), shared, s, a);
    else if (nt)
        hipLaunchKernelGGL((rope_axes_kernel<false, true>), grid, dim3(256), shared, s, a);
    else
        hipLaunchKernelGGL((rope_axes_kernel<false, false>), grid, dim3(256), shared, s, a);
    return mme_check_launch("mme_rope_axes");
}
