// Rotary positions with several axes (time, height, width, ...): pair i of every head turns by the angle
// positions[axis_i][row] * freq_i,
//   y_a = x_a cos - x_b sin,  y_b = x_b cos + x_a sin,
// with (a, b) = (i, i + pairs) or (2 i, 2 i + 1). The inverse rotation (-angle) is its gradient.
//
// Bound: HBM (each element read once and written once, 6 flops a pair). The angle is taken in 64 bits and only
// its fraction of a turn goes on in 32, so a position of 10^6 keeps its angle; products and the sum are fp32,
// one rounding to bf16 at the end. v_sin_f32 / v_cos_f32 take the angle in turns as it is.
#include "common.h"

namespace {

struct RopeArgs {
    const bf16* x;
    bf16* y;
    const int32_t* pos;
    const double* freqs;
    const int32_t* axes;
    long ldx, ldy, ldp, items;
    int npc, per_row, nheads, hd, pairs, naxes;
    float sign;
};

template <int V>
struct Bits {
    unsigned short u[V];
};
template <int V>
__device__ __forceinline__ Bits<V> load_bits(const bf16* p) {
    Bits<V> b;
    __builtin_memcpy(&b, __builtin_assume_aligned(p, V * 2), V * 2);
    return b;
}
template <int V>
__device__ __forceinline__ void store_bits(bf16* p, const Bits<V>& b) {
    __builtin_memcpy(__builtin_assume_aligned(p, V * 2), &b, V * 2);
}
__device__ __forceinline__ unsigned short f2bits(float f) { return __builtin_bit_cast(unsigned short, f2bf(f)); }

// One thread: V pairs of one row (their sines and cosines computed once) through HPT heads, whose loads are all
// issued before the first product. Items past npc of a row copy V elements behind the rotated ones.
template <int V, bool ADJ, int HPT>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeArgs a) {
    const long gid = (long)blockIdx.x * 256 + threadIdx.x;
    if (gid >= a.items) return;
    const int it = (int)(gid % a.per_row);
    const long row = gid / a.per_row;
    const int h0 = blockIdx.y * HPT;
    const bf16* xr = a.x + row * a.ldx;
    bf16* yr = a.y + row * a.ldy;
    if (it >= a.npc) {
        const int e = 2 * a.pairs + (it - a.npc) * V;
#pragma unroll
        for (int h = 0; h < HPT; ++h)
            if (h0 + h < a.nheads) store_bits<V>(yr + (long)(h0 + h) * a.hd + e, load_bits<V>(xr + (long)(h0 + h) * a.hd + e));
        return;
    }
    const int i0 = it * V;
    const int ea = ADJ ? 2 * i0 : i0, eb = ADJ ? 2 * i0 + V : i0 + a.pairs;
    Bits<V> ua[HPT], ub[HPT];
#pragma unroll
    for (int h = 0; h < HPT; ++h) {
        const long o = (long)min(h0 + h, a.nheads - 1) * a.hd;
        ua[h] = load_bits<V>(xr + o + ea);
        ub[h] = load_bits<V>(xr + o + eb);
    }
    float cs[V], sn[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int ax = min(max(a.axes[i0 + j], 0), a.naxes - 1);
        const double t = (double)a.pos[ax * a.ldp + row] * a.freqs[i0 + j] * 0.15915494309189535;
        const float f = (float)(t - __builtin_rint(t));
        cs[j] = __builtin_amdgcn_cosf(f);
        sn[j] = __builtin_amdgcn_sinf(f) * a.sign;
    }
#pragma unroll
    for (int h = 0; h < HPT; ++h) {
        if (h0 + h >= a.nheads) break;
        const long o = (long)(h0 + h) * a.hd;
        Bits<V> va, vb;
        if constexpr (ADJ) {
            unsigned short u[2 * V], w[2 * V];
#pragma unroll
            for (int j = 0; j < V; ++j) u[j] = ua[h].u[j], u[V + j] = ub[h].u[j];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = bits2f(u[2 * j]), q = bits2f(u[2 * j + 1]);
                w[2 * j] = f2bits(p * cs[j] - q * sn[j]);
                w[2 * j + 1] = f2bits(q * cs[j] + p * sn[j]);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) va.u[j] = w[j], vb.u[j] = w[V + j];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = bits2f(ua[h].u[j]), q = bits2f(ub[h].u[j]);
                va.u[j] = f2bits(p * cs[j] - q * sn[j]);
                vb.u[j] = f2bits(q * cs[j] + p * sn[j]);
            }
        }
        store_bits<V>(yr + o + ea, va);
        store_bits<V>(yr + o + eb, vb);
    }
}

template <int V, bool ADJ>
void launch_rope(const RopeArgs& a, hipStream_t s) {
    // Heads a thread: one where the rows are few (the angles of a row computed per head, latency), four otherwise.
    const int blocks = cdiv(a.items, 256);
    if ((long)blocks * a.nheads <= 2048)
        hipLaunchKernelGGL((rope_axes_kernel<V, ADJ, 1>), dim3(blocks, a.nheads), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((rope_axes_kernel<V, ADJ, 4>), dim3(blocks, cdiv(a.nheads, 4)), dim3(256), 0, s, a);
}

}  // namespace

extern "C" int mme_rope_axes(const void* x, long ldx, void* y, long ldy, int rows, int nheads, int hd, int pairs,
                             const int32_t* positions, long ld_pos, int naxes, const double* freqs, const int32_t* axes,
                             int adjacent, int inverse, void* stream) {
    MME_REQUIRE(rows >= 0 && nheads > 0 && nheads <= 65535 && naxes > 0, "mme_rope_axes: bad shape");
    MME_REQUIRE(pairs > 0 && hd > 0 && 2L * pairs <= hd, "mme_rope_axes: %d pairs do not fit a head of %d", pairs, hd);
    MME_REQUIRE(ldx >= (long)nheads * hd && ldy >= (long)nheads * hd && ld_pos >= rows, "mme_rope_axes: bad leading dims");
    if (rows == 0) return MME_OK;
    MME_REQUIRE(x && y && positions && freqs && axes, "mme_rope_axes: null pointer");
    MME_REQUIRE(x != y || ldx == ldy, "mme_rope_axes: in place with two leading dims");
    MME_REQUIRE(((uintptr_t)x & 1) == 0 && ((uintptr_t)y & 1) == 0 && ((uintptr_t)positions & 3) == 0 &&
                    ((uintptr_t)axes & 3) == 0 && ((uintptr_t)freqs & 7) == 0,
                "mme_rope_axes: misaligned pointer");
    // the widest vector that divides every offset of the two rows: 16-byte, 8-byte, or single elements
    const uintptr_t al = (uintptr_t)x | (uintptr_t)y | (uintptr_t)(2 * ldx) | (uintptr_t)(2 * ldy) | (uintptr_t)(2 * hd) |
                         (uintptr_t)(2 * pairs);
    const int V = (al & 15) == 0 ? 8 : (al & 7) == 0 ? 4 : 1;
    RopeArgs a{(const bf16*)x, (bf16*)y, positions, freqs, axes, ldx, ldy, ld_pos, 0,
               pairs / V, 0, nheads, hd, pairs, naxes, inverse ? -1.0f : 1.0f};
    a.per_row = a.npc + (x == y ? 0 : (hd - 2 * pairs) / V);
    a.items = (long)rows * a.per_row;
    MME_REQUIRE(a.items < (1L << 38), "mme_rope_axes: too many rows");
    hipStream_t s = as_stream(stream);
    if (V == 8)
        adjacent ? launch_rope<8, true>(a, s) : launch_rope<8, false>(a, s);
    else if (V == 4)
        adjacent ? launch_rope<4, true>(a, s) : launch_rope<4, false>(a, s);
    else
        adjacent ? launch_rope<1, true>(a, s) : launch_rope<1, false>(a, s);
    return mme_check_launch("mme_rope_axes");
}
