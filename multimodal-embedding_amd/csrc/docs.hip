// Attention over packed documents: documents of any lengths lie one after the other in the rows of q and of k / v,
// and a query sees keys of its own document only (all of them, those up to itself, or a prefix and those up to
// itself), its scores capped by a tanh and / or lowered by a slope times the distance.
//
//   x = scale q.k ;  x = cap tanh(x / cap) ;  x -= slope_h |p_q - p_k| ;  o = softmax over the visible keys (x) . v
//
// with p_q = i + klen - qlen for query i. Every mask here leaves a row one interval of keys, [0, hi) from its
// document's first, so a tile of scores is whole, empty, or cut by one comparison a score.
//
// One workgroup = NW waves of 32 flat rows of one document and one key head, a flat row being (query, head of the
// group), so grouped heads share the K / V tiles (and a single query fills a tile with its group's heads). Tiles of
// 32 or 64 keys land in LDS by DMA as "chunk planes" (plane c = 16-byte column chunk c of the tile's keys, V planes
// XOR-swizzled for the transposed reads), a ring of two, one barrier a tile. S^T = K.Q^T on 32x32x16 MFMA puts one
// query on a lane; softmax runs in fp32 registers in one pass (running maximum, rescale only when it grows by more
// than 2^8); P, rounded to bf16 for the matrix instruction, is directly the operand of O^T = V^T.P^T.
//
// A key outside a row's interval adds nothing to it, whatever K and V hold there: K rows past a document are never
// read, masked scores are replaced and not added to, and a cut tile whose V holds an infinity or NaN takes a path
// that keeps 0 x NaN out of the rows that do not see it.
//
// Few query rows and many keys (max_rows given): the keys of each document are split into chunks, one workgroup
// each, which leave (maximum, sum, O) in a workspace, and a second launch joins them.
#include "common.h"

#pragma clang fp contract(off)  // every fused multiply-add below is written as one

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct DocsArgs {
    const bf16 *q, *k, *v;
    bf16* out;
    const int32_t *qoff, *koff, *prefix;
    const float* slopes;
    float* part;        // split: [slot][key head][flat row] of hd + 2 floats
    long ldq, ldk, ldv, ldo;
    long nslots;
    int n, rows_q, rows_k, Hkv, group, hd, nch, max_rows, causal, chunk, part_rows;
    float scale_log2, cap_log2, cap_in;
};

__device__ __forceinline__ float xmax32(float v) {  // over lanes l, l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xsum32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int offset_at(const int32_t* off, int i, int rows) { return min(max(off[i], 0), rows); }

// Work is dealt out in slots of `per` units (flat rows, or keys). Document d owns the slots from
// off[d] * mul / per + d on: that many always hold its units, because rounding down loses less than the one slot
// that `+ d` adds, so a slot finds its document by a search in `off` and no table is needed. Surplus slots end at
// once. 64 lanes look at 64 documents a step. Offsets are clamped to [0, rows]: wrong ones give wrong rows, never a
// wrong address.
__device__ __forceinline__ long first_slot(const int32_t* off, int d, int rows, int mul, int per) {
    return (long)offset_at(off, d, rows) * mul / per + d;
}
__device__ __forceinline__ int find_doc(const int32_t* off, int n, int rows, int mul, int per, long slot) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) >> 6;
        const int i = lo + lane * step;
        const bool le = i < hi && first_slot(off, min(i, n - 1), rows, mul, per) <= slot;
        const int c = __popcll(__builtin_amdgcn_ballot_w64(le));
        if (c > 0) lo += (c - 1) * step;
        hi = min(hi, lo + step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

template <int HDP>
struct Tile {
    static constexpr int KT = HDP > 128 ? 32 : 64;   // keys a tile: head dim 256 keeps its registers and LDS at half
    static constexpr int KB = KT / 32;
    static constexpr int NKS = HDP / 16;              // k-steps of Q K^T
    static constexpr bool ONES = HDP % 32 != 0;       // a V plane of ones in the padding sums the weights
    static constexpr int NDB = (HDP + 31) / 32;       // 32-column blocks of O^T
    static constexpr int NKP = 2 * NKS, NVP = 4 * NDB;
    static constexpr int PLANE = KT * 16;
    static constexpr int BYTES = (NKP + NVP) * PLANE;
};

template <int HDP, int NW, int MINW, bool SPLIT>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(MINW))) void attn_docs_kernel(DocsArgs a) {
    using T = Tile<HDP>;
    constexpr int KT = T::KT, KB = T::KB, NKS = T::NKS, NDB = T::NDB, PLANE = T::PLANE, QB = NW * 32;
    __shared__ __attribute__((aligned(16))) char lds[2 * T::BYTES];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, hh = lane >> 5;
    long id;
    {  // consecutive slots of one key head (the same K / V) on one XCD
        const long bid = blockIdx.x, nwg = gridDim.x;
        const long xcd = bid & 7, loc = bid >> 3, q8 = nwg >> 3, r8 = nwg & 7;
        id = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + loc;
    }
    const long slot = id % a.nslots;
    const int kvh = (int)(id / a.nslots);
    const int d = SPLIT ? find_doc(a.koff, a.n, a.rows_k, 1, a.chunk, slot) : find_doc(a.qoff, a.n, a.rows_q, a.group, QB, slot);
    const int q0 = offset_at(a.qoff, d, a.rows_q), k0 = offset_at(a.koff, d, a.rows_k);
    const int qlen = max(offset_at(a.qoff, d + 1, a.rows_q) - q0, 0), klen = max(offset_at(a.koff, d + 1, a.rows_k) - k0, 0);
    const long flat = (long)min(qlen, a.max_rows) * a.group;  // flat rows of this document
    long part = slot - (SPLIT ? first_slot(a.koff, d, a.rows_k, 1, a.chunk) : first_slot(a.qoff, d, a.rows_q, a.group, QB));
    const long nparts = SPLIT ? ((long)klen + a.chunk - 1) / a.chunk : (flat + QB - 1) / QB;
    if (part < 0 || part >= nparts || flat == 0) return;
    if (!SPLIT && a.causal) part = nparts - 1 - part;  // the rows with the most keys first

    const long f0 = SPLIT ? wave * 32 : part * QB + wave * 32;
    const long fr = f0 + r;                                     // this lane's flat row
    const long frc = min(fr, flat - 1);
    const int qi = (int)(frc / a.group), gh = kvh * a.group + (int)(frc % a.group);
    const int pq = qi + klen - qlen;                            // its place among the keys
    const int pre = a.prefix ? min(max(a.prefix[d], 0), klen) : 0;
    const int hi = a.causal ? min(klen, max(pre, pq + 1)) : klen;  // it sees keys [0, hi)
    const int key_lo = SPLIT ? (int)(part * a.chunk) : 0;
    // the last row of the block sees the most keys
    int hi_blk;
    {
        const int ql = (int)(min(SPLIT ? (long)QB : (part + 1) * QB, flat) - 1) / a.group;
        hi_blk = a.causal ? min(klen, max(pre, ql + klen - qlen + 1)) : klen;
        if (SPLIT) hi_blk = min((long)hi_blk, (long)key_lo + a.chunk);
    }
    const int nkt = hi_blk > key_lo ? (hi_blk - key_lo + KT - 1) / KT : 0;

    // planes past the head dim: zeros, and the ones plane at column HDP
    for (int i = tid; i < 2 * (T::NKP + T::NVP) * KT; i += QB * 2) {
        const int pl = i / KT % (T::NKP + T::NVP), c = pl < T::NKP ? pl : pl - T::NKP;
        if (c < a.nch) continue;
        const unsigned short one = (T::ONES && pl >= T::NKP && c == HDP / 8) ? 0x3F80 : 0;
        *reinterpret_cast<u16x8*>(lds + (long)i * 16) = u16x8{one, one, one, one, one, one, one, one};
    }

    bf16x8 qf[NKS];  // B operand: Q^T[16 ks + 8 hh + j][row r]
    {
        const bf16* qrow = a.q + (q0 + (long)qi) * a.ldq + (long)gh * a.hd;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
            qf[ks] = __builtin_bit_cast(bf16x8, load_chunk_or_zero(qrow, 2 * ks + hh, a.nch));
    }
    const float slope = a.slopes ? a.slopes[gh] * LOG2E : 0.f;
    const float c = a.cap_log2 != 0.f || a.slopes ? 1.0f : a.scale_log2;  // what a score is still multiplied by

    const bf16* kbase = a.k + (long)k0 * a.ldk + (long)kvh * a.hd;
    const bf16* vbase = a.v + (long)k0 * a.ldv + (long)kvh * a.hd;
    const int nins = a.nch * 2 * KT / 64;  // DMA instructions a tile: KT 64 one plane each, KT 32 two
    auto issue = [&](int t, unsigned so) {
        for (int idx = wave; idx < nins; idx += NW) {
            const int plane = KT == 64 ? idx : 2 * idx + hh;
            const int first = KT == 64 ? idx : 2 * idx;
            const bool isV = first >= a.nch;
            const int cc = isV ? plane - a.nch : plane;
            const int kl = lane & (KT - 1);
            const int key = min(key_lo + t * KT + (isV ? kl ^ (4 * (cc & 3)) : kl), klen - 1);
            const bf16* src = isV ? vbase + (long)key * a.ldv + cc * 8 : kbase + (long)key * a.ldk + cc * 8;
            glds16_asm(src, lds + so + (isV ? T::NKP + first - a.nch : first) * PLANE);
        }
    };

    const unsigned lds0 = (unsigned)(uintptr_t)(LDS_AS char*)lds;
    const unsigned kb0 = lds0 + hh * PLANE + r * 16;
    unsigned vbj[2];  // V^T fragment: two transposed reads, keys 16 s + 8 j + 4 hh + q at columns 16 half + 4 p ..
    {
        const int i16 = lane & 15, q = i16 >> 2, p = i16 & 3, half = (lane >> 4) & 1;
        const int cc = 2 * half + (p >> 1);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            vbj[j] = lds0 + (T::NKP + cc) * PLANE + (((8 * j + 4 * hh + q) ^ (4 * cc)) * 16) + (p & 1) * 8;
    }
    auto vfrag = [&](unsigned so, int i, int db) __attribute__((always_inline)) {  // key step i = 2 kb + s
        const unsigned off = so + db * 4 * PLANE + i * 256;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(uintptr_t)(vbj[0] + off));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(uintptr_t)(vbj[1] + off));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    f32x16 o[NDB];
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, lsum = 0.f;

    auto tile = [&](int t, const unsigned so) __attribute__((always_inline)) {
        const int key0 = key_lo + t * KT;
        f32x16 sc[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 z;
#pragma unroll
            for (int e = 0; e < 16; ++e) z[e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                const bf16x8 kf = *reinterpret_cast<const LDS_AS bf16x8*>((uintptr_t)(kb0 + so + kb * 512 + ks * 2 * PLANE));
                z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], z, 0, 0, 0);
            }
            sc[kb] = z;
        }
        // register e of block kb scores key key0 + 32 kb + (e & 3) + 8 (e >> 2) + 4 hh
        if (a.cap_log2 != 0.f) {  // cap tanh(x / cap) = cap - 2 cap / (1 + e^(2 x / cap)), log2(e) folded in
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float w = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sc[kb][e] * a.cap_in));
                    sc[kb][e] = __builtin_fmaf(-2.0f * a.cap_log2, w, a.cap_log2);
                }
        } else if (a.slopes) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[kb][e] *= a.scale_log2;
        }
        if (a.slopes) {
            const float db = (float)(pq - key0 - 4 * hh);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    sc[kb][e] = __builtin_fmaf(-slope, fabsf(db - (float)(32 * kb + (e & 3) + 8 * (e >> 2))), sc[kb][e]);
        }
        const int lim = hi - key0;
        const bool cut = __builtin_amdgcn_ballot_w64(lim < KT) != 0;
        if (cut) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * kb + (e & 3) + 8 * (e >> 2) + 4 * hh >= lim) sc[kb][e] = -INFINITY;
        }

        float mloc = fmaxf(sc[0][0], sc[0][1]);
#pragma unroll
        for (int e = 2; e < 16; ++e) mloc = fmaxf(mloc, sc[0][e]);
#pragma unroll
        for (int kb = 1; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) mloc = fmaxf(mloc, sc[kb][e]);
        mloc = xmax32(mloc);
        if (__builtin_amdgcn_ballot_w64((mloc - m) * c > 8.0f)) {  // P stays under 2^8 otherwise
            const float mnew = fmaxf(m, mloc);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mnew) * c);
            if (!T::ONES) lsum *= alpha;
#pragma unroll
            for (int i = 0; i < NDB; ++i) o[i] *= alpha;
            m = mnew;
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
        float cf = c;
        if (__builtin_amdgcn_ballot_w64(fabsf(mc) > 0x1p20f)) {
            // m c is rounded, s c inside the fused exponent is not: where that alone is worth whole powers of two,
            // round both
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[kb][e] *= c;
            cf = 1.0f;
        }
        bf16x8 pk[2 * KB];
        float psum = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][e], cf, -mc));
                if (!T::ONES) psum += p;
                pk[2 * kb + (e >> 3)][e & 7] = f2bf(p);
            }
        if (!T::ONES) lsum += psum;

        bool odd = false;
        if (cut) {  // does V of this tile hold an infinity or NaN?
            u16x4 least = {0xffff, 0xffff, 0xffff, 0xffff};
#pragma unroll
            for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
                for (int db = 0; db < NDB; ++db) {
                    const u16x8 w = ~__builtin_bit_cast(u16x8, vfrag(so, i, db)) & (unsigned short)0x7f80;
                    least = __builtin_elementwise_min(least, __builtin_elementwise_min(
                        __builtin_shufflevector(w, w, 0, 1, 2, 3), __builtin_shufflevector(w, w, 4, 5, 6, 7)));
                }
            const bool bad = least[0] == 0 || least[1] == 0 || least[2] == 0 || least[3] == 0;
            odd = __builtin_amdgcn_ballot_w64(bad) != 0;
        }
        if (!odd) {
#pragma unroll
            for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
                for (int db = 0; db < NDB; ++db)
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vfrag(so, i, db), pk[i], o[db], 0, 0, 0);
        } else {  // key by key, a row that does not see the key keeping what it had
#pragma unroll
            for (int i = 0; i < 2 * KB; ++i)
                for (int kk = 0; kk < 16; ++kk) {  // element kk & 7 of lane half kk >> 3
                    const int j = kk & 7, h1 = kk >> 3;
                    const bool sees = 16 * i + (j & 3) + 8 * (j >> 2) + 4 * h1 < lim;
                    u32x4 keep;
#pragma unroll
                    for (int w = 0; w < 4; ++w) keep[w] = (hh == h1 && (j >> 1) == w) ? 0xffffu << (16 * (j & 1)) : 0u;
                    const bf16x8 p1 = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, pk[i]) & keep);
#pragma unroll
                    for (int db = 0; db < NDB; ++db) {
                        const bf16x8 v1 = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, vfrag(so, i, db)) & keep);
                        const f32x16 s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v1, p1, o[db], 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[db][e] = sees ? s[e] : o[db][e];
                    }
                }
        }
    };

    // this wave's part of the next tile has landed and its LDS reads are done; then everybody's
    auto meet = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (nkt > 0) issue(0, 0);
    for (int t = 0; t < nkt; t += 2) {
        meet();
        if (t + 1 < nkt) issue(t + 1, T::BYTES);
        tile(t, 0);
        if (t + 1 < nkt) {
            meet();
            if (t + 2 < nkt) issue(t + 2, 0);
            tile(t + 1, T::BYTES);
        }
    }

    const float l = T::ONES ? o[HDP / 32][4 * ((HDP % 32) / 8)] : xsum32(lsum);
    if constexpr (SPLIT) {
        if (fr < flat) {
            float* row = a.part + ((slot * a.Hkv + kvh) * a.part_rows + fr) * (a.hd + 2);
            if (hh == 0) *reinterpret_cast<float2*>(row) = make_float2(m * c, l);
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int mm = 0; mm < 4; ++mm) {
                    const int d0 = 32 * db + 8 * mm + 4 * hh;
                    if (d0 < a.hd) {
                        *reinterpret_cast<float2*>(row + 2 + d0) = make_float2(o[db][4 * mm], o[db][4 * mm + 1]);
                        *reinterpret_cast<float2*>(row + 4 + d0) = make_float2(o[db][4 * mm + 2], o[db][4 * mm + 3]);
                    }
                }
        }
        return;
    }
    const float inv = hi > 0 ? 1.0f / l : 0.f;  // a row that sees nothing is 0
    bf16* orow = a.out + (q0 + (long)qi) * a.ldo + (long)gh * a.hd;
    // registers 4 mm .. of block db = columns 32 db + 8 mm + 4 hh ..; the swap of the lane halves makes 16 bytes
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int mm = 0; mm < 4; mm += 2) {
            bf16x4 v0, v1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v0[e] = f2bf(o[db][4 * mm + e] * inv);
                v1[e] = f2bf(o[db][4 * mm + 4 + e] * inv);
            }
            const uint2 x = __builtin_bit_cast(uint2, v0), y = __builtin_bit_cast(uint2, v1);
            const auto sx = __builtin_amdgcn_permlane32_swap(x.x, y.x, false, false);
            const auto sy = __builtin_amdgcn_permlane32_swap(x.y, y.y, false, false);
            const int d0 = 32 * db + 8 * (mm + hh);
            if (fr < flat && d0 < a.hd) *reinterpret_cast<uint4*>(orow + d0) = make_uint4(sx[0], sy[0], sx[1], sy[1]);
        }
}

// Joins a document's chunks: one wave a (document, flat row, key head), 64 columns a step.
__global__ __launch_bounds__(256) void join_docs_kernel(DocsArgs a) {
    const int lane = threadIdx.x & 63;
    const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long fr = w % a.part_rows;
    const int kvh = (int)(w / a.part_rows % a.Hkv);
    const int d = (int)(w / a.part_rows / a.Hkv);
    if (d >= a.n) return;
    const int q0 = offset_at(a.qoff, d, a.rows_q), k0 = offset_at(a.koff, d, a.rows_k);
    const int qlen = max(offset_at(a.qoff, d + 1, a.rows_q) - q0, 0), klen = max(offset_at(a.koff, d + 1, a.rows_k) - k0, 0);
    if (fr >= (long)min(qlen, a.max_rows) * a.group) return;
    const int qi = (int)(fr / a.group), gh = kvh * a.group + (int)(fr % a.group);
    const int pre = a.prefix ? min(max(a.prefix[d], 0), klen) : 0;
    const int hi = a.causal ? min(klen, max(pre, qi + klen - qlen + 1)) : klen;
    const int nparts = (int)(((long)klen + a.chunk - 1) / a.chunk);
    const long step = (long)a.Hkv * a.part_rows * (a.hd + 2);
    const float* p0 = a.part + ((first_slot(a.koff, d, a.rows_k, 1, a.chunk) * a.Hkv + kvh) * a.part_rows + fr) * (a.hd + 2);
    float m = -INFINITY;
    for (int s = lane; s < nparts; s += 64) m = fmaxf(m, p0[s * step]);
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
    const float mr = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = 0; s < nparts; ++s) l = __builtin_fmaf(__builtin_amdgcn_exp2f(p0[s * step] - mr), p0[s * step + 1], l);
    const float inv = hi > 0 ? 1.0f / l : 0.f;
    bf16* orow = a.out + (q0 + (long)qi) * a.ldo + (long)gh * a.hd;
    for (int col = lane; col < a.hd; col += 64) {
        float acc = 0.f;
        for (int s = 0; s < nparts; ++s) acc = __builtin_fmaf(__builtin_amdgcn_exp2f(p0[s * step] - mr), p0[s * step + 2 + col], acc);
        orow[col] = f2bf(hi > 0 ? acc * inv : 0.f);
    }
}

struct Plan {
    bool split;
    int NW, chunk, part_rows;
    long nslots;
    size_t ws;
};

int padded(int hd) { return hd <= 64 ? 64 : hd <= 80 ? 80 : hd <= 128 ? 128 : 256; }

Plan make_plan(int n, int rows_q, int rows_k, int Hkv, int group, int hd, int max_rows) {
    Plan p{};
    const long mean = n ? (long)rows_q * group / n : 0;
    p.NW = mean <= 48 ? 1 : 4;
    p.nslots = (long)rows_q * group / (p.NW * 32) + n;
    const long mr = (long)max_rows * group;
    const long blocks = p.nslots * Hkv;
    if (n && mr <= 32 && rows_k / n > 256 && blocks < 2048) {
        p.split = true;
        p.NW = 1;
        const long want = (2048 + Hkv - 1) / Hkv;  // chunks in all
        long chunk = ((long)rows_k / want + 63) / 64 * 64;
        p.chunk = (int)(chunk < 128 ? 128 : chunk);
        p.part_rows = (int)mr;
        p.nslots = (long)rows_k / p.chunk + n;
        p.ws = (size_t)p.nslots * Hkv * mr * (hd + 2) * 4;
    }
    return p;
}

template <int HDP, int NW, int MINW, bool SPLIT>
void launch_docs(const DocsArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((attn_docs_kernel<HDP, NW, MINW, SPLIT>), dim3((unsigned)(a.nslots * a.Hkv)), dim3(NW * 64), 0, s, a);
}

template <int HDP, int MINW>
void launch_width(const DocsArgs& a, const Plan& p, hipStream_t s) {
    if (p.split)
        launch_docs<HDP, 1, MINW, true>(a, s);
    else if (p.NW == 1)
        launch_docs<HDP, 1, MINW, false>(a, s);
    else
        launch_docs<HDP, 4, MINW, false>(a, s);
}

int check_docs(int n, int rows_q, int rows_k, int Hq, int Hkv, int hd, int max_rows) {
    MME_REQUIRE(n >= 0 && rows_q >= 0 && rows_k >= 0 && max_rows >= 0, "mme_attention_docs: bad shape");
    MME_REQUIRE(Hkv > 0 && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0, "mme_attention_docs: %d heads over %d key heads", Hq, Hkv);
    MME_REQUIRE(hd > 0 && (hd <= 128 ? hd % 8 == 0 : hd <= 256 && hd % 16 == 0),
                "mme_attention_docs: head_dim %d unsupported (multiples of 8 to 128, of 16 to 256)", hd);
    return MME_OK;
}

}  // namespace

extern "C" size_t mme_attention_docs_workspace_bytes(int n, int rows_q, int rows_k, int Hq, int Hkv, int hd, int max_rows) {
    if (check_docs(n, rows_q, rows_k, Hq, Hkv, hd, max_rows) != MME_OK) return 0;
    return make_plan(n, rows_q, rows_k, Hkv, Hq / Hkv, hd, max_rows < rows_q ? max_rows : rows_q).ws;
}

extern "C" int mme_attention_docs(const void* q, long ldq, const void* k, long ldk, const void* v, long ldv, void* out,
                                  long ldo, const int32_t* q_offsets, const int32_t* k_offsets, int n, int rows_q,
                                  int rows_k, int Hq, int Hkv, int hd, int max_rows, int causal, const int32_t* prefix,
                                  float softcap, const float* slopes, float scale, void* workspace, size_t ws_bytes,
                                  void* stream) {
    if (int rc = check_docs(n, rows_q, rows_k, Hq, Hkv, hd, max_rows)) return rc;
    MME_REQUIRE(scale > 0.f && scale < INFINITY, "mme_attention_docs: scale must be positive and finite");
    MME_REQUIRE(softcap >= 0.f && softcap < INFINITY, "mme_attention_docs: softcap must be 0 (none) or positive and finite");
    MME_REQUIRE(causal || !prefix, "mme_attention_docs: a prefix goes with the causal mask");
    if (n == 0 || rows_q == 0) return MME_OK;
    MME_REQUIRE(q && out && q_offsets && k_offsets && (rows_k == 0 || (k && v)), "mme_attention_docs: null pointer");
    MME_REQUIRE(ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldo % 8 == 0 && ldq >= (long)Hq * hd &&
                    ldo >= (long)Hq * hd && ldk >= (long)Hkv * hd && ldv >= (long)Hkv * hd,
                "mme_attention_docs: bad leading dims");
    MME_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0 &&
                    (((uintptr_t)q_offsets | (uintptr_t)k_offsets | (uintptr_t)prefix | (uintptr_t)slopes) & 3) == 0,
                "mme_attention_docs: misaligned pointer");
    const int mr = max_rows < rows_q ? max_rows : rows_q;
    if (mr == 0) return MME_OK;
    const Plan p = make_plan(n, rows_q, rows_k, Hkv, Hq / Hkv, hd, mr);
    MME_REQUIRE(p.nslots * Hkv < (1L << 31) && (long)n * Hkv * p.part_rows < (1L << 33), "mme_attention_docs: too many rows");
    MME_REQUIRE(p.ws == 0 || (workspace && ws_bytes >= p.ws && ((uintptr_t)workspace & 15) == 0),
                "mme_attention_docs: workspace of %zu bytes, %zu needed", ws_bytes, p.ws);
    DocsArgs a{};
    a.q = (const bf16*)q, a.k = (const bf16*)k, a.v = (const bf16*)v, a.out = (bf16*)out;
    a.qoff = q_offsets, a.koff = k_offsets, a.prefix = prefix, a.slopes = slopes, a.part = (float*)workspace;
    a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo, a.nslots = p.nslots;
    a.n = n, a.rows_q = rows_q, a.rows_k = rows_k, a.Hkv = Hkv, a.group = Hq / Hkv, a.hd = hd, a.nch = hd / 8;
    a.max_rows = mr, a.causal = causal ? 1 : 0, a.chunk = p.chunk, a.part_rows = p.part_rows;
    a.scale_log2 = scale * LOG2E;
    a.cap_log2 = softcap * LOG2E;
    a.cap_in = softcap != 0.f ? 2.0f * a.scale_log2 / softcap : 0.f;
    hipStream_t s = as_stream(stream);
    switch (padded(hd)) {
        case 64: launch_width<64, 2>(a, p, s); break;
        case 80: launch_width<80, 2>(a, p, s); break;
        case 128: launch_width<128, 2>(a, p, s); break;
        default: launch_width<256, 1>(a, p, s); break;
    }
    if (p.split) {
        if (int rc = mme_check_launch("mme_attention_docs")) return rc;
        hipLaunchKernelGGL(join_docs_kernel, dim3((unsigned)cdiv((long)n * Hkv * p.part_rows, 4)), dim3(256), 0, s, a);
    }
    return mme_check_launch("mme_attention_docs");
}
