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
// 32 or 64 keys land in LDS by DMA, row after row as they lie in memory (a wave's 1 KiB piece covers whole 128-byte
// lines: 16-byte pieces of 64 rows made the copy the bound), a ring of two, one barrier a tile; where a row is a
// power of two of 16-byte chunks, a chunk's place is XORed with its row so that a column of rows spreads over the
// banks. S^T = K.Q^T on 32x32x16 MFMA puts one query on a lane; softmax runs in fp32 registers in one pass (running
// maximum, rescale only when it grows by more than 2^8); P, rounded to bf16 for the matrix instruction, is directly
// the operand of O^T = V^T.P^T, V^T by transposed LDS reads.
//
// A key outside a row's interval adds nothing to it, whatever K and V hold there: rows of another document are never
// read (a tile's rows behind the document are zeros in V), masked scores are replaced and not added to, and where a
// causal row comes out not finite while V holds an infinity or NaN at a key that its tile has and it does not see
// (0 x NaN), the row is taken again from its own keys.
//
// Few query rows and many keys (max_rows given): the keys of each document are split into chunks, one workgroup
// each, which leave (maximum, sum, O) in a workspace, and a second launch joins them.
#include <type_traits>

#include "common.h"

#pragma clang fp contract(off)  // every fused multiply-add below is written as one

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f;

struct DocsArgs {
    const bf16 *q, *k, *v;
    bf16* out;
    const int32_t *qoff, *koff, *prefix;
    const float* slopes;
    float *part, *stat;  // split: O [slot][key head][flat row][hd], and (maximum, sum) [slot][key head][flat row][2]
    long ldq, ldk, ldv, ldo;
    int nslots, n, rows_q, rows_k, Hkv, group, hd, max_rows, causal, part_rows, row_blocks, sorted;
    int per;  // a slot's flat rows, or keys (split)
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
// 16 bytes a lane from base + off to LDS at `at` (wave-uniform, as base is) + 16 lane, retired by the caller's wait.
// The wait states cover an M0 write, and base in SGPRs that a vector instruction (a spill's reload) has just written.
__device__ __forceinline__ void dma16(const char* base, unsigned off, unsigned at) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(at) : "memory", "m0");
}
__device__ __forceinline__ int clamp_row(int x, int rows) { return min(max(x, 0), rows); }

// Work is dealt out in slots of `per` units (flat rows, or keys). Document d owns the slots from off[d] * mul / per + d
// on: that many always hold its units, because rounding down loses less than the one slot that `+ d` adds, so a slot
// finds its document by a search in `off` and no table is needed. Surplus slots end at once. Offsets are clamped to
// [0, rows]: wrong ones give wrong rows, never a wrong address.
__device__ __forceinline__ int first_slot(int off, int d, int mul, int per) {
    return (int)((unsigned)off * (unsigned)mul / (unsigned)per) + d;  // off * mul < 2^31
}

struct Doc {
    int d, q0, qlen, k0, klen, pre, first;
};
// SORT: with at most 63 documents and many workgroups (a.sorted) the slots go by documents, the one with most keys
// first, so that no long document is begun when the others are done.
template <bool SPLIT, bool SORT>
__device__ __forceinline__ Doc find_doc(const DocsArgs& a, int slot) {
    const int lane = threadIdx.x & 63;
    const int32_t* off = SPLIT ? a.koff : a.qoff;
    const int rows = SPLIT ? a.rows_k : a.rows_q, mul = SPLIT ? 1 : a.group;
    int lo = 0, hi = a.n;
    while (hi - lo > 63) {  // 64 documents a step
        const int step = (hi - lo + 63) >> 6;
        const int i = lo + lane * step;
        const bool le = i < hi && first_slot(clamp_row(off[min(i, a.n)], rows), i, mul, a.per) <= slot;
        const int c = __popcll(__builtin_amdgcn_ballot_w64(le));
        if (c > 0) lo += (c - 1) * step;
        hi = min(hi, lo + step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    // the last step's documents: lane l holds the offsets of document lo + l, all arrays in one round trip
    const int i = min(lo + lane, a.n);
    const int qo = clamp_row(a.qoff[i], a.rows_q), ko = clamp_row(a.koff[i], a.rows_k);
    const int pr = a.prefix ? a.prefix[min(i, a.n - 1)] : 0;
    int fs = first_slot(SPLIT ? ko : qo, i, mul, a.per), l;
    if (SORT && a.sorted) {
        // every lane takes part in the exchange: document n - 1 needs lane n's offsets
        const int ql = __shfl_down(qo, 1, 64) - qo, kd = __shfl_down(ko, 1, 64) - ko;
        const int kl = lane < a.n ? max(kd, 0) : -1;
        const int parts = lane < a.n ? (min(max(ql, 0), a.max_rows) * mul + a.per - 1) / a.per : 0;
        fs = 0;  // the slots of the documents before this lane's
        for (int j = 0; j < a.n; ++j) {
            const int kj = __builtin_amdgcn_readlane(kl, j), pj = __builtin_amdgcn_readlane(parts, j);
            fs += kj > kl || (kj == kl && j < lane) ? pj : 0;
        }
        const unsigned long at = __builtin_amdgcn_ballot_w64(fs <= slot && slot < fs + parts);
        l = at ? __builtin_ctzll(at) : 63;  // none: the last lane, whose document has no rows
    } else {
        const int c = __popcll(__builtin_amdgcn_ballot_w64(lo + lane < hi && fs <= slot));
        l = c > 0 ? c - 1 : 0;
    }
    Doc r;
    r.d = lo + l;
    r.q0 = __builtin_amdgcn_readlane(qo, l);
    r.k0 = __builtin_amdgcn_readlane(ko, l);
    r.qlen = max(__builtin_amdgcn_readlane(qo, min(l + 1, 63)) - r.q0, 0);
    r.klen = max(__builtin_amdgcn_readlane(ko, min(l + 1, 63)) - r.k0, 0);
    r.pre = min(max(__builtin_amdgcn_readlane(pr, l), 0), r.klen);
    r.first = __builtin_amdgcn_readlane(fs, l);
    return r;
}

// HD: the head dim, or with GEN the least of 64, 128, 256 that holds it. KT: keys a tile, 64, or 32 where head dim 256
// keeps its registers and LDS at half, and for short documents.
template <int HD, bool GEN, int KT>
struct Tile {
    static constexpr int KB = KT / 32;
    static constexpr int NKS = (HD + 15) / 16;        // k-steps of Q K^T
    static constexpr int NDB = (HD + 31) / 32;        // 32-column blocks of O^T
    // Where a row is a power of two of chunks, columns of rows would meet in the same banks: a chunk's place is XORed
    // with bits of its row and the 1 KiB pieces get a gap, so that the 16 rows of a K read, and the 4 rows of
    // a transposed V read (64 bytes each), take 256 bytes of banks between them. X is the XOR's unit in chunks: the
    // addresses of a lane are one register for each of its NX values (and constants), not one for each k-step.
    static constexpr bool XOR = !GEN && (HD & (HD - 1)) == 0;
    static constexpr int KX = HD == 64 ? 2 : HD == 128 ? 4 : 8, KNX = !XOR ? 1 : HD == 256 ? 2 : 4;
    static constexpr int VX = HD == 256 ? 8 : 4, VNX = !XOR ? 1 : HD == 128 ? 4 : 2;
    static constexpr int KGAP = XOR ? 16 : 0, VGAP = XOR && HD == 256 ? 64 : 0;
    static __device__ __forceinline__ int kx(int row) { return !XOR ? 0 : KX * ((HD == 64 ? row >> 1 : row) & (KNX - 1)); }
    static __device__ __forceinline__ int vx(int row) { return !XOR ? 0 : VX * ((HD == 64 ? row >> 1 : row) & (VNX - 1)); }
    // Head dims 72 and 80 leave columns of O^T free: V's rows in LDS have 12 chunks, which the copies fill up to the head
    // dim; the next holds ones, which sums the weights. 12 chunks put the 4 rows of a transposed read, and an odd number
    // the 16 rows of a K read, into banks of their own.
    static constexpr bool ONES = HD == 72 || HD == 80;
    static constexpr int KP = ONES ? 9 + (HD == 80 ? 2 : 0) : HD / 8, VP = ONES ? 12 : HD / 8;  // chunks a row (not GEN)
    static constexpr int NPK = (KT * KP + 63) / 64, NPV = (KT * VP + 63) / 64;                  // pieces of K, and of V
    static constexpr int VOFF = NPK * (1024 + KGAP);
    static constexpr int BYTES = VOFF + NPV * (1024 + VGAP);
    // where row `row` of K or V begins (rows of a piece are contiguous); nch: chunks a row
    static __device__ __forceinline__ int at(int row, int nch, int gap) {
        return row * nch * 16 + (XOR ? row / (512 / HD) * gap : 0);
    }
};

// One flat row from its own keys alone, [lo, hi) of its document, by one wave: 64 keys a step, a lane each for the
// scores and a lane for each column of V (columns lane + 64 c in acc[c]); m in powers of two, weights not
// rounded. Latency: 0.14 ms for 1 100 keys of 128 (0.45 with one key of V at a time).
template <int HD>
__device__ __forceinline__ void row_alone(const DocsArgs& a, const Doc& D, int gh, int kvh, int pq, int qi, int lo, int hi,
                                       float& m, float& l, float (&acc)[(HD + 63) / 64]) {
    const int lane = threadIdx.x & 63;
    const bf16* q = a.q + (D.q0 + (long)qi) * a.ldq + (long)gh * a.hd;
    const float slope = a.slopes ? a.slopes[gh] * LOG2E : 0.f;
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int c = 0; c < (HD + 63) / 64; ++c) acc[c] = 0.f;
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        float x = -INFINITY;
        if (j < hi) {
            const bf16* k = a.k + (D.k0 + (long)j) * a.ldk + (long)kvh * a.hd;
            float s = 0.f;
#pragma unroll 8
            for (int e = 0; e < a.hd; ++e) s = __builtin_fmaf(bf2f(q[e]), bf2f(k[e]), s);
            if (a.cap_log2 != 0.f)
                x = __builtin_fmaf(-2.0f * a.cap_log2, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s * a.cap_in)), a.cap_log2);
            else
                x = s * a.scale_log2;
            if (a.slopes) x = __builtin_fmaf(-slope, fabsf((float)(pq - j)), x);
        }
        float mx = x;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float p = j < hi ? __builtin_amdgcn_exp2f(x - ref) : 0.f;
        m = mn;
        l = l * alpha + wave_sum(p);
#pragma unroll
        for (int c = 0; c < (HD + 63) / 64; ++c) acc[c] *= alpha;
        const int nj = min(64, hi - j0);
#pragma unroll 1
        for (int jj = 0; jj < nj; jj += 8) {  // eight loads in flight
            float x8[8][(HD + 63) / 64];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const bf16* v = a.v + (D.k0 + (long)j0 + min(jj + u, nj - 1)) * a.ldv + (long)kvh * a.hd;
#pragma unroll
                for (int c = 0; c < (HD + 63) / 64; ++c)
                    x8[u][c] = bf2f(v[min(lane + 64 * c, a.hd - 1)]);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float pj = __shfl(p, jj + u, 64);
#pragma unroll
                for (int c = 0; c < (HD + 63) / 64; ++c)
                    if (jj + u < nj) acc[c] = __builtin_fmaf(pj, x8[u][c], acc[c]);
            }
        }
    }
}

// Whole calls measured beside a matrix product's 1 400 TF/s and a copy's 5.2 TB/s, and what bounds them (MFMA busy: of
// the SIMD cycles of CUs that had waves; of all 256 CUs through the kernel it is 30 / 43 / 53 %):
//   12 pages of 1 030 - 1 100 tokens, 8 heads to 1 of 256, prefix, capped: 142 - 165 us, 0.64 - 0.74 PF/s. 806
//     workgroups over the 512 places that 256 registers leave are two rounds, the second part full; MFMA 38 % busy.
//   14 images of 64 - 2 916 patches, 16 heads of 72: 118 - 126 us, 0.67 - 0.72 PF/s; 72 is padded to 80 and 96 columns, and
//     the softmax's vector instructions share the issue with MFMA (53 % busy).
//   3 texts, the longest 6 143, 32 heads to 8 of 128, causal: 296 - 322 us, 0.96 - 1.05 PF/s; MFMA 59 % busy.
//   256 captions of 5 - 77 tokens, 12 heads of 64, biased: 15 us; a wave's chain of a copy, a product, a softmax.
//   One query against 1 030 keys: 14 us, two launches, latency; 64 against 256 - 4 096 keys, 16 heads of 72: 92 us, 4.4 TB/s;
//     5 against 3 001 - 65 536 keys, 8 key heads of 128: 160 us, 4.8 TB/s.
// MODE: 1 = capped scores, 2 = biased by distance, 3 = both
// AHEAD: the next tile's scores are formed beside this one's weights
template <int HD, bool GEN, int NW, int MINW, bool AHEAD, bool SPLIT, int MODE>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(MINW))) void attn_docs_kernel(DocsArgs a) {
    constexpr int KT = HD > 128 || (NW == 1 && !SPLIT) ? 32 : 64;
    using T = Tile<HD, GEN, KT>;
    constexpr int KB = T::KB, NKS = T::NKS, NDB = T::NDB, QB = NW * 32;
    constexpr bool HALF = GEN || HD % 16 != 0;  // the last k-step may reach past the head dim
    constexpr int ZERO = 2 * T::BYTES;           // 16 zero bytes for it
    __shared__ __attribute__((aligned(16))) char lds[2 * T::BYTES + (HALF ? 16 : 0)];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, hh = lane >> 5;
    // Workgroups go round the 8 XCDs. Where the K / V of a slot are its own, the key heads go side by side, as their
    // rows lie in shared lines; else an XCD keeps to as few key heads as it can, whose K / V its slots share, and takes
    // their slots side by side, so that all heads' first slots (the longest, where they are sorted) start first.
    constexpr bool OWN = SPLIT || NW == 1;
    int slot, kvh, rb = 0;
    {
        const int bid = blockIdx.x, nwg = gridDim.x;
        const int xcd = bid & 7, loc = bid >> 3, q8 = nwg >> 3, r8 = nwg & 7;
        const int id = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + loc;
        if constexpr (OWN) {
            const int x = SPLIT ? id / a.row_blocks : id;  // split: the blocks of rows of one chunk side by side too
            rb = id - x * (SPLIT ? a.row_blocks : 1), slot = x / a.Hkv, kvh = x - slot * a.Hkv;
        } else if ((a.Hkv & 7) == 0) {
            slot = loc / (a.Hkv >> 3), kvh = xcd * (a.Hkv >> 3) + loc - slot * (a.Hkv >> 3);
        } else {
            kvh = id / a.nslots, slot = id - kvh * a.nslots;
        }
    }
    const Doc D = find_doc<SPLIT, !OWN>(a, slot);
    const int qlen = D.qlen, klen = D.klen;
    const int flat = min(qlen, a.max_rows) * a.group;  // flat rows of this document
    int part = slot - D.first;
    const int nparts = (int)(((unsigned)(SPLIT ? klen : flat) + (unsigned)a.per - 1) / (unsigned)a.per);
    if (part < 0 || part >= nparts || flat == 0) return;
    if (!SPLIT && a.causal) part = nparts - 1 - part;  // the rows with the most keys first

    const int f0 = SPLIT ? rb * QB : part * QB;                 // the block's first flat row
    if (SPLIT && f0 >= flat) return;
    const int fr = f0 + wave * 32 + r;                          // this lane's
    const int qi = min(fr, flat - 1) / a.group, gh = kvh * a.group + min(fr, flat - 1) - qi * a.group;
    const int pq = qi + klen - qlen;                            // its place among the keys
    const int hi = a.causal ? min(klen, max(D.pre, pq + 1)) : klen;  // it sees keys [0, hi)
    const int key_lo = SPLIT ? part * a.per : 0;
    // the block's first row sees the fewest keys, its last row the most
    const int q_first = f0 / a.group, q_last = (min(f0 + QB, flat) - 1) / a.group;
    int hi_min = a.causal ? min(klen, max(D.pre, q_first + klen - qlen + 1)) : klen;
    int hi_max = a.causal ? min(klen, max(D.pre, q_last + klen - qlen + 1)) : klen;
    if (SPLIT) {
        hi_min = min((long)hi_min, (long)key_lo + a.per);
        hi_max = min((long)hi_max, (long)key_lo + a.per);
    }
    const int nfull = (hi_min - key_lo) / KT;  // tiles that every row sees whole (none where negative)
    const int nkt = hi_max > key_lo ? (hi_max - key_lo + KT - 1) / KT : 0;

    const int nch = GEN ? a.hd >> 3 : HD / 8;                               // 16-byte chunks of a row
    const int kp = GEN ? nch : T::KP, vp = GEN ? nch : T::VP;               // and between rows in LDS
    if (HALF && tid == 0) *reinterpret_cast<u16x8*>(lds + ZERO) = u16x8{0, 0, 0, 0, 0, 0, 0, 0};

    const unsigned lds0 = (unsigned)(uintptr_t)(LDS_AS char*)lds;
    const char* kbase = (const char*)(a.k + (D.k0 + (long)key_lo) * a.ldk + (long)kvh * a.hd);
    const char* vbase = (const char*)(a.v + (D.k0 + (long)key_lo) * a.ldv + (long)kvh * a.hd);
    // a tile of K (V) is kp (vp) * KT / 64 pieces; piece p: LDS chunks 64 p .. + 63, chunk c of row (64 p + lane) / kp.
    // A lane's places in them are the same in every tile but one that reaches past the document.
    const int npk = GEN ? (nch * KT + 63) / 64 : T::NPK, npv = GEN ? npk : T::NPV;
    if (T::ONES)
        for (int i = tid; i < 2 * KT; i += NW * 64)
            *reinterpret_cast<u16x8*>(lds + i / KT * T::BYTES + T::VOFF + (i % KT * T::VP + HD / 8) * 16) =
                u16x8{0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80};
    auto row_of = [&](bool isV, int i) __attribute__((always_inline)) { return ((wave + NW * i) * 64 + lane) / (isV ? vp : kp); };
    auto chunk_of = [&](bool isV, int i) __attribute__((always_inline)) { return ((wave + NW * i) * 64 + lane) % (isV ? vp : kp); };
    auto place = [&](bool isV, int i, int most) __attribute__((always_inline)) {
        const int row = row_of(isV, i), ch = chunk_of(isV, i);
        return isV ? (unsigned)min(row, most) * (unsigned)(2 * a.ldv) + (ch ^ T::vx(row)) * 16
                   : (unsigned)min(row, most) * (unsigned)(2 * a.ldk) + (ch ^ T::kx(row)) * 16;
    };
    constexpr int PK = (T::NPK + NW - 1) / NW, PV = (T::NPV + NW - 1) / NW;
    // no chunk to leave out: behind a row's data, or behind the tile in a last piece that is half one
    constexpr bool KFULL = GEN ? KT == 64 : T::KP == HD / 8 && KT * T::KP % 64 == 0;
    constexpr bool VFULL = GEN ? KT == 64 : T::VP == HD / 8 && KT * T::VP % 64 == 0;
    auto has = [&](bool isV, int i) __attribute__((always_inline)) { return chunk_of(isV, i) < nch && row_of(isV, i) < KT; };
    unsigned atk[PK], atv[PV];
    bool dok[PK], dov[PV];
#pragma unroll
    for (int i = 0; i < PK; ++i) atk[i] = place(false, i, KT), dok[i] = has(false, i);
#pragma unroll
    for (int i = 0; i < PV; ++i) atv[i] = place(true, i, KT), dov[i] = has(true, i);
    auto issue = [&](auto v_c, int t, unsigned slot) __attribute__((always_inline)) {
        constexpr bool isV = decltype(v_c)::value;
        const char* base = isV ? vbase + (long)t * KT * 2 * a.ldv : kbase + (long)t * KT * 2 * a.ldk;
        const unsigned to = lds0 + (isV ? T::VOFF : 0) + slot, pitch = 1024 + (isV ? T::VGAP : T::KGAP);
        const int most = klen - 1 - key_lo - t * KT, np = isV ? npv : npk;
        if (most >= KT - 1) {
#pragma unroll
            for (int i = 0; i < (isV ? PV : PK); ++i)
                if (wave + NW * i < np && ((isV ? VFULL : KFULL) || (isV ? dov[i] : dok[i])))
                    dma16(base, isV ? atv[i] : atk[i], to + (wave + NW * i) * pitch);
        } else {
#pragma unroll 1
            for (int i = 0; wave + NW * i < np; ++i) {
                const unsigned piece = to + (wave + NW * i) * pitch;
                if (!(isV ? VFULL : KFULL) && !has(isV, i)) continue;
                if (isV && row_of(isV, i) > most)  // behind the document: what its weight 0 makes nothing of
                    *reinterpret_cast<LDS_AS u32x4*>((uintptr_t)(piece + lane * 16)) = u32x4{0, 0, 0, 0};
                else
                    dma16(base, place(isV, i, most), piece);
            }
        }
    };
    if (nkt > 0) issue(std::false_type{}, 0, 0);

    bf16x8 qf[NKS];  // B operand: Q^T[16 ks + 8 hh + j][row r]
    {
        const bf16* qrow = a.q + (D.q0 + (long)qi) * a.ldq + (long)gh * a.hd;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
            qf[ks] = HALF ? __builtin_bit_cast(bf16x8, load_chunk_or_zero(qrow, 2 * ks + hh, nch))
                          : *reinterpret_cast<const bf16x8*>(qrow + (2 * ks + hh) * 8);
    }
    const float slope = MODE & 2 ? a.slopes[gh] * LOG2E : 0.f;
    const float c = MODE ? 1.0f : a.scale_log2;  // what a score is still multiplied by

    unsigned ka[T::KNX];
#pragma unroll
    for (int g = 0; g < T::KNX; ++g) ka[g] = lds0 + T::at(r, kp, T::KGAP) + (((g * T::KX) ^ T::kx(r)) + hh) * 16;
    auto kfrag = [&](unsigned so, int kb, int ks) __attribute__((always_inline)) {
        constexpr int U = T::KX / 2, W = T::KNX * U;  // k-steps a unit, and all units
        unsigned at = (T::XOR ? ka[ks / U % T::KNX] + (ks % U + ks / W * W) * 32 : ka[0] + ks * 32) + so +
                      kb * T::at(32, kp, T::KGAP);
        if (HALF && (GEN || ks == NKS - 1)) at = 2 * ks + hh < nch ? at : lds0 + ZERO;
        return *reinterpret_cast<const LDS_AS bf16x8*>((uintptr_t)at);
    };
    // V^T fragment of key step i: two transposed reads, keys 16 i + 8 j + 4 hh + q at columns 32 db + 16 half + 4 p ..
    unsigned va[T::VNX];
    {
        const int i16 = lane & 15, q = i16 >> 2, p = i16 & 3, half = (lane >> 4) & 1;
#pragma unroll
        for (int g = 0; g < T::VNX; ++g)
            va[g] = lds0 + T::VOFF + T::at(4 * hh + q, vp, T::VGAP) + (((g * T::VX) ^ T::vx(q)) + 2 * half + (p >> 1)) * 16 +
                    (p & 1) * 8;
    }
    auto vfrag = [&](unsigned so, int i, int db) __attribute__((always_inline)) {
        constexpr int U = T::VX / 4, W = T::VNX * U;
        const unsigned at = (T::XOR ? va[db / U % T::VNX] + (db % U + db / W * W) * 64 : va[0] + db * 64) + so +
                            i * T::at(16, vp, T::VGAP);
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(uintptr_t)at);
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(uintptr_t)(at + T::at(8, vp, T::VGAP)));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    f32x16 o[NDB];
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, lsum = 0.f;

    float mc = 0.f, cf = c;  // a weight is 2^(cf score - mc)
    f32x16 sa[KB], sb[KB];

    auto qk = [&](f32x16(&sc)[KB], const unsigned so) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 z;
#pragma unroll
            for (int e = 0; e < 16; ++e) z[e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
                if (!GEN || 2 * ks < nch) z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kfrag(so, kb, ks), qf[ks], z, 0, 0, 0);
            sc[kb] = z;
        }
        if (!GEN) {  // reads four ahead of the products that take them
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int x = 0; x < KB * NKS - 4; ++x) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
        }
    };
    // register e of block kb scores key key0 + 32 kb + (e & 3) + 8 (e >> 2) + 4 hh; CUT: some row may not see all keys
    auto score = [&](auto cut_c, f32x16(&sc)[KB], int t) __attribute__((always_inline)) {
        constexpr bool CUT = decltype(cut_c)::value;
        const int key0 = key_lo + t * KT;
        if (MODE & 1) {
            // cap tanh(x / cap) = cap - 2 cap / (1 + e^(2 x / cap)), log2(e) folded in: the exponential and reciprocal
            // units' errors and the difference are worth 3 steps of the cap (4e-4 at a cap of 1 000, 2e-5 at 50)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float w = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sc[kb][e] * a.cap_in));
                    sc[kb][e] = __builtin_fmaf(-2.0f * a.cap_log2, w, a.cap_log2);
                }
        } else if (MODE & 2) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[kb][e] *= a.scale_log2;
        }
        if (MODE & 2) {
            const float db = (float)(pq - key0 - 4 * hh);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    sc[kb][e] = __builtin_fmaf(-slope, fabsf(db - (float)(32 * kb + (e & 3) + 8 * (e >> 2))), sc[kb][e]);
        }
        if (CUT) {
            const int lim = hi - key0 - 4 * hh;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * kb + (e & 3) + 8 * (e >> 2) >= lim) sc[kb][e] = -INFINITY;
        }
    };
    auto largest = [&](const f32x16(&sc)[KB]) __attribute__((always_inline)) {
        float x = sc[0][0];  // (a NaN among them stays: the row is NaN)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) x = __builtin_elementwise_maximum(x, sc[kb][e]);
        return xmax32(x);
    };
    // the running maximum takes in a tile's; O and the sum follow only where some row's grew by more than 2^8
    auto raise = [&](float mloc, f32x16(&sc)[KB]) __attribute__((always_inline)) {
        if (__builtin_amdgcn_ballot_w64((mloc - m) * c > 8.0f)) {
            const float mnew = fmaxf(m, mloc);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mnew) * c);
            if (!T::ONES) lsum *= alpha;
#pragma unroll
            for (int i = 0; i < NDB; ++i) o[i] *= alpha;
            m = mnew;
            mc = m == -INFINITY ? 0.f : m * c;
        }
        if (__builtin_amdgcn_ballot_w64(fabsf(mc) > 0x1p20f)) {
            // m c is rounded, s c inside the fused exponent is not: where that alone is worth whole powers of two,
            // round both
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[kb][e] *= c;
            cf = 1.0f;
        } else {
            cf = c;
        }
    };
    auto weigh = [&](const f32x16(&sc)[KB], bf16x8(&pk)[2 * KB]) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                pk[2 * kb + (e >> 3)][e & 7] = f2bf(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][e], cf, -mc)));
        // the rounded weights are summed: where one weight is nearly all, its rounding divides out
#pragma unroll
        for (int i = 0; i < (T::ONES ? 0 : 2 * KB); ++i) {
            const bf16x2 one = {1.0f, 1.0f};
            lsum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(pk[i], pk[i], 0, 1), one, lsum, false);
            lsum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(pk[i], pk[i], 2, 3), one, lsum, false);
            lsum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(pk[i], pk[i], 4, 5), one, lsum, false);
            lsum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(pk[i], pk[i], 6, 7), one, lsum, false);
        }
    };
    auto pv = [&](const bf16x8(&pk)[2 * KB], const unsigned so) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
            for (int db = 0; db < NDB; ++db)
                o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vfrag(so, i, db), pk[i], o[db], 0, 0, 0);
        if (!GEN) {  // and three
            __builtin_amdgcn_sched_group_barrier(0x100, 6, 1);
#pragma unroll
            for (int x = 0; x < 2 * KB * NDB - 3; ++x) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 3, 1);
        }
    };
    // this wave's part of the next tile has landed and its LDS reads are done; then everybody's
    auto meet = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    constexpr std::false_type K{}, WHOLE{};
    constexpr std::true_type V{}, CUT{};
    int t = 0;
    unsigned now = 0, other = T::BYTES;  // tile t's slot, and the other
    if (nkt > 0) {
        if (!AHEAD) issue(V, 0, 0);
        auto turn = [&]() __attribute__((always_inline)) {
            const unsigned x = now;
            now = other, other = x, ++t;
        };
        if constexpr (!AHEAD) {
            auto step = [&](auto cut_c) __attribute__((always_inline)) {
                meet();
                if (t + 1 < nkt) issue(K, t + 1, other), issue(V, t + 1, other);
                bf16x8 pk[2 * KB];
                qk(sa, now);
                score(cut_c, sa, t);
                raise(largest(sa), sa);
                weigh(sa, pk);
                pv(pk, now);
                turn();
            };
#pragma unroll 1
            while (t < nfull) step(WHOLE);
#pragma unroll 1
            while (t < nkt) step(CUT);
        } else {
            // Tile t's weights and products beside tile t + 1's scores, which do not depend on them: the matrix pipe
            // has work while the wave's vector instructions run. K runs one tile ahead of V.
            auto step = [&](auto cut_c, f32x16(&s0)[KB], f32x16(&s1)[KB]) __attribute__((always_inline)) {
                const bool more = !decltype(cut_c)::value || t + 1 < nkt;
                meet();
                if (t + 2 < nkt) issue(K, t + 2, now);
                if (t + 1 < nkt) issue(V, t + 1, other);
                bf16x8 pk[2 * KB];
                if (more) qk(s1, other);
                weigh(s0, pk);
                pv(pk, now);
                if (more) {
                    score(cut_c, s1, t + 1);
                    raise(largest(s1), s1);
                }
                turn();
            };
            meet();
            if (nkt > 1) issue(K, 1, other);
            issue(V, 0, 0);
            qk(sa, 0);
            score(CUT, sa, 0);
            raise(largest(sa), sa);
#pragma unroll 1
            while (t + 2 < nfull) {
                step(WHOLE, sa, sb);
                step(WHOLE, sb, sa);
            }
#pragma unroll 1
            while (t < nkt) {
                step(CUT, sa, sb);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) sa[kb] = sb[kb];
            }
        }
    }

    const float l = T::ONES ? o[HD / 32][4 * (HD % 32 / 8)] : xsum32(lsum);
    const float inv = hi > 0 ? 1.0f / l : 0.f;  // a row that sees nothing is 0
    if constexpr (SPLIT) {
        if (fr < flat) {
            const long at = ((long)slot * a.Hkv + kvh) * a.part_rows + fr;
            if (hh == 0) *reinterpret_cast<float2*>(a.stat + 2 * at) = make_float2(m * c, l);
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int mm = 0; mm < 4; ++mm) {
                    const int d0 = 32 * db + 8 * mm + 4 * hh;
                    if (d0 < a.hd)
                        *reinterpret_cast<float4*>(a.part + at * a.hd + d0) =
                            make_float4(o[db][4 * mm], o[db][4 * mm + 1], o[db][4 * mm + 2], o[db][4 * mm + 3]);
                }
        }
    } else {
        bf16* orow = a.out + (D.q0 + (long)qi) * a.ldo + (long)gh * a.hd;
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
    if (!a.causal) return;  // all rows saw the same keys

    float nan = 0.f;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (32 * db + 8 * (e >> 2) < (GEN ? a.hd : HD)) nan = __builtin_fmaf(o[db][e], 0.f, nan);
    unsigned long bad = __builtin_amdgcn_ballot_w64(fr < flat && nan != 0.f);
    bad = (bad | bad >> 32) & 0xffffffffu;
    if (bad == 0) return;
    // keys that the block's tiles had and some of this wave's rows do not see: does V hold an infinity or NaN there?
    bool found = false;
    {
        int least = hi;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) least = min(least, __shfl_xor(least, x, 64));
        const int end = (int)min((long)klen, key_lo + (long)nkt * KT);
        for (int j = max(least, key_lo); j < end; ++j) {
            const bf16* v = a.v + (D.k0 + (long)j) * a.ldv + (long)kvh * a.hd;
            for (int e = lane; e < a.hd; e += 64) found |= !(fabsf(bf2f(v[e])) < INFINITY);
        }
    }
    if (__builtin_amdgcn_ballot_w64(found) == 0) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows' first stores come before their second
    for (int x = 0; x < 32; ++x) {
        if (!(bad >> x & 1)) continue;
        const int fx = f0 + wave * 32 + x, qx = fx / a.group, gx = kvh * a.group + fx - qx * a.group, px = qx + klen - qlen;
        const int hx = min(klen, max(D.pre, px + 1));
        float mx, lx, acc[(HD + 63) / 64];
        row_alone<HD>(a, D, gx, kvh, px, qx, key_lo, SPLIT ? (int)min((long)hx, (long)key_lo + a.per) : hx, mx, lx, acc);
        const long at = ((long)slot * a.Hkv + kvh) * a.part_rows + fx;
        if (SPLIT && lane == 0) a.stat[2 * at] = mx, a.stat[2 * at + 1] = lx;
#pragma unroll
        for (int cc = 0; cc < (HD + 63) / 64; ++cc) {
            const int e = lane + 64 * cc;
            if (e >= a.hd) continue;
            if (SPLIT)
                a.part[at * a.hd + e] = acc[cc];
            else
                a.out[(D.q0 + (long)qx) * a.ldo + (long)gx * a.hd + e] = f2bf(hx > 0 ? acc[cc] / lx : 0.f);
        }
    }
}

// Joins a document's chunks: one workgroup a (document, flat row, key head), a thread four columns of every SG-th
// chunk, the chunks' factors 2^(m_s - max m) in LDS. Latency: it reads a few MB at most; 3.9 us for 8 rows of 33 chunks, 6.4
// us for 160 rows of up to 61 (a workgroup a row keeps all of a row's loads in flight).
__global__ __launch_bounds__(256) void join_docs_kernel(DocsArgs a) {
    __shared__ float wide[4], w[256], sums[4 * 256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int fr = (int)(blockIdx.x % a.part_rows), kvh = (int)(blockIdx.x / a.part_rows % a.Hkv);
    const int d = (int)(blockIdx.x / a.part_rows / a.Hkv);
    const int q0 = clamp_row(a.qoff[d], a.rows_q), k0 = clamp_row(a.koff[d], a.rows_k);
    const int qlen = max(clamp_row(a.qoff[d + 1], a.rows_q) - q0, 0), klen = max(clamp_row(a.koff[d + 1], a.rows_k) - k0, 0);
    if (fr >= min(qlen, a.max_rows) * a.group) return;
    const int qi = fr / a.group, gh = kvh * a.group + fr % a.group;
    const int pre = a.prefix ? min(max(a.prefix[d], 0), klen) : 0;
    const int hi = a.causal ? min(klen, max(pre, qi + klen - qlen + 1)) : klen;
    const int nparts = (int)(((unsigned)klen + (unsigned)a.per - 1) / (unsigned)a.per);
    const long row = ((long)first_slot(k0, d, 1, a.per) * a.Hkv + kvh) * a.part_rows + fr;
    const long step = (long)a.Hkv * a.part_rows;
    const float2* stat = reinterpret_cast<const float2*>(a.stat) + row;
    float m = -INFINITY;
    for (int s = tid; s < nparts; s += 256) m = fmaxf(m, stat[s * step].x);
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
    if (lane == 0) wide[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(wide[0], wide[1]), fmaxf(wide[2], wide[3]));
    const float mr = m == -INFINITY ? 0.f : m;
    const int C4 = a.hd >> 2, SG = 256 / C4, col = tid % C4, sg = tid / C4;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int s0 = 0; s0 < nparts; s0 += 256) {
        const int ns = min(256, nparts - s0);
        __syncthreads();
        if (tid < ns) {
            const float2 st = stat[(s0 + tid) * step];
            w[tid] = __builtin_amdgcn_exp2f(st.x - mr);
            l = __builtin_fmaf(w[tid], st.y, l);
        }
        __syncthreads();
        if (sg < SG) {
            const float* p = a.part + (row + s0 * step) * a.hd + 4 * col;
#pragma unroll 4
            for (int s = sg; s < ns; s += SG) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(p + s * step * a.hd);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(w[s], v[e], acc[e]);
            }
        }
    }
    l = wave_sum(l);
    __syncthreads();
    if (lane == 0) wide[wave] = l;
    if (sg < SG) *reinterpret_cast<f32x4*>(sums + 4 * tid) = acc;  // [sg][column]
    __syncthreads();
    const float inv = hi > 0 ? 1.0f / ((wide[0] + wide[1]) + (wide[2] + wide[3])) : 0.f;
    if (tid < a.hd) {
        float o = 0.f;
        for (int s = 0; s < SG; ++s) o += sums[s * a.hd + tid];
        a.out[(q0 + (long)qi) * a.ldo + (long)gh * a.hd + tid] = f2bf(hi > 0 ? o * inv : 0.f);
    }
}

struct Plan {
    bool split;
    int NW, per, part_rows, row_blocks;
    long nslots;
    size_t stat, ws;
};

// How the work is cut, from the sizes alone (the lengths are on the device).
Plan make_plan(int n, int rows_q, int rows_k, int Hkv, int group, int hd, int max_rows) {
    Plan p{};
    if (n == 0 || max_rows == 0) return p;
    const long flat = (long)rows_q * group, keys = (long)rows_k / n;
    // One wave a workgroup (and tiles of 32 keys, so that many fit a CU) for short documents, where there are workgroups
    // enough; else four, which share the tiles and the copying. 12 000 rows in documents of 48 / 128 / 256 rows, 12
    // heads of 64: one wave 20 / 22 / 28 us, four 24 / 25 / 31; documents of 12 / 32 / 64 rows, 4 heads of 128 to each of
    // 8 key heads, 92 / 72 / 86 and 121 / 98 / 62.
    p.NW = hd <= 128 && (flat / n <= 32 || (flat / n <= 128 && keys <= 256)) && (flat / 32 + n) * Hkv >= 512 ? 1 : 4;
    p.per = p.NW * 32;
    p.row_blocks = 1;
    long nslots = flat / p.per + n;
    // Few flat rows a document: its keys in parts. The bound of 256 keeps the workspace small and is not a measured
    // optimum: beyond it the keys stay whole, and few such documents leave most CUs idle (8 heads to 1 of 256 against
    // 65 536 keys: 32 queries 95 us in parts, 33 queries 4.6 ms whole).
    // As many parts as make nearly three rounds of the workgroups that fit the device by their LDS (documents of
    // different lengths at just over two rounds 195 us, at 2.7 157: the last is half empty).
    // Two parts at least, and enough for a workgroup to read without: one query against 512 / 1 024 / 4 096 keys of 8
    // documents, 8 heads of 128, whole 14.9 / 23 / 81 us, in parts 14.7 / 17 / 43; 16 documents, 16 heads of 72, 1 024 /
    // 4 096 keys 21 / 85 and 25 / 71 (more workgroups need longer documents). Documents of 1 353 keys on average, 256
    // to 4 096, 64 x 16 heads of 72: 119 and 100 us.
    const long mr = (long)max_rows * group, rb = (mr + 31) / 32, blocks = nslots * Hkv;
    const long resident = 256 * (hd <= 64 ? 4 : hd <= 80 ? 3 : 2);
    const long parts = mr <= 256 ? resident * 11 / 4 / ((long)n * Hkv * rb) : 0;
    if (parts >= 2 && keys * hd >= (blocks <= 128 ? 40960 : 81920)) {
        p.split = true;
        p.NW = 1;
        const long kt = hd > 128 ? 32 : 64;  // keys a tile
        p.per = (int)((keys + parts * kt - 1) / (parts * kt) * kt);
        p.part_rows = (int)mr, p.row_blocks = (int)rb;
        nslots = (long)rows_k / p.per + n;
        p.stat = (size_t)nslots * Hkv * mr * hd;  // where the statistics begin, in floats
        p.ws = (p.stat + (size_t)nslots * Hkv * mr * 2) * 4;
    }
    p.nslots = nslots;
    return p;
}

template <int HD, bool GEN, int NW, int MINW, bool AHEAD, bool SPLIT>
void launch_docs(const DocsArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.nslots * a.Hkv * a.row_blocks)), block(NW * 64);
    switch ((a.cap_log2 != 0.f ? 1 : 0) | (a.slopes ? 2 : 0)) {
        case 0: hipLaunchKernelGGL((attn_docs_kernel<HD, GEN, NW, MINW, AHEAD, SPLIT, 0>), grid, block, 0, s, a); break;
        case 1: hipLaunchKernelGGL((attn_docs_kernel<HD, GEN, NW, MINW, AHEAD, SPLIT, 1>), grid, block, 0, s, a); break;
        case 2: hipLaunchKernelGGL((attn_docs_kernel<HD, GEN, NW, MINW, AHEAD, SPLIT, 2>), grid, block, 0, s, a); break;
        default: hipLaunchKernelGGL((attn_docs_kernel<HD, GEN, NW, MINW, AHEAD, SPLIT, 3>), grid, block, 0, s, a);
    }
}

template <int HD, bool GEN, int MINW, bool AHEAD>
void launch_width(const DocsArgs& a, const Plan& p, hipStream_t s) {
    if (p.split) return launch_docs<HD, GEN, 1, 1, false, true>(a, s);
    if constexpr (HD <= 128) {
        if (p.NW == 1) return launch_docs<HD, GEN, 1, HD <= 80 ? 2 : 1, false, false>(a, s);
    }
    launch_docs<HD, GEN, 4, MINW, AHEAD, false>(a, s);
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
    MME_REQUIRE(softcap == 0.f || (softcap >= 1e-3f && softcap <= 1e3f), "mme_attention_docs: softcap must be 0 (none) or from 1e-3 to 1e3");
    const float scale_log2 = scale * LOG2E, cap_in = softcap != 0.f ? 2.0f * scale_log2 / softcap : 0.f;
    MME_REQUIRE(scale_log2 < INFINITY && cap_in < INFINITY, "mme_attention_docs: scale too large (%g, softcap %g)", scale, softcap);
    MME_REQUIRE(causal || !prefix, "mme_attention_docs: a prefix goes with the causal mask");
    if (n == 0 || rows_q == 0) return MME_OK;
    MME_REQUIRE(q && out && q_offsets && k_offsets && (rows_k == 0 || (k && v)), "mme_attention_docs: null pointer");
    MME_REQUIRE(ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldo % 8 == 0 && ldq >= (long)Hq * hd &&
                    ldo >= (long)Hq * hd && ldk >= (long)Hkv * hd && ldv >= (long)Hkv * hd,
                "mme_attention_docs: bad leading dims");
    MME_REQUIRE(ldk < (1L << 24) && ldv < (1L << 24), "mme_attention_docs: leading dims of k and v must be under 2^24");
    MME_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0 &&
                    (((uintptr_t)q_offsets | (uintptr_t)k_offsets | (uintptr_t)prefix | (uintptr_t)slopes) & 3) == 0,
                "mme_attention_docs: misaligned pointer");
    const int mr = max_rows < rows_q ? max_rows : rows_q;
    if (mr == 0) return MME_OK;
    const Plan p = make_plan(n, rows_q, rows_k, Hkv, Hq / Hkv, hd, mr);
    // a launch has under 2^32 threads
    MME_REQUIRE(p.nslots * Hkv * p.row_blocks * p.NW < (1L << 26) && (long)n * Hkv * p.part_rows < (1L << 24) &&
                    (long)rows_q * (Hq / Hkv) < (1L << 31) - 512 && rows_k < 0x7fff0000,
                "mme_attention_docs: too many rows");
    MME_REQUIRE(p.ws == 0 || (workspace && ws_bytes >= p.ws && ((uintptr_t)workspace & 15) == 0),
                "mme_attention_docs: workspace of %zu bytes, %zu needed", ws_bytes, p.ws);
    const long wq = (long)Hq * hd, wk = (long)Hkv * hd;
    MME_REQUIRE(!mme_rows_overlap(out, ldo, rows_q, wq, q, ldq, rows_q, wq) &&
                    !mme_rows_overlap(out, ldo, rows_q, wq, k, ldk, rows_k, wk) &&
                    !mme_rows_overlap(out, ldo, rows_q, wq, v, ldv, rows_k, wk),
                "mme_attention_docs: out overlaps q, k or v");
    DocsArgs a{};
    a.q = (const bf16*)q, a.k = (const bf16*)k, a.v = (const bf16*)v, a.out = (bf16*)out;
    a.qoff = q_offsets, a.koff = k_offsets, a.prefix = prefix, a.slopes = slopes, a.part = (float*)workspace, a.stat = a.part + p.stat;
    a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo, a.nslots = (int)p.nslots;
    a.n = n, a.rows_q = rows_q, a.rows_k = rows_k, a.Hkv = Hkv, a.group = Hq / Hkv, a.hd = hd;
    a.sorted = !p.split && n > 1 && n <= 63 && p.nslots * Hkv >= 512;
    a.max_rows = mr, a.causal = causal ? 1 : 0, a.per = p.per, a.part_rows = p.part_rows, a.row_blocks = p.row_blocks;
    a.scale_log2 = scale_log2;
    a.cap_log2 = softcap * LOG2E;
    a.cap_in = cap_in;
    hipStream_t s = as_stream(stream);
    switch (hd) {
        case 64: launch_width<64, false, 3, false>(a, p, s); break;
        case 72: launch_width<72, false, 3, false>(a, p, s); break;
        case 80: launch_width<80, false, 3, false>(a, p, s); break;
        case 128: launch_width<128, false, 2, true>(a, p, s); break;
        case 256: launch_width<256, false, 2, false>(a, p, s); break;
        default:
            if (hd < 64)
                launch_width<64, true, 3, false>(a, p, s);
            else if (hd < 128)
                launch_width<128, true, 2, false>(a, p, s);
            else
                launch_width<256, true, 1, false>(a, p, s);
    }
    if (p.split) {
        if (int rc = mme_check_launch("mme_attention_docs")) return rc;
        hipLaunchKernelGGL(join_docs_kernel, dim3((unsigned)((long)n * Hkv * p.part_rows)), dim3(256), 0, s, a);
    }
    return mme_check_launch("mme_attention_docs");
}
