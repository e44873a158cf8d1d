// kr_kv_dev.h -- device helpers of the paged-cache operators: page lookup, page formats, visibility, the search for a workgroup's sequence.
#pragma once
#include "kr_device.h"
#include "kr_kv.h"

typedef __bf16 kv_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 kv_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 kv_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv_h8 __attribute__((ext_vector_type(8)));
typedef float kv_f4 __attribute__((ext_vector_type(4)));
typedef float kv_f16 __attribute__((ext_vector_type(16)));

// x / d for 0 <= x < 2^32 with the d's floor(2^32 / d), at most 2^32 - 1: the high product is short by at most one
__host__ __device__ __forceinline__ uint32_t kv_div(uint32_t x, KvDiv d, uint32_t& rest) {
    uint32_t n = (uint32_t)(((uint64_t)x * d.magic) >> 32);
    rest = x - n * d.d;
    if (rest >= d.d) { n++; rest -= d.d; }
    return n;
}
__host__ __device__ __forceinline__ uint32_t kv_div(uint32_t x, KvDiv d) { uint32_t rest; return kv_div(x, d, rest); }
__device__ __forceinline__ uint32_t kv_page(const KvPages& p, uint32_t j, uint32_t& off) { return kv_div(j, p.page, off); }

// two neighbouring codes of a dword times the scale as a packed pair of bf16.  E4M3 and E2M1 have at most four significant bits and scales are powers of two of at least 2^-100:
// every product is exact in bf16.
template <int FMT, int SEL> __device__ __forceinline__ uint32_t kv_pair(uint32_t w, float scale) {
    if constexpr (FMT == 1) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, SEL != 0));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
// the conversions take the scale's exponent field, of which 255 is NaN for any code (measured): the byte needs no case of its own
__device__ __forceinline__ float kv_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

template <bool H> __device__ __forceinline__ uint32_t kv_pack(float a, float b) {      // round to nearest even
    if constexpr (H) { kv_h2 x; x[0] = (_Float16)a; x[1] = (_Float16)b; return __builtin_bit_cast(uint32_t, x); }
    else { kv_b2 x; x[0] = (__bf16)a; x[1] = (__bf16)b; return __builtin_bit_cast(uint32_t, x); }
}
__device__ __forceinline__ kv_h2 kv_halves(uint32_t w) { return __builtin_bit_cast(kv_h2, w); }      // by value: a bit cast of a vector's element takes the vector's first
__device__ __forceinline__ float kv_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float kv_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
// the sum of a packed pair and c, in 32 bits
template <bool H> __device__ __forceinline__ float kv_sum2(uint32_t w, float c) {
    if constexpr (H) return __builtin_amdgcn_fdot2(__builtin_bit_cast(kv_h2, w), __builtin_bit_cast(kv_h2, 0x3C003C00u), c, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(kv_b2, w), __builtin_bit_cast(kv_b2, 0x3F803F80u), c, false);
}
// what a packed pair of bf16 leaves of two floats
__device__ __forceinline__ uint32_t kv_rest(float a, float b, uint32_t w) { return kv_pack<false>(a - kv_lo(w), b - kv_hi(w)); }

// ancestors of the drafts of one sequence, lane i: bit j set when draft j is draft i or an ancestor.  Parents are doubled up: after k rounds a lane knows 2^k ancestors.
// par: the parent of draft `lane`; one that is no earlier draft counts as none.
__device__ __forceinline__ uint64_t kv_ancestors(int par, int lane) {
    if (par >= lane || par < 0) par = -1;
    uint64_t seen = 1ull << lane;
    for (int r = 0; r < 6 && __any(par >= 0); r++) {
        const int from = par < 0 ? lane : par;
        const uint32_t lo = __shfl((uint32_t)seen, from), hi = __shfl((uint32_t)(seen >> 32), from);
        const int up = __shfl(par, from);
        if (par >= 0) { seen |= (uint64_t)hi << 32 | lo; par = up; }
    }
    return seen;
}

// inclusive sum over the lanes
__device__ __forceinline__ int kv_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);      // one, two, four, eight lanes up within rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);     // row 0's sum to row 1, row 2's to row 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);     // the first half's to the second
    return x;
}

struct KvItem { int b, rt, split, kvh, nsplit, len, cnt, row0, page0, base, row_tiles; };      // base: the sequence's first item
// item -> sequence, row tile, share of the keys, head.  A lane counts the items of one sequence, 64 sequences at a time; heads lie side by side (they read the same lines of scales),
// the last row tiles first (a prompt's last rows see the most keys).  In a launch over row tiles alone (SHARES false) each has `sub` parts.
template <bool SHARES> __device__ __forceinline__ KvItem kv_item(const KvAttnArgs& a, int idx, int bm, int kt, KvDiv sub) {
    const int lane = threadIdx.x & 63;
    KvItem it;
    int base = 0, ibase = 0;
    for (int b0 = 0; b0 < a.s.batch; b0 += 64) {
        const int b = b0 + lane;
        int n = 0, full = 0, len = 0, cnt = 0, ns = 1, row0 = 0, page0 = 0, rts = 0;
        if (b < a.s.batch) {
            row0 = a.s.row0[b]; cnt = a.s.row0[b + 1] - row0; len = a.s.lens[b]; page0 = a.s.page0[b];
            const int rows = cnt * (int)a.G.d;
            if (rows >= a.min_rows && rows <= a.max_rows) {
                ns = (int)kv_div((uint32_t)(kv_tiles_ub(len, cnt, a.G, a.window, a.first, a.parents != nullptr, bm, kt) + (int)a.tps.d - 1), a.tps);
                rts = kv_row_tiles(cnt, (int)a.G.d, bm);
                full = rts * ns * (int)a.kv_heads.d;
                n = SHARES ? full : (ns > 1 ? rts * (int)(sub.d * a.kv_heads.d) : 0);
            }
        }
        const int end = kv_scan(n), iend = SHARES ? 0 : kv_scan(full);
        const uint64_t hit = __ballot(base + end > idx);
        if (hit) {
            const int w = __builtin_ctzll(hit);
            it.b = b0 + w;
            it.nsplit = __builtin_amdgcn_readlane(ns, w); it.len = __builtin_amdgcn_readlane(len, w); it.cnt = __builtin_amdgcn_readlane(cnt, w); it.row0 = __builtin_amdgcn_readlane(row0, w);
            it.page0 = __builtin_amdgcn_readlane(page0, w); it.row_tiles = __builtin_amdgcn_readlane(rts, w);
            const int e = __builtin_amdgcn_readlane(end, w), nn = __builtin_amdgcn_readlane(n, w);
            it.base = SHARES ? base + e - nn : ibase + __builtin_amdgcn_readlane(iend, w) - __builtin_amdgcn_readlane(full, w);
            uint32_t kvh;
            const uint32_t r = kv_div((uint32_t)(idx - (base + e - nn)), a.kv_heads, kvh);
            it.kvh = (int)kvh;
            if (SHARES) { const uint32_t t = it.nsplit == 1 ? r : r / (uint32_t)it.nsplit; it.split = (int)(r - t * it.nsplit); it.rt = it.row_tiles - 1 - (int)t; }
            else { uint32_t part; it.rt = it.row_tiles - 1 - (int)kv_div(r, sub, part); it.split = (int)part; }
            return it;
        }
        base += __builtin_amdgcn_readlane(end, 63);
        if (!SHARES) ibase += __builtin_amdgcn_readlane(iend, 63);
    }
    it.b = -1;
    return it;
}
// the item that holds a row tile's share, for the one who joins them
__device__ __forceinline__ int kv_item_of(const KvAttnArgs& a, const KvItem& it, int split) {
    return it.base + ((it.row_tiles - 1 - it.rt) * it.nsplit + split) * (int)a.kv_heads.d + it.kvh;
}

// the keys of a row tile: tiles of kept first keys that lie apart from the window's, then one range
struct KvRange { int lo, hi, kept, start, tiles, before, t0, t1; };      // [lo, hi) without the kept ones, tiles of kept keys, first key of the range, tiles in all
__device__ __forceinline__ KvRange kv_range(const KvAttnArgs& a, const KvItem& it, int bm, int kt) {
    KvRange r;
    r.before = it.len - it.cnt;
    r.t0 = (int)kv_div((uint32_t)(it.rt * bm), a.G);
    r.t1 = min(it.cnt, (int)kv_div((uint32_t)((it.rt + 1) * bm - 1), a.G) + 1);
    r.hi = r.before + r.t1;                  // a draft's ancestors come before it
    r.lo = 0; r.kept = 0; r.start = 0;
    if (a.window > 0) {
        r.lo = max(0, r.before + (a.parents ? 0 : r.t0) - a.window + 1);
        const int at = r.lo / kt * kt;
        if (a.first > 0 && at < a.first) r.start = 0;
        else { r.start = at; r.kept = (min(a.first, r.hi) + kt - 1) / kt; }
    }
    r.tiles = r.kept + (r.hi - r.start + kt - 1) / kt;
    return r;
}

// ---- references of the softmax: weights are exp2(score - m), and m, -infinity until the row has seen a key, is no more than a measure that sums and weights share.  It stands while a lane's
// sum of weights (of 8 keys or 16) lies in bounds and may move, with what was summed so far, when it does not.
// bf16 weights have the range of 32 bits.  The reference is 2^8 times the largest weight it was taken from, and moves up when a sum passes 1: no weight is over 1, so that values up to the end of
// the numbers have no larger sums than the definition gives them, and weights end at 2^-118 of the largest
// (two prompts over eight bits, queries 1, 2, 3, 5 and 10 times as large: 1.29, 1.24, 1.30, 1.35, 1.40 ms; weights of up to 2^30, which moved it less, 1.34, 1.26, 1.27, 1.28, 1.32).
// f16 weights (HM) are subnormal numbers below 2^-14 and end at 2^16.  A reference goes up to 2^-10 of the largest weight when a lane's sum passes 2^15, so that no weight is off by more than
// 2^-35 of the row's largest.  A key may draw nearly all attention and be worth nothing, though, and the many far under it are the result: when a lane's sum falls under 2^-10 (16 equal weights are
// 2^-14 each) the reference comes down, as far as the tile's largest key allows, and its weights are off by 2^-11 of their sum again.  It stays within 2^60 of what was summed, where 32-bit sums of
// 16-bit numbers have their end far away, and comes down four times at most in a wave's share of the keys: scores that vary by more than the 2^25 between the bounds would move it to and fro
// (portions of f16 pages, queries 1, 2, 3, 5 and 10 times as large: 1.72, 1.64, 1.83, 1.73, 1.71 ms; down without end 1.75, 2.10, 2.32, 2.33, 2.33; never down 1.74, 1.66, 1.64, 1.61, 1.62).
// Weights are worked out as exp2(fma(product, scale, -m)), and once more where a reference moves: as exp2(score - m) of scores rounded to 32 bits, as m is.  Past 2^20 the rounding of m is no
// longer small, and would be all that a weight from the fma is made of past 2^27: there all weights are worked out twice.
struct KvBounds { float most, least; };      // of a lane's sum.  most: -1, which every sum passes, until the row has seen a key, and for references past 2^20; least: 0 where it comes down no more
constexpr float KV_LEAST = 0x1p-10f;
template <bool HM> __device__ __forceinline__ bool kv_out_of_bounds(float sum, const KvBounds& b) { return sum > b.most || (HM && sum < b.least); }
template <bool HM> __device__ __forceinline__ float kv_most(float m) { return fabsf(m) > 1048576.0f ? -1.0f : HM ? 32768.0f : 1.0f; }
// the reference after keys whose largest score is t, in one lane no more than low; sum: all of the row's weights so far
template <bool HM> __device__ __forceinline__ float kv_reference(float m, float t, float low, float sum, KvBounds& b) {
    if constexpr (!HM) return fmaxf(m, t + 8.0f);
    else {
        if (t == -INFINITY) return m;
        const float ten = t - 10.0f, under = t - ten > 10.0f ? t : ten;      // past 2^27 the numbers lie 16 apart
        if (t - m > 10.0f) return under;
        const float end = m + __builtin_amdgcn_logf(sum) - 60.0f, to = fmaxf(fmaxf(low + 8.0f, under), end);
        if (!(m - low > 10.0f && to < m - 2.0f && b.least > 0.0f)) return m;
        b.least = to == end ? 0.0f : b.least - KV_LEAST / 4;
        return to;
    }
}

// the keys [first, first + 32) that a row sees, of those before `end`: bit k for key first + k.  pos: the row's position; seen: its drafts (those outside its window left out)
__device__ __forceinline__ uint32_t kv_below(int n) { return n >= 32 ? 0xFFFFFFFFu : (1u << max(n, 0)) - 1; }
__device__ __forceinline__ uint32_t kv_visible(const KvAttnArgs& a, const KvRange& rg, int first, int end, int pos, uint64_t seen) {
    const int before = rg.before - first;
    uint32_t ok = a.parents ? kv_below(before) : kv_below(pos + 1 - first);
    if (a.window > 0) ok &= ~kv_below(pos - a.window + 1 - first) | kv_below(a.first - first);
    if (a.parents) {
        const uint32_t up = before >= 32 ? 0u : (uint32_t)(seen << (before & 31)), down = before <= -64 ? 0u : (uint32_t)(seen >> (-before & 63));
        ok |= before >= 0 ? up : down;
    }
    return ok & kv_below(end - first);
}
