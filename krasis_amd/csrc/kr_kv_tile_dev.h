// kr_kv_tile_dev.h -- attention over the paged cache for sequences with more than 16 rows of new tokens: prompts and their portions, drafted trees.
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over the stored keys j that row i sees; a row is a new token with one head of a group, so that a tile of keys serves the whole group.
// Hundreds of operations a byte: the matrix cores bound it.  A workgroup takes 4 waves x RB blocks of 32 rows, one key / value head and a share of the key tiles.  Tiles of 64 keys come
// from the pages into registers ahead of time, are converted there (exact, kr_kv_dev.h) and stand in LDS as rows of 16-bit numbers, two tiles of each.
//   S^T[key][row] = K Q^T    v_mfma_f32_32x32x16; queries stay in registers; a lane's scores belong to one row of each block, whose softmax is lane-local but for one exchange
//   O^T[d][row] += V^T P^T   the weights go from the accumulators to the operand in place (the order of keys within a product is free); V's columns come from the transposing LDS read
// A wave is alone on its SIMD where it has two blocks (a fragment read from LDS then serves two products: with one, LDS reads take as long as the products), so its own work has to
// overlap: the scores of tile t + 1 are multiplied while the weights of tile t are formed, and the maxima of tile t + 1 and the next tiles' conversion go under the product with V.
// Weights are measured from a reference that follows the row's maximum only when that has grown by more than 2^8: sums of 32 bits and weights of 16 hold the difference, and the
// rescaling of O all but vanishes.
#pragma once
#include "kr_kv_dev.h"
#include "kr_lds_optin.h"
#include <type_traits>

typedef __fp16 kvt_h4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
constexpr int KT = KV_TILE_KT;
constexpr int kvt_ldk(int dim) { return 2 * dim + 16; }                                   // neighbouring rows four banks apart: reads of 16 bytes down the keys
constexpr int kvt_ldv(int dim) { return (2 * dim) % 128 == 64 ? 2 * dim : 2 * dim + 64; }   // an odd multiple of 64 bytes: the transposing read takes 64 bytes of eight rows
constexpr int kvt_lds(int dim) { return 2 * KT * (kvt_ldk(dim) + kvt_ldv(dim)) + 2 * KT * 4 + KV_MAX_TREE * 4 + 16; }

template <bool H> __device__ __forceinline__ kv_f16 kvt_mfma(u32x4 x, u32x4 y, kv_f16 c) {
    if constexpr (H) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(kv_h8, x), __builtin_bit_cast(kv_h8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(kv_b8, x), __builtin_bit_cast(kv_b8, y), c, 0, 0, 0);
}

// the order of a step's instructions: after every matrix product some of the vector unit's work
#define KVT_MIX(products, vector, exps) \
    _Pragma("unroll") for (int x_ = 0; x_ < (products); x_++) { \
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); __builtin_amdgcn_sched_group_barrier(0x002, (vector), 0); __builtin_amdgcn_sched_group_barrier(0x400, (exps), 0); }

template <int DIM, int FMT, bool HQ, int RB>
__global__ void __launch_bounds__(256, kv_tile_waves(DIM, RB)) kr_kv_tile_kernel(const KvAttnArgs a) {
    constexpr bool HM = HQ && FMT == 0;
    constexpr int NP = HQ && !HM ? 2 : 1;                     // bf16 pieces of an f16 query and of its weights
    constexpr int BITS = FMT == 0 ? 16 : FMT == 1 ? 8 : 4, CPR = DIM * BITS / 128, NCH = KT * CPR, PT = (NCH + 255) / 256, CD = 128 / BITS;      // chunks of 16 bytes, CD channels
    constexpr int LDK = kvt_ldk(DIM), LDV = kvt_ldv(DIM), KS = DIM / 16, DB = DIM / 32, BM = 128 * RB, RING = 4;
    extern __shared__ __attribute__((aligned(16))) char kvt_lds_[];
    char* Ks = kvt_lds_; char* Vs = Ks + 2 * KT * LDK;
    uint32_t* Sl = (uint32_t*)(Vs + 2 * KT * LDV);            // [2][KT] where a tile's keys lie, in units of 16 bytes
    int* Dp = (int*)(Sl + 2 * KT);                            // [KV_MAX_TREE] depths of the drafts
    int* Odd = Dp + KV_MAX_TREE;                              // some value of a tile that not all rows see was not finite
    const KvItem it = kv_item<true>(a, blockIdx.x, BM, KT, 1);
    if (it.b < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, h = lane >> 5;
    const KvRange rg = kv_range(a, it, BM, KT);
    const int c0 = it.split * a.tps, c1 = min(rg.tiles, c0 + a.tps);
    const int rows = it.cnt * a.G, rw = it.rt * BM + wave * 32 * RB;
    const int w0 = min(it.cnt - 1, rw / a.G), w1 = min(it.cnt - 1, (rw + 32 * RB - 1) / a.G);      // the wave's first and last token
    const int* table = a.s.pages + it.page0;
    const float scale = fmaxf(fabsf(a.scale_log2), 1.1754944e-38f);      // its sign goes into the queries: scores that are not seen are -infinity before it, too

    int tk[RB], pos[RB]; uint64_t seen[RB];
    uint64_t all = 0;
    if (a.parents) {
        all = kv_ancestors(a.parents + it.row0, it.cnt, lane);
        if (tid < KV_MAX_TREE) Dp[tid] = __popcll(all) - 1;
    }
    u32x4 qf[RB][NP][KS];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        const int r = min(rw + 32 * rb + col, rows - 1);
        tk[rb] = r / a.G; pos[rb] = rg.before + tk[rb]; seen[rb] = 0;
        if (a.parents) {
            seen[rb] = (uint64_t)__shfl((uint32_t)(all >> 32), tk[rb]) << 32 | __shfl((uint32_t)all, tk[rb]);
            pos[rb] = rg.before + __popcll(seen[rb]) - 1;
        }
        const uint16_t* qp = a.q + (size_t)(it.row0 + tk[rb]) * a.q_tok + (size_t)(it.kvh * a.G + r - tk[rb] * a.G) * a.q_head + 8 * h;
        const uint32_t sign = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(qp + 16 * i) ^ sign;
            if constexpr (NP == 1) qf[rb][0][i] = x;
            else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const kv_h2 y = kv_halves(x[e]);
                    const float u = (float)y[0], w = (float)y[1];
                    const uint32_t hi = kv_pack<false>(u, w);
                    qf[rb][0][i][e] = hi; qf[rb][1][i][e] = kv_rest(u, w, hi);
                }
            }
        }
    }
    auto first_key = [&](int c) { return c < rg.kept ? KT * c : rg.start + KT * (c - rg.kept); };
    auto place = [&](int c, int k) {                          // keys no row sees give way to one that is seen
        const int j = first_key(c) + k;
        return kv_slot(a.p, table, (uint32_t)(j < rg.lo && j >= a.first ? rg.lo : min(j, rg.hi - 1))) * a.p.row16;
    };
    // this thread's chunks: row of the tile, place in the row
    u32x4 kn[PT], vn[PT]; uint32_t ksn[PT], vsn[PT], off[PT];
    const uint8_t* kb = a.p.k + (size_t)it.kvh * a.p.head_bytes; const uint8_t* vb = a.p.v + (size_t)it.kvh * a.p.head_bytes;
    const uint8_t* ksb = a.p.ks + it.kvh * a.p.shead_bytes; const uint8_t* vsb = a.p.vs + it.kvh * a.p.shead_bytes;
    auto chunk = [&](int j, int& row, int& dc) { const int ch = tid + 256 * j; row = ch / CPR; dc = ch - row * CPR; return NCH % 256 == 0 || ch < NCH; };
    auto request = [&](const uint8_t* base, const uint8_t* sbase, u32x4* w, uint32_t* s) {
#pragma unroll
        for (int j = 0; j < PT; j++) {
            int row, dc;
            if (!chunk(j, row, dc)) break;
            w[j] = *reinterpret_cast<const u32x4*>(base + (((uint64_t)off[j] << 4) + dc * 16));
            if constexpr (FMT != 0) s[j] = sbase[(off[j] >> a.p.scale_shift) + (uint32_t)(dc * CD / 32)];
        }
    };
    auto places = [&](int buf) {
#pragma unroll
        for (int j = 0; j < PT; j++) { int row, dc; if (!chunk(j, row, dc)) break; off[j] = Sl[buf * KT + row]; }
    };
    auto convert = [&](const u32x4& w, uint32_t s, uint32_t* o) {      // 16 bytes of codes as CD numbers
        const float sc = kv_scale((s & a.p.scale_and) | a.p.scale_or);
        if constexpr (FMT == 0) { o[0] = w.x; o[1] = w.y; o[2] = w.z; o[3] = w.w; }
        else if constexpr (FMT == 1) {
#pragma unroll
            for (int e = 0; e < 4; e++) { o[2 * e] = kv_pair<1, 0>(w[e], sc); o[2 * e + 1] = kv_pair<1, 1>(w[e], sc); }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) { o[4 * e] = kv_pair<2, 0>(w[e], sc); o[4 * e + 1] = kv_pair<2, 1>(w[e], sc); o[4 * e + 2] = kv_pair<2, 2>(w[e], sc); o[4 * e + 3] = kv_pair<2, 3>(w[e], sc); }
        }
    };
    auto commit = [&](char* dst, int ld, const u32x4* src, const uint32_t* s, int j) {
        int row, dc;
        if (!chunk(j, row, dc)) return;
        uint32_t w[CD / 2];
        convert(src[j], s[j], w);
#pragma unroll
        for (int e = 0; e < CD / 8; e++) *reinterpret_cast<u32x4*>(dst + row * ld + (dc * CD + 8 * e) * 2) = u32x4{w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]};
    };
    constexpr uint32_t EXP = HM ? 0x7C00u : 0x7F80u;
    // every row from token ta to token tb sees all keys of the tile
    auto open = [&](int c, int ta, int tb) {
        const int j0 = first_key(c), jn = c < rg.kept ? min(a.first, rg.hi) : rg.hi;
        if (j0 + KT > jn || j0 + KT - 1 > rg.before + (a.parents ? -1 : ta)) return false;
        return a.window <= 0 || rg.before + tb - j0 < a.window || j0 + KT <= a.first;
    };
    // A value that is not finite may belong to a key that some rows do not see, and 0 times it would not be 0: in tiles that are not open to all rows such values become 0 here, and what
    // they do to the rows that see them is added at the end.
    auto look = [&]() {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < PT; j++) {
            int row, dc;
            if (!chunk(j, row, dc)) break;
            if constexpr (FMT == 0) {
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int u = 0; u < 32; u += 16) if ((vn[j][e] >> u & EXP) == EXP) { vn[j][e] &= ~(0xFFFFu << u); odd = true; }
            } else {
                if (((vsn[j] & a.p.scale_and) | a.p.scale_or) == 255u) { vn[j] = u32x4{0, 0, 0, 0}; vsn[j] = 127; odd = true; }
                if constexpr (FMT == 1)
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int u = 0; u < 32; u += 8) if ((vn[j][e] >> u & 0x7Fu) == 0x7Fu) { vn[j][e] &= ~(0xFFu << u); odd = true; }
            }
        }
        if (odd) *Odd = 1;
    };
    float m[RB], l[RB], base[RB], t[RB];
    kv_f16 o[RB][DB], sa[RB], sb[RB];
    u32x4 pf[RB][NP][2];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        m[rb] = -INFINITY; l[rb] = base[rb] = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[rb][d][i] = 0.0f;
    }
    const int kofs = col * LDK + 16 * h, vofs = (4 * h + ((lane & 15) >> 2)) * LDV + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
    auto key = [&](const char* kl, int i) { return *reinterpret_cast<const u32x4*>(kl + 32 * i); };
    auto value = [&](const char* vl, int d, int s) {
        const char* va = vl + 16 * s * LDV + 64 * d;
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) kvt_h4*)(va)));
        const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) kvt_h4*)(va + 8 * LDV)));
        return u32x4{x.x, x.y, y.x, y.y};
    };
    // the weights of scores 2 e, 2 e + 1 of a half tile
    auto weigh = [&](const kv_f16 (&s)[RB], int e) {
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][2 * e], scale, -base[rb])), p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][2 * e + 1], scale, -base[rb]));
            l[rb] += p0 + p1;
            const uint32_t w = kv_pack<HM>(p0, p1);
            pf[rb][0][e >> 2][e & 3] = w;
            if constexpr (NP == 2) pf[rb][1][e >> 2][e & 3] = kv_rest(p0, p1, w);
        }
    };
    // Scores of half tile b of tile c into n, while the weights of s are formed: the eight pairs of s are spread over the KS steps of the product.
    auto scores = [&](int c, int b, kv_f16 (&n)[RB], const kv_f16 (&s)[RB], auto WEIGH) {
        const char* kl = Ks + (c & 1) * KT * LDK + 32 * b * LDK + kofs;
        u32x4 ring[RING];
#pragma unroll
        for (int rb = 0; rb < RB; rb++)
#pragma unroll
            for (int i = 0; i < 16; i++) n[rb][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < RING; i++) ring[i] = key(kl, i);
#pragma unroll
        for (int i = 0; i < KS; i++) {
#pragma unroll
            for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                for (int rb = 0; rb < RB; rb++) n[rb] = kvt_mfma<HM>(ring[i % RING], qf[rb][p][i], n[rb]);
            if (i + RING < KS) ring[i % RING] = key(kl, i + RING);
            if constexpr (WEIGH) {
#pragma unroll
                for (int e = 8 * i / KS; e < 8 * (i + 1) / KS; e++) weigh(s, e);
                KVT_MIX(RB * NP, 7 * RB * 8 / KS / (RB * NP) + 1, 2 * RB * 8 / KS / (RB * NP) + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto mask = [&](int c, int b, kv_f16 (&s)[RB]) {          // scores of keys that a row does not see
        const int j0 = first_key(c), end = c < rg.kept ? min(a.first, rg.hi) : rg.hi;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int key = j0 + 32 * b + (i & 3) + 8 * (i >> 2) + 4 * h, n = key - rg.before;
            const int at = a.parents && n >= 0 ? rg.before + Dp[n & (KV_MAX_TREE - 1)] : key;
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
                bool ok = key < end;
                if (a.parents) { if (n >= 0) ok = ok && (seen[rb] >> (n & 63) & 1); }
                else ok = ok && key <= pos[rb];
                if (a.window > 0) ok = ok && (pos[rb] - at < a.window || at < a.first);
                if (!ok) s[rb][i] = -INFINITY;
            }
        }
    };
    auto top = [&](const kv_f16 (&s)[RB], int e) {            // the maximum grows by scores 2 e, 2 e + 1
#pragma unroll
        for (int rb = 0; rb < RB; rb++) t[rb] = e == 0 ? fmaxf(s[rb][0], s[rb][1]) : fmaxf(fmaxf(t[rb], s[rb][2 * e]), s[rb][2 * e + 1]);
    };
    auto follow = [&]() {                                     // the rows' references after a half tile's maxima; NaN scores are in no maximum
        bool grown = false;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) { t[rb] = fmaxf(t[rb], __shfl_xor(t[rb], 32)) * scale; grown = grown || t[rb] > m[rb] + 8.0f; }
        if (!__any(grown)) return;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            const float mn = t[rb] > m[rb] + 8.0f ? t[rb] : m[rb];
            base[rb] = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m[rb] - base[rb]);
            m[rb] = mn; l[rb] *= f;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[rb][d][i] *= f;
        }
    };
    // The product with half tile b's values, while the maxima of n are found and, in the second half, the coming tiles go to LDS: keys of tile c + 2 where tile c's were, values of c + 1.
    auto sums = [&](int c, int b, const kv_f16 (&n)[RB], auto COMMIT) {
        const char* vl = Vs + (c & 1) * KT * LDV + vofs;
        constexpr int STEPS = 2 * DB;
        u32x4 ring[RING];
#pragma unroll
        for (int i = 0; i < RING; i++) ring[i] = value(vl, i >> 1, 2 * b + (i & 1));
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
#pragma unroll
            for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                for (int rb = 0; rb < RB; rb++) o[rb][i >> 1] = kvt_mfma<HM>(ring[i % RING], pf[rb][p][i & 1], o[rb][i >> 1]);
            if (i + RING < STEPS) ring[i % RING] = value(vl, (i + RING) >> 1, 2 * b + ((i + RING) & 1));
#pragma unroll
            for (int e = 8 * i / STEPS; e < 8 * (i + 1) / STEPS; e++) top(n, e);
            if constexpr (COMMIT) {
#pragma unroll
                for (int j = 2 * PT * i / STEPS; j < 2 * PT * (i + 1) / STEPS; j++) {
                    if (j < PT) commit(Ks + (c & 1) * KT * LDK, LDK, kn, ksn, j);
                    else commit(Vs + ((c + 1) & 1) * KT * LDV, LDV, vn, vsn, j - PT);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    using yes = std::integral_constant<bool, true>; using no = std::integral_constant<bool, false>;
    if (c0 < c1) {
        const int cc = c0 & 1;                                // buffers go by the tile's number
        if (tid == 0) *Odd = 0;
        if (tid < 2 * KT) { const int c = min(c0 + tid / KT, c1 - 1); Sl[(cc ^ (tid / KT)) * KT + tid % KT] = place(c, tid % KT); }
        __syncthreads();
        places(cc);
        request(kb, ksb, kn, ksn); request(vb, vsb, vn, vsn);
        uint32_t ahead = 0;
        if (tid < 2 * KT) ahead = place(min(c0 + 2 + tid / KT, c1 - 1), tid % KT);
        if (!open(c0, rg.t0, rg.t1 - 1)) look();
#pragma unroll
        for (int j = 0; j < PT; j++) { commit(Ks + cc * KT * LDK, LDK, kn, ksn, j); commit(Vs + cc * KT * LDV, LDV, vn, vsn, j); }
        places(cc ^ 1);
        request(kb, ksb, kn, ksn); request(vb, vsb, vn, vsn);      // tile c0 + 1, or the last one again
        __syncthreads();
        if (tid < 2 * KT) Sl[(cc ^ (tid / KT)) * KT + tid % KT] = ahead;
#pragma unroll
        for (int j = 0; j < PT; j++) commit(Ks + (cc ^ 1) * KT * LDK, LDK, kn, ksn, j);
        scores(c0, 0, sa, sb, no());
        if (!open(c0, w0, w1)) mask(c0, 0, sa);
#pragma unroll
        for (int e = 0; e < 8; e++) top(sa, e);
        follow();
        __syncthreads();
        if (c0 + 2 < c1) { places(cc); request(kb, ksb, kn, ksn); }
        // A tile: the scores of its first half are in sa, their maxima followed; its values and the next tile's keys are in LDS behind the barrier.
        for (int c = c0; c < c1; c++) {
            __syncthreads();
            ahead = 0;
            if (tid < KT && c + 4 < c1) ahead = place(c + 4, tid);
            scores(c, 1, sb, sa, yes());
            if (!open(c, w0, w1)) mask(c, 1, sb);
            sums(c, 0, sb, no());
            follow();
            scores(c + 1, 0, sa, sb, yes());                  // behind the last tile: of no use, and harmless
            const bool more = c + 1 < c1;
            if (more && !open(c + 1, w0, w1)) mask(c + 1, 0, sa);
            if (more && !open(c + 1, rg.t0, rg.t1 - 1)) look();
            sums(c, 1, sa, yes());
            if (more) follow();
            if (tid < KT && c + 4 < c1) Sl[(c & 1) * KT + tid] = ahead;      // where tile c + 2's were, read an iteration ago
            if (c + 2 < c1) request(vb, vsb, vn, vsn);
            if (c + 3 < c1) { places((c + 3) & 1); request(kb, ksb, kn, ksn); }
        }
        __syncthreads();
        if (*Odd) {                                           // the values that became 0 above: every row takes those that it sees
#pragma unroll 1
            for (int c = c0; c < c1; c++) {
                if (open(c, rg.t0, rg.t1 - 1)) continue;
                const int j0 = first_key(c), end = c < rg.kept ? min(a.first, rg.hi) : rg.hi;
#pragma unroll 1
                for (int k = 0; k < KT && j0 + k < end; k++) {
                    const int key = j0 + k, n = key - rg.before, at = a.parents && n >= 0 ? rg.before + Dp[n & (KV_MAX_TREE - 1)] : key;
                    const uint32_t pl = place(c, k);
                    const uint8_t* vp = vb + ((uint64_t)pl << 4);
                    const uint8_t* sp = vsb + (pl >> a.p.scale_shift);
                    bool ok[RB];
#pragma unroll
                    for (int rb = 0; rb < RB; rb++) {
                        ok[rb] = a.parents && n >= 0 ? (seen[rb] >> (n & 63) & 1) != 0 : key <= pos[rb];
                        if (a.window > 0) ok[rb] = ok[rb] && (pos[rb] - at < a.window || at < a.first);
                    }
#pragma unroll
                    for (int d = 0; d < DB; d++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int x = 32 * d + 8 * (i >> 2) + 4 * h + (i & 3);
                            float add = 0.0f;
                            if constexpr (FMT == 0) {
                                const uint32_t z = reinterpret_cast<const uint16_t*>(vp)[x];
                                if ((z & EXP) == EXP) add = (z & (HM ? 0x3FFu : 0x7Fu)) ? NAN : z >> 15 ? -INFINITY : INFINITY;
                            } else {
                                if (((sp[x / 32] & a.p.scale_and) | a.p.scale_or) == 255u) add = NAN;
                                if constexpr (FMT == 1) if ((vp[x] & 0x7Fu) == 0x7Fu) add = NAN;
                            }
#pragma unroll
                            for (int rb = 0; rb < RB; rb++) if (ok[rb]) o[rb][d][i] += add;
                        }
                }
            }
        }
    }
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        l[rb] += __shfl_xor(l[rb], 32);
        const int r = rw + 32 * rb + col;
        if (r >= rows) continue;
        if (it.nsplit == 1) {
            const float inv = l[rb] == 0.0f ? 0.0f : 1.0f / l[rb];
            uint16_t* op = a.out + ((size_t)(it.row0 + tk[rb]) * a.heads + it.kvh * a.G + r - tk[rb] * a.G) * DIM + 4 * h;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *reinterpret_cast<u32x2*>(op + 32 * d + 8 * g) = u32x2{kv_pack<HQ>(o[rb][d][4 * g] * inv, o[rb][d][4 * g + 1] * inv), kv_pack<HQ>(o[rb][d][4 * g + 2] * inv, o[rb][d][4 * g + 3] * inv)};
        } else {
            const size_t at = (size_t)blockIdx.x * BM + wave * 32 * RB + 32 * rb + col;
            float* wp = a.ws + at * DIM + 4 * h;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int g = 0; g < 4; g++) *reinterpret_cast<float4*>(wp + 32 * d + 8 * g) = make_float4(o[rb][d][4 * g], o[rb][d][4 * g + 1], o[rb][d][4 * g + 2], o[rb][d][4 * g + 3]);
            if (h == 0) { float* sp = a.ws + (size_t)a.items * BM * DIM + at * 2; sp[0] = m[rb]; sp[1] = l[rb]; }
        }
    }
}

template <int DIM, int FMT, bool HQ, int RB> static int kvt_launch(const KvAttnArgs& a, hipStream_t st) {
    constexpr size_t lds = kvt_lds(DIM);
    if (lds > 65536 && kr_lds_optin((const void*)kr_kv_tile_kernel<DIM, FMT, HQ, RB>, lds)) return 1;
    hipLaunchKernelGGL((kr_kv_tile_kernel<DIM, FMT, HQ, RB>), dim3(a.items), dim3(256), lds, st, a);
    return 0;
}
template <int DIM, int FMT> static int kvt_launch(const KvAttnArgs& a, int half, int blocks, hipStream_t st) {
    if constexpr (kv_tile_two(DIM, FMT, 0)) if (blocks == 2 && !half) return kvt_launch<DIM, FMT, false, 2>(a, st);
    if constexpr (kv_tile_two(DIM, FMT, 1)) if (blocks == 2 && half) return kvt_launch<DIM, FMT, true, 2>(a, st);
    if (blocks != 1) return 1;
    return half ? kvt_launch<DIM, FMT, true, 1>(a, st) : kvt_launch<DIM, FMT, false, 1>(a, st);
}
template <int FMT> static int kvt_dim(const KvAttnArgs& a, int dim, int half, int blocks, hipStream_t st) {
    switch (dim) {
        case 64: return kvt_launch<64, FMT>(a, half, blocks, st);
        case 96: return kvt_launch<96, FMT>(a, half, blocks, st);
        case 128: return kvt_launch<128, FMT>(a, half, blocks, st);
        case 192: return kvt_launch<192, FMT>(a, half, blocks, st);
        case 256: return kvt_launch<256, FMT>(a, half, blocks, st);
    }
    return 1;
}
