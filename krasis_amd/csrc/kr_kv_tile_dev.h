// kr_kv_tile_dev.h -- attention over the paged cache for sequences with more than 16 rows of new tokens: prompts and their portions, drafted trees.
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over the stored keys j that row i sees; a row is a new token with one head of a group, so that a tile of keys serves the whole group.
// Hundreds of operations a byte: the matrix cores bound it.  A workgroup takes four or eight waves of 32 rows, one key / value head and a share of the key tiles.  Tiles of 64 keys come from the
// pages into registers ahead of time, are converted there (exact, kr_kv_dev.h) and stand in LDS as rows of 16-bit numbers, two tiles of each.
//   S^T[key][row] = K Q^T    v_mfma_f32_32x32x16; queries stay in registers; a lane's scores belong to one row, whose softmax is lane-local but for one exchange
//   O^T[d][row] += V^T P^T   the weights go from the accumulators to the operand in place (the order of keys within a product is free); V's columns come from the transposing LDS read
// One or two waves share a SIMD, so a wave's own work has to overlap: the scores of the next half tile are multiplied while the weights of this one are formed, and the maxima of the
// next half and the coming tiles' conversion go under the product with V; the first fragments of each product are read from LDS under the one before.
// Weights are measured from a reference of the row (kr_kv_dev.h) that moves only when a half tile's sum of weights gets out of bounds.  No maxima are formed on the way, and O is hardly ever
// rescaled.
// Weights are rounded to the products' type: bf16 to half a step of 2^-8, as far as the result is rounded itself, f16 2^-11; their sum is of the rounded ones, so that equal values come out as they
// are.  A second bf16 piece would leave 2^-16 and half as many products again: two prompts of 8192 and 3001 tokens 1215 -> 1657 us, 64 drafts late in four documents 119 -> 157, a dozen of eight
// chats 21.2 -> 21.9.  f16 queries over pages that become bf16 have two pieces of queries and weights.
// Measured: those two prompts (64 / 4 heads of 128, eight bits) 1.02 PFLOP/s where a library product of 8192^3 reaches 1.21, the matrix pipe 47 % busy at the 1.9 GHz that its
// power leaves; portions with heads of 256 channels over f16 pages 850 TFLOP/s, one wave a SIMD, 4.8 vector instructions a matrix instruction.  A workgroup's start takes 3 us and up, a
// tile of 128 channels 1.3 us alone: short sequences are bound by that.
#include "kr_kv_dev.h"
#include "kr_lds_optin.h"
#include <type_traits>

typedef __fp16 kvt_h4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
constexpr int KT = KV_TILE_KT;
constexpr int kvt_ldk(int dim) { return 2 * dim + 16; }                                   // neighbouring rows four banks apart: reads of 16 bytes down the keys
constexpr int kvt_ldv(int dim) { return (2 * dim) % 128 == 64 ? 2 * dim : 2 * dim + 64; }   // an odd multiple of 64 bytes: the transposing read takes 64 bytes of eight rows
constexpr int KVT_PLACES = 8;                             // tiles whose places are known: four are looked up at a time, by all threads
constexpr int kvt_lds(int dim) { return 2 * KT * (kvt_ldk(dim) + kvt_ldv(dim)) + KVT_PLACES * KT * 4 + KV_MAX_TREE * 4 + 16; }

template <bool H> __device__ __forceinline__ kv_f16 kvt_mfma(u32x4 x, u32x4 y, kv_f16 c) {
    if constexpr (H) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(kv_h8, x), __builtin_bit_cast(kv_h8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(kv_b8, x), __builtin_bit_cast(kv_b8, y), c, 0, 0, 0);
}

template <int DIM, int FMT, bool HQ, int W>
__global__ void __launch_bounds__(64 * W, W == 8 ? 2 : kv_tile_waves(DIM, FMT, HQ)) kr_kv_tile_kernel(const KvAttnArgs a) {
    constexpr bool HM = HQ && FMT == 0;
    constexpr int NP = HQ && !HM ? 2 : 1;                     // bf16 pieces of an f16 query and of its weights
    constexpr int BITS = FMT == 0 ? 16 : FMT == 1 ? 8 : 4, CPR = DIM * BITS / 128, NCH = KT * CPR, NT = 64 * W, PT = (NCH + NT - 1) / NT, CD = 128 / BITS;      // chunks of 16 bytes, CD channels
    constexpr int LDK = kvt_ldk(DIM), LDV = kvt_ldv(DIM), KS = DIM / 16, DB = DIM / 32, BM = 32 * W, RING = 4, NS = KVT_PLACES;
    extern __shared__ __attribute__((aligned(16))) char kvt_lds_[];
    char* Ks = kvt_lds_; char* Vs = Ks + 2 * KT * LDK;
    uint32_t* Sl = (uint32_t*)(Vs + 2 * KT * LDV);            // [NS][KT] where the keys of tile c lie, in units of 16 bytes, at c modulo NS
    int* Dp = (int*)(Sl + NS * KT);                           // [KV_MAX_TREE] depths of the drafts
    int* Odd = Dp + KV_MAX_TREE;                              // some value of a tile that not all rows see was not finite
    const KvItem it = kv_item<true>(a, blockIdx.x, BM, KT, KvDiv{});
    if (it.b < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, h = lane >> 5;
    const KvRange rg = kv_range(a, it, BM, KT);
    const int c0 = it.split * (int)a.tps.d, c1 = min(rg.tiles, c0 + (int)a.tps.d);
    const int G = (int)a.G.d, rows = it.cnt * G, rw = it.rt * BM + wave * 32;
    const int w0 = min(it.cnt - 1, (int)kv_div((uint32_t)rw, a.G)), w1 = min(it.cnt - 1, (int)kv_div((uint32_t)(rw + 31), a.G));      // the wave's first and last token
    const int* table = a.s.pages + it.page0;
    const float scale = fmaxf(fabsf(a.scale_log2), 1.1754944e-38f);      // its sign goes into the queries: scores that are not seen are -infinity before it, too

    auto first_key = [&](int c) { return c < rg.kept ? KT * c : rg.start + KT * (c - rg.kept); };
    auto page_of = [&](int c, int k, uint32_t& in) {          // keys no row sees give way to one that is seen
        const int j = first_key(c) + k;
        return kv_page(a.p, (uint32_t)(j < rg.lo && j >= a.first ? rg.lo : min(j, rg.hi - 1)), in);
    };
    auto place = [&](int c, int k) {
        uint32_t in;
        const uint32_t n = page_of(c, k, in);
        return ((uint32_t)table[n] * a.p.page.d + in) * a.p.row16;
    };
    // What depends on nothing is asked for first: the pages of the first eight tiles' keys, the queries, the drafts' parents.
    uint32_t page[NS * KT / NT], in[NS * KT / NT];
    if (c0 < c1)
#pragma unroll
        for (int i = 0; i < NS * KT / NT; i++) page[i] = (uint32_t)table[page_of(min(c0 + W * i + (tid >> 6), c1 - 1), lane, in[i])];
    u32x4 qf[NP][KS];
    const int r = min(rw + col, rows - 1), tk = (int)kv_div((uint32_t)r, a.G);
    {
        const uint16_t* qp = a.q + (size_t)(it.row0 + tk) * a.q_tok + (size_t)(it.kvh * G + r - tk * G) * a.q_head + 8 * h;
#pragma unroll
        for (int i = 0; i < KS; i++) qf[0][i] = *reinterpret_cast<const u32x4*>(qp + 16 * i);
    }
    const int parent = a.parents && lane < it.cnt ? a.parents[it.row0 + lane] : -1;
    int pos = rg.before + tk; uint64_t seen = 0;
    auto queries = [&]() {                                    // as they enter the products: the scale's sign, two pieces of f16 where the products are bf16
        const uint32_t sign = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const u32x4 x = qf[0][i] ^ sign;
            if constexpr (NP == 1) qf[0][i] = x;
            else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const kv_h2 y = kv_halves(x[e]);
                    const float u = (float)y[0], w = (float)y[1];
                    const uint32_t hi = kv_pack<false>(u, w);
                    qf[0][i][e] = hi; qf[1][i][e] = kv_rest(u, w, hi);
                }
            }
        }
    };
    // this thread's chunks: row of the tile, place in the row
    u32x4 kn[PT], vn[PT]; uint32_t ksn[PT], vsn[PT], off[PT], coming[PT];
    const uint8_t* kb = a.p.k + (size_t)it.kvh * a.p.head_bytes; const uint8_t* vb = a.p.v + (size_t)it.kvh * a.p.head_bytes;
    const uint8_t* ksb = a.p.ks + it.kvh * a.p.shead_bytes; const uint8_t* vsb = a.p.vs + it.kvh * a.p.shead_bytes;
    auto chunk = [&](int j, int& row, int& dc) { const int ch = tid + NT * j; row = ch / CPR; dc = ch - row * CPR; return NCH % NT == 0 || ch < NCH; };
    auto request = [&](const uint8_t* base, const uint8_t* sbase, u32x4* w, uint32_t* s, uint32_t at, int j) {
        int row, dc;
        if (!chunk(j, row, dc)) return;
        w[j] = *reinterpret_cast<const u32x4*>(base + (((uint64_t)at << 4) + dc * 16));
        if constexpr (FMT != 0) s[j] = sbase[(at >> a.p.scale_shift) + (uint32_t)(dc * CD / 32)];
    };
    auto places = [&](int c, uint32_t* at) {
#pragma unroll
        for (int j = 0; j < PT; j++) { int row, dc; if (!chunk(j, row, dc)) break; at[j] = Sl[(c & (NS - 1)) * KT + row]; }
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
    // the tiles [from, to) behind the kept ones of which every row from token ta to token tb sees all keys
    auto open = [&](int ta, int tb, int& from, int& to) {
        const int last = rg.before + (a.parents ? -1 : ta) + 1 - KT - rg.start;      // where the last such tile may begin
        to = last < 0 ? rg.kept : min(rg.tiles, rg.kept + last / KT + 1);
        const int low = rg.before + tb - a.window + 1 - rg.start;
        from = rg.kept + (a.window > 0 && low > 0 ? (low + KT - 1) / KT : 0);
    };
    int wf, wt, gf, gt;                                       // for the wave's rows, for all rows
    open(w0, w1, wf, wt); open(rg.t0, rg.t1 - 1, gf, gt);
    wf = __builtin_amdgcn_readfirstlane(wf); wt = __builtin_amdgcn_readfirstlane(wt); gf = __builtin_amdgcn_readfirstlane(gf); gt = __builtin_amdgcn_readfirstlane(gt);
    // A value that is not finite may belong to a key that some rows do not see, and 0 times it would not be 0: in tiles that are not open to all rows such values become 0 here, and what
    // they do to the rows that see them is added at the end.
    auto look = [&]() {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < PT; j++) {
            int row, dc;
            if (!chunk(j, row, dc)) break;
            // all ones in a field, and one more: a carry into the sign's place of its number
            if constexpr (FMT == 0) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t bad = ((vn[j][e] & EXP * 0x10001u) + (EXP & -EXP) * 0x10001u) & 0x80008000u;
                    vn[j][e] &= ~((bad << 1) - (bad >> 15)); odd = odd || bad;
                }
            } else {
                if (((vsn[j] & a.p.scale_and) | a.p.scale_or) == 255u) { vn[j] = u32x4{0, 0, 0, 0}; vsn[j] = 127; odd = true; }
                if constexpr (FMT == 1)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t bad = ((vn[j][e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                        vn[j][e] &= ~((bad << 1) - (bad >> 7)); odd = odd || bad;
                    }
            }
        }
        if (odd) *Odd = 1;
    };
    float m = -INFINITY, l = 0.0f, base = 0.0f, hs = 0.0f; KvBounds bounds = {-1.0f, KV_LEAST};
    kv_f16 o[DB], sa, sb;
    u32x4 pf[NP][2];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    const int kofs = col * LDK + 16 * h, vofs = (4 * h + ((lane & 15) >> 2)) * LDV + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
    auto key = [&](const char* kl, int i) { return *reinterpret_cast<const u32x4*>(kl + 32 * i); };
    auto value = [&](const char* vl, int d, int s) {
        const char* va = vl + 16 * s * LDV + 64 * d;
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) kvt_h4*)(va)));
        const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) kvt_h4*)(va + 8 * LDV)));
        return u32x4{x.x, x.y, y.x, y.y};
    };
    using yes = std::integral_constant<bool, true>; using no = std::integral_constant<bool, false>;
    // The weights of scores 2 e, 2 e + 1 of a half tile, and the lane's sum of them as they enter the product, in four stages that different pairs are at in one step: each waits
    // for the one before it, and a wave issues in order.  The empty asm statements keep a stage in its step.
    float x0[4], x1[4];
    auto stage = [&](const kv_f16& s, int e, int k, auto AGAIN) {
        float& a0 = x0[e & 3]; float& a1 = x1[e & 3];
        if (k == 0) {
            if constexpr (AGAIN) { a0 = s[2 * e] * scale - base; a1 = s[2 * e + 1] * scale - base; }
            else { a0 = __builtin_fmaf(s[2 * e], scale, -base); a1 = __builtin_fmaf(s[2 * e + 1], scale, -base); }
            asm volatile("" : "+v"(a0), "+v"(a1));
        }
        else if (k == 1) { a0 = __builtin_amdgcn_exp2f(a0); a1 = __builtin_amdgcn_exp2f(a1); asm volatile("" : "+v"(a0), "+v"(a1)); }
        else if (k == 2) {
            uint32_t w = kv_pack<HM>(a0, a1);
            asm volatile("" : "+v"(w));
            pf[0][e >> 2][e & 3] = w;
        } else {
            const float had = e == 0 ? 0.0f : hs;
            const uint32_t w = pf[0][e >> 2][e & 3];
            if constexpr (NP == 2) { hs = had + (a0 + a1); uint32_t x = kv_rest(a0, a1, w); asm volatile("" : "+v"(x)); pf[1][e >> 2][e & 3] = x; }
            else hs = kv_sum2<HM>(w, had);
            asm volatile("" : "+v"(hs));
        }
    };
    auto weigh = [&](const kv_f16& s, int t, auto AGAIN) {    // pair t begins, those before it go on; t = 0 .. 10
#pragma unroll
        for (int k = 3; k >= 0; k--) if (t - k >= 0 && t - k < 8) stage(s, t - k, k, AGAIN);
    };
    // Scores of half tile b of tile c into n, while the weights of s are formed: spread over the KS steps of the product.  The first fragments of a product are
    // read from LDS in the last steps of the one before: vb_ is the half whose values come next.
    u32x4 kr[RING], vr[RING];
    auto keys_at = [&](int c, int b) { return Ks + (c & 1) * KT * LDK + 32 * b * LDK + kofs; };
    auto values_at = [&](int c, int b) { return Vs + (c & 1) * KT * LDV + 32 * b * LDV + vofs; };
    auto scores = [&](int c, int b, kv_f16& n, const kv_f16& s, int vc, int vb_, auto WEIGH) {
        const char* kl = keys_at(c, b); const char* vl = values_at(vc, vb_);
#pragma unroll
        for (int i = 0; i < 16; i++) n[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; i++) {
#pragma unroll
            for (int p = NP - 1; p >= 0; p--) {
                // queries that do not fit into the first 256 registers stay in the accumulation registers, which a product reads in place
                if constexpr (DIM > 128) asm volatile("" : "+a"(qf[p][i]));
                n = kvt_mfma<HM>(kr[i % RING], qf[p][i], n);
            }
            if (i + RING < KS) kr[i % RING] = key(kl, i + RING);
            else vr[i + RING - KS] = value(vl, (i + RING - KS) >> 1, (i + RING - KS) & 1);
            if constexpr (WEIGH) {
#pragma unroll
                for (int t = 11 * i / KS; t < 11 * (i + 1) / KS; t++) weigh(s, t, no());
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Scores of keys that a row does not see: 32 keys from the lane's first one on are a word, put together without a branch.  Key by key, with the drafts' depths from LDS, a half tile
    // took 3 us where this takes a tenth.
    auto mask = [&](int c, int b, kv_f16& s) {
        const int first = first_key(c) + 32 * b + 4 * h;
        const uint32_t ok = kv_visible(a, rg, first, c < rg.kept ? min(a.first, rg.hi) : rg.hi, pos, seen);
#pragma unroll
        for (int i = 0; i < 16; i++) if (!(ok >> ((i & 3) + 8 * (i >> 2)) & 1)) s[i] = -INFINITY;
    };
    auto halves = [&](float x) {                              // the wave's lower half and its upper one, a register each (through LDS the exchange waits for a round trip)
        const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return make_float2(__uint_as_float(y[0]), __uint_as_float(y[1]));
    };
    // The weights stand when no sum of a half tile is out of bounds; else, and until a row has seen its first key, the references move, and what was summed so far with them.  NaN scores
    // move nothing and are in the sums.
    auto settle = [&](const kv_f16& s) {
        if (__any(kv_out_of_bounds<HM>(hs, bounds))) {
            float t = s[0];
#pragma unroll
            for (int i = 1; i < 16; i++) t = fmaxf(t, s[i]);
            const auto ts = halves(t), ls = halves(l);         // of the row's two lanes
            t = fmaxf(ts.x, ts.y);
            const float low = ts.x == -INFINITY ? ts.y : ts.y == -INFINITY ? ts.x : fminf(ts.x, ts.y), sum = ls.x + ls.y;
            const float mn = kv_reference<HM>(m, t * scale, low * scale, sum, bounds);
            if (__any(mn != m || bounds.most < 0.0f)) {
                base = mn == -INFINITY ? 0.0f : mn;
                const float f = __builtin_amdgcn_exp2f(m - base);
                m = mn; l *= f; bounds.most = kv_most<HM>(mn);
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[d][i] *= f;
#pragma unroll
                for (int t = 0; t < 11; t++) weigh(s, t, yes());
            }
        }
        l += hs;
    };
    // The product with half tile b's values, while the coming tiles go to LDS and those after them are asked for (behind the last tile: some tile's again): keys of tile c + 2 where tile
    // c's were in the first half, values of tile c + 1 in the second.
    auto sums = [&](int c, int b, int kc, int kb_) {
        const char* vl = values_at(c, b); const char* kl = keys_at(kc, kb_);
        constexpr int STEPS = 2 * DB;
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
#pragma unroll
            for (int p = NP - 1; p >= 0; p--) o[i >> 1] = kvt_mfma<HM>(vr[i % RING], pf[p][i & 1], o[i >> 1]);
            if (i + RING < STEPS) vr[i % RING] = value(vl, (i + RING) >> 1, (i + RING) & 1);
            else kr[i + RING - STEPS] = key(kl, i + RING - STEPS);
#pragma unroll
            for (int j = PT * i / STEPS; j < PT * (i + 1) / STEPS; j++) {
                if (b == 0) { commit(Ks + (c & 1) * KT * LDK, LDK, kn, ksn, j); request(kb, ksb, kn, ksn, coming[j], j); }
                else { commit(Vs + ((c + 1) & 1) * KT * LDV, LDV, vn, vsn, j); request(vb, vsb, vn, vsn, off[j], j); off[j] = coming[j]; }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (c0 < c1) {
        if (tid == 0) *Odd = 0;
#pragma unroll
        for (int i = 0; i < NS * KT / NT; i++) Sl[((c0 + W * i + (tid >> 6)) & (NS - 1)) * KT + lane] = (page[i] * a.p.page.d + in[i]) * a.p.row16;
        __syncthreads();
        places(c0, off); places(c0 + 1, coming);
        u32x4 k2[PT]; uint32_t ks2[PT];
#pragma unroll
        for (int j = 0; j < PT; j++) { request(kb, ksb, kn, ksn, off[j], j); request(vb, vsb, vn, vsn, off[j], j); request(kb, ksb, k2, ks2, coming[j], j); }
        if (a.parents) {
            const uint64_t all = kv_ancestors(parent, lane);
            if (tid < KV_MAX_TREE) Dp[tid] = __popcll(all) - 1;
            seen = (uint64_t)__shfl((uint32_t)(all >> 32), tk) << 32 | __shfl((uint32_t)all, tk);
            pos = rg.before + __popcll(seen) - 1;
        }
        queries();
        if (c0 < gf || c0 >= gt) look();
        places(c0 + 2, off);
#pragma unroll
        for (int j = 0; j < PT; j++) {
            commit(Ks + (c0 & 1) * KT * LDK, LDK, kn, ksn, j); commit(Vs + (c0 & 1) * KT * LDV, LDV, vn, vsn, j);
            request(vb, vsb, vn, vsn, coming[j], j); request(kb, ksb, kn, ksn, off[j], j);
        }
#pragma unroll
        for (int j = 0; j < PT; j++) commit(Ks + ((c0 + 1) & 1) * KT * LDK, LDK, k2, ks2, j);
        __syncthreads();
        if (a.parents && a.window > 0 && it.cnt > a.window) {  // ancestors outside the window, eight drafts at a time
            const int last = pos - rg.before - a.window, least = a.first - rg.before;
            for (int n = 0; n < it.cnt; n += 8) {
                int d[8]; uint32_t out = 0;
                *reinterpret_cast<int4*>(d) = *reinterpret_cast<const int4*>(Dp + n); *reinterpret_cast<int4*>(d + 4) = *reinterpret_cast<const int4*>(Dp + n + 4);
#pragma unroll
                for (int u = 0; u < 8; u++) out |= d[u] <= last && d[u] >= least ? 1u << u : 0u;
                seen &= ~((uint64_t)out << n);
            }
        }
#pragma unroll
        for (int i = 0; i < RING; i++) kr[i] = key(keys_at(c0, 0), i);
        scores(c0, 0, sa, sa, c0, 0, no());
#pragma unroll
        for (int i = 0; i < RING; i++) kr[i] = key(keys_at(c0, 1), i);
        if (c0 < wf || c0 >= wt) mask(c0, 0, sa);
        // A tile: the scores of its first half are in sa, masked; its values and the next tile's keys are in LDS behind the barrier.
        for (int c = c0; c < c1; c++) {
            __syncthreads();
            // the places of tiles c + 8 .. c + 11: their pages are asked for, and a tile later they take the place of tiles whose keys have all been asked for
            const int turn = (c - c0) & 3;
            if (turn == 0 && wave < 4) page[0] = (uint32_t)table[page_of(min(c + NS + (tid >> 6), c1 - 1), lane, in[0])];
            scores(c, 1, sb, sa, c, 0, yes());
            if (c < wf || c >= wt) mask(c, 1, sb);
            places(c + 3, coming);                            // not used where there is no such tile
            settle(sa);
            __syncthreads();                                  // every wave has multiplied tile c's keys: the next ones may take their place
            sums(c, 0, c + 1, 0);
            scores(c + 1, 0, sa, sb, c, 1, yes());            // behind the last tile: of no use, and harmless
            const bool more = c + 1 < c1;
            if (more && (c + 1 < wf || c + 1 >= wt)) mask(c + 1, 0, sa);
            if (more && (c + 1 < gf || c + 1 >= gt)) look();
            settle(sb);
            sums(c, 1, c + 1, 1);
            if (turn == 1 && wave < 4) Sl[((c - 1 + (tid >> 6)) & (NS - 1)) * KT + lane] = (page[0] * a.p.page.d + in[0]) * a.p.row16;
        }
        __syncthreads();
        if (*Odd) {                                           // the values that became 0 above: every row takes those that it sees
#pragma unroll 1
            for (int c = c0; c < c1; c++) {
                if (c >= gf && c < gt) continue;
                const int j0 = first_key(c), end = c < rg.kept ? min(a.first, rg.hi) : rg.hi;
#pragma unroll 1
                for (int k = 0; k < KT && j0 + k < end; k++) {
                    const int key = j0 + k, n = key - rg.before, at = a.parents && n >= 0 ? rg.before + Dp[n & (KV_MAX_TREE - 1)] : key;
                    const uint32_t pl = place(c, k);
                    const uint8_t* vp = vb + ((uint64_t)pl << 4);
                    const uint8_t* sp = vsb + (pl >> a.p.scale_shift);
                    bool ok = a.parents && n >= 0 ? (seen >> (n & 63) & 1) != 0 : key <= pos;
                    if (a.window > 0) ok = ok && (pos - at < a.window || at < a.first);
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
                            if (ok) o[d][i] += add;
                        }
                }
            }
        }
    }
    {
        l += __shfl_xor(l, 32);
        if (rw + col >= rows) return;
        if (it.nsplit == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint16_t* op = a.out + ((size_t)(it.row0 + tk) * a.heads + it.kvh * G + r - tk * G) * DIM + 4 * h;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *reinterpret_cast<u32x2*>(op + 32 * d + 8 * g) = u32x2{kv_pack<HQ>(o[d][4 * g] * inv, o[d][4 * g + 1] * inv), kv_pack<HQ>(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv)};
        } else {
            const size_t at = (size_t)blockIdx.x * BM + wave * 32 + col;
            float* wp = a.ws + at * DIM + 4 * h;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int g = 0; g < 4; g++) *reinterpret_cast<float4*>(wp + 32 * d + 8 * g) = make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
            if (h == 0) { float* sp = a.ws + (size_t)a.items * BM * DIM + at * 2; sp[0] = m; sp[1] = l; }
        }
    }
}

template <int DIM, int FMT, bool HQ, int W> static int kvt_launch(const KvAttnArgs& a, hipStream_t st) {
    constexpr size_t lds = kvt_lds(DIM);
    if (lds > 65536 && kr_lds_optin((const void*)kr_kv_tile_kernel<DIM, FMT, HQ, W>, lds)) return 1;
    hipLaunchKernelGGL((kr_kv_tile_kernel<DIM, FMT, HQ, W>), dim3(a.items), dim3(64 * W), lds, st, a);
    return 0;
}
template <int DIM, int FMT> static int kvt_waves(const KvAttnArgs& a, int half, int waves, hipStream_t st) {
    if constexpr (DIM == 96 || DIM == 128) if (waves == 8) return half ? kvt_launch<DIM, FMT, true, 8>(a, st) : kvt_launch<DIM, FMT, false, 8>(a, st);
    return waves != 4 ? 1 : half ? kvt_launch<DIM, FMT, true, 4>(a, st) : kvt_launch<DIM, FMT, false, 4>(a, st);
}
template <int FMT> static int kvt_dim(const KvAttnArgs& a, int dim, int half, int waves, hipStream_t st) {
    switch (dim) {
        case 64: return kvt_waves<64, FMT>(a, half, waves, st);
        case 96: return kvt_waves<96, FMT>(a, half, waves, st);
        case 128: return kvt_waves<128, FMT>(a, half, waves, st);
        case 192: return kvt_waves<192, FMT>(a, half, waves, st);
        case 256: return kvt_waves<256, FMT>(a, half, waves, st);
    }
    return 1;
}
