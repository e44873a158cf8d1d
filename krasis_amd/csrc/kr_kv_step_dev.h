// kr_kv_step_dev.h -- attention over the paged cache for sequences with at most 16 rows of new tokens (one token of a group of up to 16 heads, a few tokens of smaller groups):
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over the stored keys j that row i sees.
// A row of keys serves 16 rows of queries: 4 * 16 operations a channel against one to four bytes of it, far under the matrix rate, so the launch is bound by HBM and its latency.
// Keys and values go from the pages to registers once, converted there to bf16 (exact, kr_kv_dev.h), and meet the queries in v_mfma_f32_16x16x32:
//   S^T[key][row] = K Q^T    first operand: 16 key rows; a lane holds a quarter of a row, so a microscaled row costs it one scale and loads of 16 bytes
//   O^T[d][row] += V^T P^T   a lane holds 8 keys and c neighbouring columns; byte permutes make them the columns' fragments
// A workgroup takes one sequence, one key / value head and a share of its key tiles; its waves, as many as a CU has registers for, take tiles of 32 keys in turn, each with a reference and a sum per row, and
// meet in LDS.  Over pages that become bf16 weights are two bf16 pieces (off by 2^-16), and so are f16 queries; over f16 pages weights are f16 (2^-11, as the result is rounded itself).
// (One piece is no faster where memory bounds the launch: 32 requests of up to 8192 tokens 43.4 us a call with either, two of 131071 and 100003 40.5 and 40.7.)
// Measured: 32 requests of up to 8192 tokens at eight bits (142 MB) 31.3 us, 4.5 TB/s, two of 131071 and 100003 at four bits (126 MB) 32.1 us, 3.9 TB/s; 97 tokens of a chat 7 us, which is one
// round trip after the other (arguments, plan, page table, keys).
#pragma once
#include "kr_kv_dev.h"
#include "kr_lds_optin.h"
#include <type_traits>

template <int DIM> struct KvsCols { static constexpr int C = DIM == 96 ? 2 : DIM == 192 ? 4 : DIM / 16, GROUPS = DIM / (16 * C); };      // columns of V a lane holds: groups of 16 C
constexpr int kvs_lds(int dim, int waves) { return (waves * 16 * (dim + 4) + waves * 32 + 32) * (int)sizeof(float); }

template <int BYTES> __device__ __forceinline__ void kvs_load(const uint8_t* p, uint32_t* w) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; i++) { const u32x4 x = *reinterpret_cast<const u32x4*>(p + 16 * i); w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w; }
    } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 8; i++) { const u32x2 x = *reinterpret_cast<const u32x2*>(p + 8 * i); w[2 * i] = x.x; w[2 * i + 1] = x.y; }
    } else if constexpr (BYTES % 4 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 4; i++) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
    } else if constexpr (BYTES == 2) w[0] = *reinterpret_cast<const uint16_t*>(p);
    else w[0] = *p;
}
// pair e of packed codes as two 16-bit numbers
template <int FMT> __device__ __forceinline__ uint32_t kvs_two(const uint32_t* w, int e, float scale) {
    if constexpr (FMT == 0) return w[e];
    else if constexpr (FMT == 1) return (e & 1) ? kv_pair<1, 1>(w[e >> 1], scale) : kv_pair<1, 0>(w[e >> 1], scale);
    else return (e & 3) == 0 ? kv_pair<2, 0>(w[e >> 2], scale) : (e & 3) == 1 ? kv_pair<2, 1>(w[e >> 2], scale) : (e & 3) == 2 ? kv_pair<2, 2>(w[e >> 2], scale) : kv_pair<2, 3>(w[e >> 2], scale);
}
template <bool H> __device__ __forceinline__ kv_f4 kvs_mfma(u32x4 x, u32x4 y, kv_f4 c) {
    if constexpr (H) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(kv_h8, x), __builtin_bit_cast(kv_h8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kv_b8, x), __builtin_bit_cast(kv_b8, y), c, 0, 0, 0);
}

// HQ: q and out are f16.  Products are f16 where the pages are f16 too, else bf16.  ONE: every sequence of the launch has one new token and no tree, so that its rows see the same keys.
template <int DIM, int FMT, bool HQ, bool ONE>
__global__ void __launch_bounds__(64 * kv_step_waves(DIM, FMT, HQ, ONE), kv_step_waves(DIM, FMT, HQ, ONE) / 4) kr_kv_step_kernel(const KvAttnArgs a) {
    constexpr int WAVES = kv_step_waves(DIM, FMT, HQ, ONE);
    constexpr bool HM = HQ && FMT == 0;                       // f16 products
    constexpr int NP = HQ && !HM ? 2 : 1, NW = HM ? 1 : 2;    // pieces of a query, of a weight
    constexpr int BITS = FMT == 0 ? 16 : FMT == 1 ? 8 : 4, U = DIM / 32, KB = DIM / 4 * BITS / 8, KW = KB / 4;
    constexpr int C = KvsCols<DIM>::C, GROUPS = KvsCols<DIM>::GROUPS, VB = C * BITS / 8, VW = VB < 4 ? 1 : VB / 4;
    constexpr int NB = DIM == 64 || DIM == 128 ? 1 : 2;       // blocks of 32 channels that a quarter of a row meets
    extern __shared__ float kvs_lds_[];
    // Workgroups go round the eight XCDs in turn, and heads lie side by side in a token's row: all heads of a share go to one XCD, whose L2 then fetches a line that two of them have parts
    // of (64 bytes of a head at four bits, the scales of any) once.  32 x 8192 tokens at four bits 56 -> 36 us.
    int idx = blockIdx.x;
    if (const int whole = a.whole; idx < whole) {
        uint32_t head;
        const uint32_t group = kv_div((uint32_t)idx >> 3, a.kv_heads, head) * 8 + (idx & 7);
        idx = (int)(group * a.kv_heads.d + head);
    }
    const KvItem it = kv_item<true>(a, idx, 16, KV_STEP_KT, KvDiv{});
    if (it.b < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = lane & 15, q = lane >> 4;
    const KvRange rg = kv_range(a, it, 16, KV_STEP_KT);
    const int c0 = it.split * (int)a.tps.d, c1 = min(rg.tiles, c0 + (int)a.tps.d);
    const int G = (int)a.G.d, rows = it.cnt * G, r = min(row, rows - 1), t = (int)kv_div((uint32_t)r, a.G), head = it.kvh * G + r - t * G;
    const int* table = a.s.pages + it.page0;
    const uint8_t* kbase = a.p.k + (size_t)it.kvh * a.p.head_bytes + q * KB;
    const uint8_t* vbase = a.p.v + (size_t)it.kvh * a.p.head_bytes;
    const uint8_t* ksb = a.p.ks + it.kvh * a.p.shead_bytes; const uint8_t* vsb = a.p.vs + it.kvh * a.p.shead_bytes;
    auto scale_of = [&](uint32_t byte) { return kv_scale((byte & a.p.scale_and) | a.p.scale_or); };

    // the row's position, and which drafts it sees
    int pos = rg.before + t; uint64_t seen = 0;
    if (!ONE && a.parents) {
        const uint64_t all = kv_ancestors(lane < it.cnt ? a.parents[it.row0 + lane] : -1, lane);
        const int depth = __popcll(all) - 1;                  // of draft `lane`
        seen = (uint64_t)__shfl((uint32_t)(all >> 32), t) << 32 | __shfl((uint32_t)all, t);
        pos = rg.before + __shfl(depth, t);
        if (a.window > 0 && it.cnt > a.window)                // ancestors outside the window
            for (int n = 0; n < it.cnt; n++) {
                const int d = __shfl(depth, n);
                if (pos - rg.before - d >= a.window && rg.before + d >= a.first) seen &= ~(1ull << n);
            }
    }
    // the query row: dims q DIM / 4 + 8 i
    u32x4 qf[NP][U];
    {
        const uint16_t* qp = a.q + (size_t)(it.row0 + t) * a.q_tok + (size_t)head * a.q_head + q * (DIM / 4);
        const uint32_t sign = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int i = 0; i < U; i++) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(qp + 8 * i) ^ sign;
            if constexpr (NP == 1) qf[0][i] = x;
            else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const kv_h2 h = kv_halves(x[e]);
                    const float u = (float)h[0], w = (float)h[1];
                    qf[0][i][e] = kv_pack<false>(u, w); qf[1][i][e] = kv_rest(u, w, qf[0][i][e]);
                }
            }
        }
    }

    // A wave asks for the next tile's keys when it has used this one's, for its values likewise, and for pages a tile earlier still: one set of registers for each, so that more waves
    // than with two sets have a tile on its way.
    uint32_t kn[2][KW], vn[8][GROUPS][VW]; uint32_t ksn[2][NB], vsn[8][GROUPS];
    // where key `lane` of a tile lies: its page is asked for a tile before the place is formed; keys no row sees give way to one that is seen
    uint32_t page = 0, in = 0;
    auto find = [&](int c) {
        c = min(c, c1 - 1);
        const int j = (c < rg.kept ? 32 * c : rg.start + 32 * (c - rg.kept)) + (lane & 31);
        page = (uint32_t)table[kv_page(a.p, (uint32_t)(j < rg.lo && j >= a.first ? rg.lo : min(j, rg.hi - 1)), in)];
    };
    auto place = [&]() { return (page * a.p.page.d + in) * a.p.row16; };      // in units of 16 bytes
    auto request_k = [&](uint32_t s) {
        uint32_t at[2];
#pragma unroll
        for (int b = 0; b < 2; b++) at[b] = __shfl(s, b * 16 + row);
#pragma unroll
        for (int b = 0; b < 2; b++) {
            kvs_load<KB>(kbase + ((uint64_t)at[b] << 4), kn[b]);
            if constexpr (FMT != 0) {
                const uint32_t b0 = (uint32_t)(q * U) >> 2;
#pragma unroll
                for (int i = 0; i < NB; i++) ksn[b][i] = ksb[(at[b] >> a.p.scale_shift) + min(b0 + i, (uint32_t)DIM / 32 - 1)];
            }
        }
    };
    auto request_v = [&](uint32_t s) {
        uint32_t at[8];
#pragma unroll
        for (int i = 0; i < 8; i++) at[i] = __shfl(s, (i >> 2) * 16 + 4 * q + (i & 3));
#pragma unroll
        for (int i = 0; i < 8; i++) {
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                kvs_load<VB>(vbase + row * VB + g * 16 * VB + ((uint64_t)at[i] << 4), vn[i][g]);
                if constexpr (FMT != 0) vsn[i][g] = vsb[(at[i] >> a.p.scale_shift) + (uint32_t)(g * 16 * C + row * C) / 32];
            }
        }
    };

    const float scale = fmaxf(fabsf(a.scale_log2), 1.1754944e-38f);      // its sign goes into the queries: scores that are not seen are -infinity before it, too
    float m = -INFINITY, l = 0.0f, base = 0.0f; KvBounds bounds = {-1.0f, KV_LEAST};
    kv_f4 acc[DIM / 16];
#pragma unroll
    for (int j = 0; j < DIM / 16; j++) acc[j] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
    auto tile = [&](int c, auto MORE) {                       // MORE: the wave has another tile
        const int j0 = c < rg.kept ? 32 * c : rg.start + 32 * (c - rg.kept), end = c < rg.kept ? min(a.first, rg.hi) : rg.hi;
        kv_f4 st[2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            st[b] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
            float sc[NB];
#pragma unroll
            for (int i = 0; i < NB; i++) sc[i] = FMT == 0 ? 1.0f : scale_of(ksn[b][i]);
#pragma unroll
            for (int i = 0; i < U; i++) {
                float s = sc[0];
                if constexpr (NB == 2) { if (DIM == 256 ? i >= 4 : ((q * U + i) >> 2) != (q * U) >> 2) s = sc[1]; }
                u32x4 kf;
#pragma unroll
                for (int e = 0; e < 4; e++) kf[e] = kvs_two<FMT>(&kn[b][i * KW / U], e, s);
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) st[b] = kvs_mfma<HM>(kf, qf[p][i], st[b]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        uint32_t coming = 0;
        if constexpr (MORE) { coming = place(); request_k(coming); }
        __builtin_amdgcn_sched_barrier(0);
        // scores of keys that a row does not see, where the tile has some (the copies that stand for keys no row sees among them); ok: bit 16 b + i for the lane's key i of block b
        const bool hidden = j0 + 32 > end || j0 + 31 > rg.before - (!ONE && a.parents ? 1 : 0) || (a.window > 0 && rg.before + it.cnt - 1 - j0 >= a.window && j0 + 32 > a.first);
        uint32_t ok = 0xFFFFFFFFu;
        if (hidden) {
            ok = kv_visible(a, rg, j0 + 4 * q, end, pos, seen);
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) if (!(ok >> (16 * b + i) & 1)) st[b][i] = -INFINITY;
        }
        // Weights from a reference of the row in this wave (kr_kv_dev.h), which hardly ever moves.  NaN scores move nothing and are in the sums.
        u32x4 pf[NW];
        float hs = 0.0f;
        auto weigh = [&](auto AGAIN) {
            hs = 0.0f;
            auto from = [&](float s) { return __builtin_amdgcn_exp2f(AGAIN ? s * scale - base : __builtin_fmaf(s, scale, -base)); };
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p0 = from(st[e >> 1][2 * (e & 1)]), p1 = from(st[e >> 1][2 * (e & 1) + 1]);
                const uint32_t w = kv_pack<HM>(p0, p1);
                pf[0][e] = w;
                if constexpr (NW == 2) { pf[1][e] = kv_rest(p0, p1, w); hs += p0 + p1; }
                else hs = kv_sum2<HM>(w, hs);
            }
        };
        weigh(std::integral_constant<bool, false>());
        if (__any(kv_out_of_bounds<HM>(hs, bounds))) {
            float t = st[0][0];
#pragma unroll
            for (int i = 1; i < 8; i++) t = fmaxf(t, st[i >> 2][i & 3]);
            float low = t == -INFINITY ? INFINITY : t, sum = l;
            t = fmaxf(t, __shfl_xor(t, 16)); t = fmaxf(t, __shfl_xor(t, 32));
            if constexpr (HM) {
                low = fminf(low, __shfl_xor(low, 16)); low = fminf(low, __shfl_xor(low, 32));
                sum += __shfl_xor(sum, 16); sum += __shfl_xor(sum, 32);
            }
            const float mn = kv_reference<HM>(m, t * scale, low * scale, sum, bounds);
            if (__any(mn != m || bounds.most < 0.0f)) {
                base = mn == -INFINITY ? 0.0f : mn;
                const float f = __builtin_amdgcn_exp2f(m - base);
                m = mn; l *= f; bounds.most = kv_most<HM>(mn);
#pragma unroll
                for (int j = 0; j < DIM / 16; j++) acc[j] *= f;
                weigh(std::integral_constant<bool, true>());
            }
        }
        l += hs;
        constexpr uint32_t EXP = HM ? 0x7C00u : 0x7F80u, UNIT = HM ? 0x3C00u : 0x3F80u;
        // A value that is not finite may belong to a key that some rows do not see, and 0 times it would not be 0.  Rows of one token see the same keys: what they do not see becomes 0.
        // Else such values are looked for (in tiles that all rows see entirely, too: a weight may be too small for the numbers).  A weight's second piece is 0 or negative where the weight
        // is not, so that infinities, which 16-bit pages may hold, meet the first one alone.
        constexpr bool APART = FMT == 0 && NW == 2;
        const bool look = APART || (!ONE && (hidden || it.cnt > 1));
        if constexpr (ONE) if (hidden) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (!(ok >> ((i >> 2) * 16 + (i & 3)) & 1)) {
#pragma unroll
                    for (int g = 0; g < GROUPS; g++) {
#pragma unroll
                        for (int x = 0; x < VW; x++) vn[i][g][x] = 0;
                        vsn[i][g] = 127;
                    }
                }
        }
#pragma unroll
        for (int g = 0; g < GROUPS; g++)
#pragma unroll
            for (int e2 = 0; e2 < C / 2; e2++) {
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = kvs_two<FMT>(vn[i][g], e2, FMT == 0 ? 1.0f : scale_of(vsn[i][g]));
                bool odd = false;
                if (look) {                                   // all ones in a field, and one more: a carry into the sign's place of its number
                    uint32_t bad = 0;
#pragma unroll
                    for (int i = 0; i < 8; i++) bad |= (w[i] & EXP * 0x10001u) + (EXP & -EXP) * 0x10001u;
                    odd = __any((bad & 0x80008000u) != 0);
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int j = g * C + 2 * e2 + u;
                    u32x4 vf;
#pragma unroll
                    for (int e = 0; e < 4; e++) vf[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], u ? 0x07060302u : 0x05040100u);
                    u32x4 vl = vf;                            // what a weight's second piece meets
                    if (ONE && odd) {
#pragma unroll
                        for (int e = 0; e < 4; e++) { const uint32_t bad = ((vf[e] & EXP * 0x10001u) + (EXP & -EXP) * 0x10001u) & 0x80008000u; vl[e] = vf[e] & ~((bad << 1) - (bad >> 15)); }
                    }
                    if (!ONE && odd) {                        // such values apart: whether a row sees one, by kind
                        u32x4 see;                            // ones where the row sees the key, as a fragment
#pragma unroll
                        for (int e = 0; e < 4; e++) see[e] = (ok >> ((e >> 1) * 16 + 2 * (e & 1)) & 1 ? UNIT : 0u) | (ok >> ((e >> 1) * 16 + 2 * (e & 1) + 1) & 1 ? UNIT << 16 : 0u);
                        u32x4 keep = vf;
#pragma unroll
                        for (int k = 0; k < 3; k++) {
                            u32x4 kind;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                kind[e] = 0;
#pragma unroll
                                for (int h = 0; h < 32; h += 16) {
                                    const uint32_t x = vf[e] >> h & 0xFFFFu, t = (x & EXP) != EXP ? 3u : (x & (HM ? 0x3FFu : 0x7Fu)) ? 2u : x >> 15;
                                    if (t == (uint32_t)k) kind[e] |= UNIT << h;
                                    if (t != 3u) keep[e] &= ~(0xFFFFu << h);
                                }
                            }
                            const kv_f4 n = kvs_mfma<HM>(kind, see, kv_f4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                            for (int i = 0; i < 4; i++) if (n[i] > 0.0f) acc[j][i] += k == 0 ? INFINITY : k == 1 ? -INFINITY : NAN;
                        }
                        vf = vl = keep;
                    }
                    if constexpr (NW == 2) acc[j] = kvs_mfma<HM>(vl, pf[1], acc[j]);
                    acc[j] = kvs_mfma<HM>(vf, pf[0], acc[j]);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MORE) { request_v(coming); find(c + 2 * WAVES); }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (c0 + wave < c1) {
        int c = c0 + wave;
        find(c);
        const uint32_t s = place();
        request_k(s); request_v(s);
        find(c + WAVES);
        for (; c + WAVES < c1; c += WAVES) tile(c, std::integral_constant<bool, true>());
        tile(c, std::integral_constant<bool, false>());
    }
    // ---- the waves' states meet: [waves][16][DIM + 4] sums | [waves][16] references | [waves][16] denominators | [16] largest reference | [16] denominator
    constexpr int VS = DIM + 4;
    float* ml = kvs_lds_ + WAVES * 16 * VS; float* dl = ml + WAVES * 16; float* mt = dl + WAVES * 16; float* dt = mt + 16;
    l += __shfl_xor(l, 16); l += __shfl_xor(l, 32);
    if (q == 0) { ml[wave * 16 + row] = m; dl[wave * 16 + row] = l; }
    __syncthreads();
    float top = -INFINITY, den = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) top = fmaxf(top, ml[w * 16 + row]);
    base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < WAVES; w++) den += dl[w * 16 + row] * __builtin_amdgcn_exp2f(ml[w * 16 + row] - base);
    const float f = __builtin_amdgcn_exp2f(m - base);
    float* mine = kvs_lds_ + (wave * 16 + row) * VS;
    if (wave < c1 - c0)
#pragma unroll
    for (int j = 0; j < DIM / 16; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) mine[j / C * 16 * C + (4 * q + i) * C + j % C] = m == -INFINITY ? 0.0f : acc[j][i] * f;
    if (tid < 16) { mt[tid] = top; dt[tid] = den; }
    __syncthreads();
    const bool whole = it.nsplit == 1;
    float* wo = a.ws + (size_t)idx * 16 * DIM;
    const int had = min(WAVES, c1 - c0);                      // waves that had a tile
    for (int i = tid; i < rows * (DIM / 4); i += 64 * WAVES) {
        const int rr = i / (DIM / 4), d = (i - rr * (DIM / 4)) * 4;
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int w = 0; w < had; w++) {
            const float4 x = *reinterpret_cast<const float4*>(kvs_lds_ + (w * 16 + rr) * VS + d);
            s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
        }
        if (whole) {
            const float inv = dt[rr] == 0.0f ? 0.0f : 1.0f / dt[rr];
            const int tt = (int)kv_div((uint32_t)rr, a.G), hh = it.kvh * G + rr - tt * G;
            u32x2 o = {kv_pack<HQ>(s.x * inv, s.y * inv), kv_pack<HQ>(s.z * inv, s.w * inv)};
            *reinterpret_cast<u32x2*>(a.out + ((size_t)(it.row0 + tt) * a.heads + hh) * DIM + d) = o;
        } else *reinterpret_cast<float4*>(wo + rr * DIM + d) = s;
    }
    if (!whole && tid < 16) {
        float* st = a.ws + (size_t)a.items * 16 * DIM + ((size_t)idx * 16 + tid) * 2;
        st[0] = mt[tid]; st[1] = dt[tid];
    }
}

template <int DIM, int FMT, bool HQ, bool ONE> static int kvs_launch(const KvAttnArgs& a, hipStream_t st) {
    constexpr int waves = kv_step_waves(DIM, FMT, HQ, ONE);
    constexpr size_t lds = kvs_lds(DIM, waves);
    if (lds > 65536 && kr_lds_optin((const void*)kr_kv_step_kernel<DIM, FMT, HQ, ONE>, lds)) return 1;
    hipLaunchKernelGGL((kr_kv_step_kernel<DIM, FMT, HQ, ONE>), dim3(a.items), dim3(64 * waves), lds, st, a);
    return 0;
}
template <int DIM, int FMT> static int kvs_launch(const KvAttnArgs& a, int half, hipStream_t st) {
    if (a.one) return half ? kvs_launch<DIM, FMT, true, true>(a, st) : kvs_launch<DIM, FMT, false, true>(a, st);
    return half ? kvs_launch<DIM, FMT, true, false>(a, st) : kvs_launch<DIM, FMT, false, false>(a, st);
}
template <int FMT> static int kvs_dim(const KvAttnArgs& a, int dim, int half, hipStream_t st) {
    switch (dim) {
        case 64: return kvs_launch<64, FMT>(a, half, st);
        case 96: return kvs_launch<96, FMT>(a, half, st);
        case 128: return kvs_launch<128, FMT>(a, half, st);
        case 192: return kvs_launch<192, FMT>(a, half, st);
        case 256: return kvs_launch<256, FMT>(a, half, st);
    }
    return 1;
}
