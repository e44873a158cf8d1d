// kr_kv_tile.hip -- attention over the paged cache for sequences with more than 16 rows of new tokens: prompts and their portions, drafted trees.
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over the stored keys j that row i sees; a row is a new token with one head of a group, so that a tile of keys serves the whole group.
// 4 * 128 operations a channel of a key against four bytes at most: the matrix cores bound it.  A workgroup takes 128 rows (four waves of 32), one key / value head and a share of the
// key tiles.  Tiles of 64 keys come from the pages into registers one tile ahead, are converted there (exact, kr_kv_dev.h) and stand in LDS as rows of 16-bit numbers.
//   S^T[key][row] = K Q^T    v_mfma_f32_32x32x16: queries stay in registers; a lane's 32 scores belong to one row, whose softmax is lane-local but for one exchange
//   O^T[d][row] += V^T P^T   the weights go from the accumulators to the operand in place (the order of keys within a product is free); V's columns come from the transposing LDS read
#include "kr_kv_dev.h"
#include "kr_lds_optin.h"

typedef __fp16 kvt_h4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
constexpr int KT = KV_TILE_KT, BM = KV_TILE_BM;
constexpr int kvt_ldk(int dim) { return 2 * dim + 16; }                                   // neighbouring rows four banks apart: reads of 16 bytes down the keys
constexpr int kvt_ldv(int dim) { return (2 * dim) % 128 == 64 ? 2 * dim : 2 * dim + 64; }   // an odd multiple of 64 bytes: the transposing read takes 64 bytes of eight rows
constexpr int kvt_lds(int dim) { return KT * (kvt_ldk(dim) + kvt_ldv(dim)) + 2 * KT * 4 + KV_MAX_TREE * 4 + 16; }

template <bool H> __device__ __forceinline__ kv_f16 kvt_mfma(u32x4 x, u32x4 y, kv_f16 c) {
    if constexpr (H) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(kv_h8, x), __builtin_bit_cast(kv_h8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(kv_b8, x), __builtin_bit_cast(kv_b8, y), c, 0, 0, 0);
}

template <int DIM, int FMT, bool HQ>
__global__ void __launch_bounds__(256, DIM <= 128 ? 2 : 1) kr_kv_tile_kernel(const KvAttnArgs a) {
    constexpr bool HM = HQ && FMT == 0;
    constexpr int NP = HQ && !HM ? 2 : 1;                     // bf16 pieces of an f16 query and of its weights
    constexpr int BITS = FMT == 0 ? 16 : FMT == 1 ? 8 : 4, CPR = DIM * BITS / 128, NCH = KT * CPR, PT = (NCH + 255) / 256, CD = 128 / BITS;      // chunks of 16 bytes, CD channels
    constexpr int LDK = kvt_ldk(DIM), LDV = kvt_ldv(DIM), KS = DIM / 16, DB = DIM / 32;
    extern __shared__ __attribute__((aligned(16))) char kvt_lds_[];
    char* Ks = kvt_lds_; char* Vs = Ks + KT * LDK;
    int* Sl = (int*)(Vs + KT * LDV);                          // [2][KT] slots of a tile's keys
    int* Dp = Sl + 2 * KT;                                    // [KV_MAX_TREE] depths of the drafts
    int* Odd = Dp + KV_MAX_TREE;                              // tile (plus one) that last held a value which is not finite
    const KvItem it = kv_item<true>(a, blockIdx.x, BM, KT, 1);
    if (it.b < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, h = lane >> 5;
    const KvRange rg = kv_range(a, it, BM, KT);
    const int c0 = it.split * a.tps, c1 = min(rg.tiles, c0 + a.tps);
    const int rows = it.cnt * a.G, rw = it.rt * BM + wave * 32, r = min(rw + col, rows - 1), t = r / a.G, head = it.kvh * a.G + r - t * a.G;
    const bool live = rw < rows;                              // some row of the wave is there
    const int w0 = rw / a.G, w1 = min(it.cnt - 1, (rw + 31) / a.G);      // its first and last token
    const int* table = a.s.pages + it.page0;
    const bool scaled = FMT != 0 && a.p.ks != nullptr;

    int pos = rg.before + t; uint64_t seen = 0;
    if (a.parents) {
        const uint64_t all = kv_ancestors(a.parents + it.row0, it.cnt, lane);
        const int depth = __popcll(all) - 1;
        seen = (uint64_t)__shfl((uint32_t)(all >> 32), t) << 32 | __shfl((uint32_t)all, t);
        pos = rg.before + __shfl(depth, t);
        if (tid < KV_MAX_TREE) Dp[tid] = depth;
    }
    u32x4 qf[NP][KS];
    {
        const uint16_t* qp = a.q + (size_t)(it.row0 + t) * a.q_tok + (size_t)head * a.q_head + 8 * h;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(qp + 16 * i);
            if constexpr (NP == 1) qf[0][i] = x;
            else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const kv_h2 y = kv_halves(x[e]);
                    const float u = (float)y[0], w = (float)y[1];
                    qf[0][i][e] = kv_pack<false>(u, w); qf[1][i][e] = kv_rest(u, w, qf[0][i][e]);
                }
            }
        }
    }
    auto first_key = [&](int c) { return c < rg.kept ? KT * c : rg.start + KT * (c - rg.kept); };
    auto slot = [&](int c, int k) {                           // keys no row sees give way to one that is seen
        const int j = first_key(c) + k;
        return (int)kv_slot(a.p, table, (uint32_t)(j < rg.lo && j >= a.first ? rg.lo : min(j, rg.hi - 1)));
    };
    u32x4 kn[PT], vn[PT]; uint32_t ksn[PT], vsn[PT];
    auto request = [&](int buf) {
#pragma unroll
        for (int j = 0; j < PT; j++) {
            const int c = tid + 256 * j;
            if (NCH % 256 && c >= NCH) break;
            const int row = c / CPR, dc = c - row * CPR;
            const size_t sl = (uint32_t)Sl[buf * KT + row], off = sl * a.p.row_bytes + (size_t)it.kvh * a.p.head_bytes + dc * 16;
            kn[j] = *reinterpret_cast<const u32x4*>(a.p.k + off); vn[j] = *reinterpret_cast<const u32x4*>(a.p.v + off);
            if (scaled) {
                const size_t so = sl * a.p.srow_bytes + (size_t)it.kvh * a.p.shead_bytes + dc * CD / 32;
                ksn[j] = a.p.ks[so]; vsn[j] = a.p.vs[so];
            }
        }
    };
    auto convert = [&](const u32x4& w, uint32_t s, uint32_t* o) {      // 16 bytes of codes as CD numbers
        const float sc = scaled ? kv_scale(s) : 1.0f;
        if constexpr (FMT == 0) { o[0] = w.x; o[1] = w.y; o[2] = w.z; o[3] = w.w; }
        else if constexpr (FMT == 1) {
#pragma unroll
            for (int e = 0; e < 4; e++) { o[2 * e] = kv_pair<1, 0>(w[e], sc); o[2 * e + 1] = kv_pair<1, 1>(w[e], sc); }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) { o[4 * e] = kv_pair<2, 0>(w[e], sc); o[4 * e + 1] = kv_pair<2, 1>(w[e], sc); o[4 * e + 2] = kv_pair<2, 2>(w[e], sc); o[4 * e + 3] = kv_pair<2, 3>(w[e], sc); }
        }
    };
    constexpr uint32_t EXP = HM ? 0x7C00u : 0x7F80u, ONE = HM ? 0x3C00u : 0x3F80u;
    // every row from token ta to token tb sees all keys of the tile
    auto open = [&](int c, int ta, int tb) {
        const int j0 = first_key(c), jn = c < rg.kept ? min(a.first, rg.hi) : rg.hi;
        if (j0 + KT > jn || j0 + KT - 1 > rg.before + (a.parents ? -1 : ta)) return false;
        return a.window <= 0 || rg.before + tb - j0 < a.window || j0 + KT <= a.first;
    };
    if (tid < 2 * KT && c0 + (tid / KT) < c1) Sl[tid] = slot(c0 + tid / KT, tid % KT);
    if (tid == 0) *Odd = 0;
    __syncthreads();
    if (c0 < c1) request(0);

    float m = -INFINITY, l = 0.0f;
    kv_f16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    const char* kl = Ks + col * LDK + 16 * h;
    const char* vl = Vs + (4 * h + ((lane & 15) >> 2)) * LDV + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
    for (int c = c0; c < c1; c++) {
        // A value that is not finite may belong to a key that some rows do not see, and 0 times it would not be 0: tiles that are not open to all rows are looked at.
        const bool ragged = !open(c, rg.t0, rg.t1 - 1);
#pragma unroll
        for (int j = 0; j < PT; j++) {
            const int ch = tid + 256 * j;
            if (NCH % 256 && ch >= NCH) break;
            const int row = ch / CPR, dc = ch - row * CPR;
            uint32_t w[CD / 2];
            convert(kn[j], ksn[j], w);
#pragma unroll
            for (int e = 0; e < CD / 8; e++) *reinterpret_cast<u32x4*>(Ks + row * LDK + (dc * CD + 8 * e) * 2) = u32x4{w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]};
            convert(vn[j], vsn[j], w);
            if (ragged) {
                bool odd = false;
#pragma unroll
                for (int e = 0; e < CD / 2; e++) odd = odd || (w[e] & EXP) == EXP || (w[e] >> 16 & EXP) == EXP;
                if (odd) *Odd = c + 1;
            }
#pragma unroll
            for (int e = 0; e < CD / 8; e++) *reinterpret_cast<u32x4*>(Vs + row * LDV + (dc * CD + 8 * e) * 2) = u32x4{w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]};
        }
        __syncthreads();
        if (c + 1 < c1) request((c + 1 - c0) & 1);
        int ahead = 0;
        if (tid < KT && c + 2 < c1) ahead = slot(c + 2, tid);
        const int j0 = first_key(c);
        if (live && j0 <= rg.before + w1) {
            kv_f16 st[2];
#pragma unroll
            for (int b = 0; b < 2; b++) {
#pragma unroll
                for (int i = 0; i < 16; i++) st[b][i] = 0.0f;
#pragma unroll
                for (int i = 0; i < KS; i++) {
                    const u32x4 kf = *reinterpret_cast<const u32x4*>(kl + 32 * b * LDK + 32 * i);
#pragma unroll
                    for (int p = NP - 1; p >= 0; p--) st[b] = kvt_mfma<HM>(kf, qf[p][i], st[b]);
                }
            }
            const bool mask = !open(c, w0, w1);
            float cm = -INFINITY;
            if (mask) {
                const int end = c < rg.kept ? min(a.first, rg.hi) : rg.hi;
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int key = j0 + 32 * b + (i & 3) + 8 * (i >> 2) + 4 * h;
                        int at = key; bool ok = key < end;
                        if (a.parents) {
                            const int n = key - rg.before;
                            if (n >= 0) { at = rg.before + Dp[n & (KV_MAX_TREE - 1)]; ok = ok && (seen >> (n & 63) & 1); }
                        } else ok = ok && key <= pos;
                        if (a.window > 0) ok = ok && (pos - at < a.window || at < a.first);
                        st[b][i] = ok ? st[b][i] * a.scale_log2 : -INFINITY;
                        cm = fmaxf(cm, st[b][i]);
                    }
            } else {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) { st[b][i] *= a.scale_log2; cm = fmaxf(cm, st[b][i]); }
            }
            cm = fmaxf(cm, __shfl_xor(cm, 32));
            const float mn = fmaxf(m, cm), base = mn == -INFINITY ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m - base);
            m = mn; l *= alpha;
            u32x4 pf[NP][2][2], vis[2][2];
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(st[b][i] - base), p1 = __builtin_amdgcn_exp2f(st[b][i + 1] - base);
                    l += p0 + p1;
                    const uint32_t w = kv_pack<HM>(p0, p1);
                    pf[0][b][i >> 3][(i & 7) >> 1] = w;
                    if constexpr (NP == 2) pf[1][b][i >> 3][(i & 7) >> 1] = kv_rest(p0, p1, w);
                }
            if (__any(alpha != 1.0f)) {
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[d][i] *= alpha;
            }
            const bool odd = ragged && *Odd == c + 1;
            if (odd) {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int i = 0; i < 16; i += 2) vis[b][i >> 3][(i & 7) >> 1] = (st[b][i] == -INFINITY ? 0u : ONE) | (st[b][i + 1] == -INFINITY ? 0u : ONE << 16);
            }
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const char* va = vl + 16 * s * LDV + 64 * d;
                    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) kvt_h4*)(va)));
                    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) kvt_h4*)(va + 8 * LDV)));
                    u32x4 vf = {x.x, x.y, y.x, y.y};
                    if (odd) {                                // such values apart: whether a row sees one, by kind
                        u32x4 kind[3];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t keep = 0; kind[0][e] = kind[1][e] = kind[2][e] = 0;
#pragma unroll
                            for (int u = 0; u < 32; u += 16) {
                                const uint32_t z = vf[e] >> u & 0xFFFFu;
                                if ((z & EXP) != EXP) keep |= z << u;
                                else if (z & (HM ? 0x3FFu : 0x7Fu)) kind[2][e] |= ONE << u;
                                else if (z & 0x8000u) kind[1][e] |= ONE << u;
                                else kind[0][e] |= ONE << u;
                            }
                            vf[e] = keep;
                        }
#pragma unroll
                        for (int k = 0; k < 3; k++) {
                            kv_f16 zero;
#pragma unroll
                            for (int i = 0; i < 16; i++) zero[i] = 0.0f;
                            const kv_f16 n = kvt_mfma<HM>(kind[k], vis[s >> 1][s & 1], zero);
#pragma unroll
                            for (int i = 0; i < 16; i++) if (n[i] > 0.0f) o[d][i] += k == 0 ? INFINITY : k == 1 ? -INFINITY : NAN;
                        }
                    }
#pragma unroll
                    for (int p = NP - 1; p >= 0; p--) o[d] = kvt_mfma<HM>(vf, pf[p][s >> 1][s & 1], o[d]);
                }
        }
        __syncthreads();
        if (tid < KT && c + 2 < c1) Sl[((c - c0) & 1) * KT + tid] = ahead;
    }
    l += __shfl_xor(l, 32);
    if (rw + col >= rows) return;
    if (it.nsplit == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* op = a.out + ((size_t)(it.row0 + t) * a.heads + head) * DIM + 4 * h;
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

template <int DIM, int FMT> static int kvt_launch(const KvAttnArgs& a, int half, hipStream_t st) {
    constexpr size_t lds = kvt_lds(DIM);
    const void* fn = half ? (const void*)kr_kv_tile_kernel<DIM, FMT, true> : (const void*)kr_kv_tile_kernel<DIM, FMT, false>;
    if (lds > 65536 && kr_lds_optin(fn, lds)) return 1;
    if (half) hipLaunchKernelGGL((kr_kv_tile_kernel<DIM, FMT, true>), dim3(a.items), dim3(256), lds, st, a);
    else hipLaunchKernelGGL((kr_kv_tile_kernel<DIM, FMT, false>), dim3(a.items), dim3(256), lds, st, a);
    return 0;
}
template <int FMT> static int kvt_dim(const KvAttnArgs& a, int dim, int half, hipStream_t st) {
    switch (dim) {
        case 64: return kvt_launch<64, FMT>(a, half, st);
        case 96: return kvt_launch<96, FMT>(a, half, st);
        case 128: return kvt_launch<128, FMT>(a, half, st);
        case 192: return kvt_launch<192, FMT>(a, half, st);
        case 256: return kvt_launch<256, FMT>(a, half, st);
    }
    return 1;
}
int kr_launch_kv_tile(const KvAttnArgs& a, int dim, int fmt, int half, hipStream_t st) {
    return fmt == 0 ? kvt_dim<0>(a, dim, half, st) : fmt == 1 ? kvt_dim<1>(a, dim, half, st) : kvt_dim<2>(a, dim, half, st);
}
