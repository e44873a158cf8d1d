// kr_kv_join.hip -- the second launch of attention over the paged cache, where sequences were shared out among workgroups.
#include "kr_kv_dev.h"

// Shares of split sequences joined.  FEW (16 shares at most): a unit is 16 rows of a row tile and one head, a thread holds four columns of a row and walks the shares, four at a time.  Else a unit is
// one row: its threads divide the shares among themselves and meet in LDS.  Bound by its three round trips (place, weights, sums): 4.7 us for the shares of 32 requests' single tokens, 5.2 for 32
// shares of two, 6.9 for 22 shares of 96 rows of eight sequences.
template <bool H, bool FEW> __global__ void __launch_bounds__(256) kr_kv_join_kernel(const KvAttnArgs a, int dim, int bm, int kt, KvDiv sub) {
    const KvItem it = kv_item<false>(a, blockIdx.x, bm, kt, sub);
    if (it.b < 0) return;
    const int G = (int)a.G.d, rows = it.cnt * G, quads = dim / 4, tid = threadIdx.x, first = kv_item_of(a, it, 0), step = (int)a.kv_heads.d;      // a row tile's shares lie kv_heads items apart
    const float* stats = a.ws + (size_t)a.items * bm * dim;
    if constexpr (FEW) {
        for (int i = tid; i < 16 * quads; i += 256) {
            const int r = it.split * 16 + i / quads, d = i % quads * 4, rr = it.rt * bm + r;
            if (rr >= rows) continue;
            float top = -INFINITY, den = 0.0f; float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float* sp = stats + ((size_t)first * bm + r) * 2; const float* wp = a.ws + ((size_t)first * bm + r) * dim + d;
            const size_t next = (size_t)step * bm;
            for (int s0 = 0; s0 < it.nsplit; s0 += 4) {       // four shares at a time, measured from the largest reference so far
                float ms[4], ls[4]; float4 x[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const size_t s = (size_t)min(s0 + u, it.nsplit - 1) * next;
                    ms[u] = sp[s * 2]; ls[u] = sp[s * 2 + 1]; x[u] = *reinterpret_cast<const float4*>(wp + s * dim);
                }
                const float mx = fmaxf(fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), top), base = mx == -INFINITY ? 0.0f : mx, was = __builtin_amdgcn_exp2f(top - base);
                if (s0) { o.x *= was; o.y *= was; o.z *= was; o.w *= was; den *= was; }
                top = mx;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    if (s0 + u >= it.nsplit || (ms[u] == -INFINITY && ls[u] == 0.0f)) continue;      // a share without keys of this row
                    const float f = __builtin_amdgcn_exp2f(ms[u] - base);
                    o.x += x[u].x * f; o.y += x[u].y * f; o.z += x[u].z * f; o.w += x[u].w * f;
                    den += ls[u] * f;
                }
            }
            const float inv = den == 0.0f ? 0.0f : 1.0f / den;
            const int t = (int)kv_div((uint32_t)rr, a.G), h = it.kvh * G + rr - t * G;
            *reinterpret_cast<u32x2*>(a.out + ((size_t)(it.row0 + t) * a.heads + h) * dim + d) = u32x2{kv_pack<H>(o.x * inv, o.y * inv), kv_pack<H>(o.z * inv, o.w * inv)};
        }
    } else {
        __shared__ float wl[KV_MAX_SHARES], dl[KV_MAX_SHARES]; __shared__ float red[8]; __shared__ float4 sums[256];
        const int r = it.split, rr = it.rt * bm + r;
        if (rr >= rows) return;
        const int groups = 256 / quads, g = tid / quads, d = tid % quads * 4;
        const float* wp = a.ws + ((size_t)first * bm + r) * dim + d; const size_t next = (size_t)step * bm * dim;
        float4 x[4];                                          // a thread's first shares, on their way while the weights are found
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = *reinterpret_cast<const float4*>(wp + (size_t)min(g + u * groups, it.nsplit - 1) * next);
        float top = -INFINITY, den = 0.0f;
        for (int s = tid; s < it.nsplit; s += 256) {
            const float2 st = *reinterpret_cast<const float2*>(stats + ((size_t)(first + s * step) * bm + r) * 2);
            wl[s] = st.x; dl[s] = st.y; top = fmaxf(top, st.x);
        }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
        if ((tid & 63) == 0) red[tid >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float base = top == -INFINITY ? 0.0f : top;
        for (int s = tid; s < it.nsplit; s += 256) {
            const bool none = wl[s] == -INFINITY && dl[s] == 0.0f;
            const float f = none ? -1.0f : __builtin_amdgcn_exp2f(wl[s] - base);      // -1: a share without keys of this row
            if (!none) den += dl[s] * f;
            wl[s] = f;
        }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) den += __shfl_xor(den, k);
        if ((tid & 63) == 0) red[4 + (tid >> 6)] = den;
        __syncthreads();
        den = red[4] + red[5] + red[6] + red[7];
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (g < groups) {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int s = g + u * groups;
                if (s >= it.nsplit || wl[s] == -1.0f) continue;
                const float f = wl[s];
                o.x += x[u].x * f; o.y += x[u].y * f; o.z += x[u].z * f; o.w += x[u].w * f;
            }
#pragma unroll 4
            for (int s = g + 4 * groups; s < it.nsplit; s += groups) {
                const float f = wl[s];
                const float4 y = *reinterpret_cast<const float4*>(wp + (size_t)s * next);
                if (f != -1.0f) { o.x += y.x * f; o.y += y.y * f; o.z += y.z * f; o.w += y.w * f; }
            }
        }
        sums[tid] = o;
        __syncthreads();
        if (tid >= quads) return;
        for (int k = 1; k < groups; k++) { const float4 y = sums[k * quads + tid]; o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w; }
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        const int t = (int)kv_div((uint32_t)rr, a.G), h = it.kvh * G + rr - t * G;
        *reinterpret_cast<u32x2*>(a.out + ((size_t)(it.row0 + t) * a.heads + h) * dim + d) = u32x2{kv_pack<H>(o.x * inv, o.y * inv), kv_pack<H>(o.z * inv, o.w * inv)};
    }
}
int kr_launch_kv_join(const KvAttnArgs& a, int dim, int bm, int kt, int units, int few, int half, hipStream_t st) {
    const KvDiv sub = kv_divisor((uint32_t)(few ? bm / 16 : bm));
    if (few) {
        if (half) hipLaunchKernelGGL((kr_kv_join_kernel<true, true>), dim3(units), dim3(256), 0, st, a, dim, bm, kt, sub);
        else hipLaunchKernelGGL((kr_kv_join_kernel<false, true>), dim3(units), dim3(256), 0, st, a, dim, bm, kt, sub);
    } else {
        if (half) hipLaunchKernelGGL((kr_kv_join_kernel<true, false>), dim3(units), dim3(256), 0, st, a, dim, bm, kt, sub);
        else hipLaunchKernelGGL((kr_kv_join_kernel<false, false>), dim3(units), dim3(256), 0, st, a, dim, bm, kt, sub);
    }
    return 0;
}
