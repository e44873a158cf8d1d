// kr_kv_store.hip -- rows into a caller's cache pages, back out of them, and from slot to slot.
// Writing quantises: a microscaled block of 32 channels gets the smallest power of two 2^s with max|x| <= M 2^s (M = 448 for E4M3, 6 for E2M1; s >= -100), its elements are
// x / 2^s (exact) rounded to nearest even.  A block that holds a NaN or an infinity gets scale byte 255 and reads back as NaN.  All of it is bound by memory: a thread takes eight
// channels (16 bytes of a row), four threads a block, whose maximum they find among themselves.
#include "kr_kv_dev.h"

__device__ __forceinline__ void kv_load8(const uint16_t* p, int half, float* x) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (half) { const kv_h2 h = kv_halves(w[e]); x[2 * e] = (float)h[0]; x[2 * e + 1] = (float)h[1]; }
        else { x[2 * e] = kv_lo(w[e]); x[2 * e + 1] = kv_hi(w[e]); }
    }
}
__device__ __forceinline__ uint32_t kv_fp8x4(const float* x) {      // magnitudes over 464, half way to the next step, have no number: NaN
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = __builtin_amdgcn_fmed3f(x[i], -448.0f, 448.0f);
    uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
#pragma unroll
    for (int i = 0; i < 4; i++) if (!(fabsf(x[i]) <= 464.0f)) w = (w & ~(0xFFu << 8 * i)) | (0x7Fu | (__float_as_uint(x[i]) >> 24 & 0x80u)) << 8 * i;
    return w;
}

template <int FORMAT> __global__ void __launch_bounds__(256) kr_kv_write_kernel(const KvRowsArgs a) {
    const uint32_t per = (uint32_t)(a.kv_heads * a.dim / 8), i = blockIdx.x * 256u + threadIdx.x, row = i / per;
    const bool on = row < (uint32_t)a.rows;
    const uint32_t u = i - row * per, head = u / (uint32_t)(a.dim / 8), c = (u - head * (a.dim / 8)) * 8;
    const bool key = blockIdx.y == 0;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    size_t slot = 0;
    if (on) {
        slot = (uint32_t)a.slots[row];
        const uint16_t* src = key ? (const uint16_t*)a.k + (size_t)row * a.k_tok + (size_t)head * a.k_head : (const uint16_t*)a.v + (size_t)row * a.v_tok + (size_t)head * a.v_head;
        kv_load8(src + c, a.half, x);
    }
    uint8_t* dst = (key ? a.p.k : a.p.v) + slot * a.p.row_bytes + (size_t)head * a.p.head_bytes;
    if constexpr (FORMAT == KR_KV_BF16 || FORMAT == KR_KV_F16) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = kv_pack<FORMAT == KR_KV_F16>(x[2 * e], x[2 * e + 1]);
        if (on) *reinterpret_cast<u32x4*>(dst + 2 * c) = w;
    } else if constexpr (FORMAT == KR_KV_E4M3) {
        if (on) *reinterpret_cast<u32x2*>(dst + c) = u32x2{kv_fp8x4(x), kv_fp8x4(x + 4)};
    } else {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);      // as integers a NaN and an infinity are the largest
        top = max(top, (uint32_t)KR_DPP((int)top, KR_DPP_XOR1));
        top = max(top, (uint32_t)KR_DPP((int)top, KR_DPP_XOR2));
        const bool bad = top >= 0x7F800000u;
        constexpr int STEP = FORMAT == KR_KV_MX8 ? 8 : 2;                       // 448 = 1.75 2^8, 6 = 1.5 2^2
        constexpr uint32_t LEAD = FORMAT == KR_KV_MX8 ? 0x600000u : 0x400000u;
        int s = (int)(top >> 23) - 127 - STEP + ((top & 0x7FFFFFu) > LEAD ? 1 : 0);
        s = bad ? 0 : max(s, -100);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = bad ? 0.0f : ldexpf(x[e], -s);
        if (on) {
            if constexpr (FORMAT == KR_KV_MX8) *reinterpret_cast<u32x2*>(dst + c) = u32x2{kv_fp8x4(x), kv_fp8x4(x + 4)};
            else {
                uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, x[0], x[1], 1.0f, 0);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], 1.0f, 1);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], 1.0f, 2);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], 1.0f, 3);
                *reinterpret_cast<uint32_t*>(dst + c / 2) = w;
            }
            if (!(c & 31)) (key ? a.p.ks : a.p.vs)[slot * a.p.srow_bytes + (size_t)head * a.p.shead_bytes + c / 32] = bad ? 255 : (uint8_t)(s + 127);
        }
    }
}

template <int FORMAT, bool H> __global__ void __launch_bounds__(256) kr_kv_read_kernel(const KvRowsArgs a) {
    const uint32_t per = (uint32_t)(a.kv_heads * a.dim / 8), i = blockIdx.x * 256u + threadIdx.x, row = i / per;
    if (row >= (uint32_t)a.rows) return;
    const uint32_t u = i - row * per, head = u / (uint32_t)(a.dim / 8), c = (u - head * (a.dim / 8)) * 8;
    const bool key = blockIdx.y == 0;
    const size_t slot = (uint32_t)a.slots[row];
    const uint8_t* src = (key ? a.p.k : a.p.v) + slot * a.p.row_bytes + (size_t)head * a.p.head_bytes;
    uint16_t* dst = key ? (uint16_t*)a.k + (size_t)row * a.k_tok + (size_t)head * a.k_head : (uint16_t*)a.v + (size_t)row * a.v_tok + (size_t)head * a.v_head;
    u32x4 o;
    if constexpr (FORMAT == KR_KV_BF16 || FORMAT == KR_KV_F16) {
        if constexpr (H == (FORMAT == KR_KV_F16)) o = *reinterpret_cast<const u32x4*>(src + 2 * c);
        else {
            float x[8];
            kv_load8((const uint16_t*)src + c, FORMAT == KR_KV_F16, x);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = kv_pack<H>(x[2 * e], x[2 * e + 1]);
        }
    } else {
        const float sc = FORMAT == KR_KV_E4M3 ? 1.0f : kv_scale((key ? a.p.ks : a.p.vs)[slot * a.p.srow_bytes + (size_t)head * a.p.shead_bytes + c / 32]);
        if constexpr (FORMAT == KR_KV_MX4) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(src + c / 2);
            o = u32x4{kv_pair<2, 0>(w, sc), kv_pair<2, 1>(w, sc), kv_pair<2, 2>(w, sc), kv_pair<2, 3>(w, sc)};
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(src + c);
            o = u32x4{kv_pair<1, 0>(w.x, sc), kv_pair<1, 1>(w.x, sc), kv_pair<1, 0>(w.y, sc), kv_pair<1, 1>(w.y, sc)};
        }
        if constexpr (H) {                       // bf16 holds the value: one rounding
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = kv_pack<true>(kv_lo(o[e]), kv_hi(o[e]));
        }
    }
    *reinterpret_cast<u32x4*>(dst + c) = o;
}

// Rows of accepted drafts move down to their places.  A path's sources never lie before their targets and both rise, so rows moved in order are never overwritten before they are
// read: a thread takes one piece of all rows of a sequence, one after the other.
__global__ void __launch_bounds__(64) kr_kv_move_kernel(const KvMoveArgs a) {
    const int seq = blockIdx.z, layer = blockIdx.y % a.layers, which = blockIdx.y / a.layers, lo = a.start[seq], hi = a.start[seq + 1];
    const int bytes = a.row_bytes[which], at = (blockIdx.x * 64 + threadIdx.x) * (which < 2 ? 16 : 1);
    if (at >= bytes) return;
    uint8_t* base = a.base[which] + (size_t)layer * a.layer_bytes[which] + at;
    for (int i = lo; i < hi; i++) {
        const size_t s = (size_t)(uint32_t)a.src[i] * bytes, d = (size_t)(uint32_t)a.dst[i] * bytes;
        if (which < 2) *reinterpret_cast<u32x4*>(base + d) = *reinterpret_cast<const u32x4*>(base + s);
        else base[d] = base[s];
    }
}

static dim3 kv_rows_grid(const KvRowsArgs& a) { return dim3((unsigned)(((uint64_t)a.rows * (a.kv_heads * a.dim / 8) + 255) / 256), 2); }
int kr_launch_kv_write(const KvRowsArgs& a, hipStream_t st) {
    switch (a.format) {
#define KV_CASE(F) case F: hipLaunchKernelGGL((kr_kv_write_kernel<F>), kv_rows_grid(a), dim3(256), 0, st, a); break
        KV_CASE(KR_KV_BF16); KV_CASE(KR_KV_F16); KV_CASE(KR_KV_E4M3); KV_CASE(KR_KV_MX8); KV_CASE(KR_KV_MX4);
#undef KV_CASE
        default: return 1;
    }
    return 0;
}
int kr_launch_kv_read(const KvRowsArgs& a, hipStream_t st) {
    switch (a.format) {
#define KV_CASE(F) case F: if (a.half) hipLaunchKernelGGL((kr_kv_read_kernel<F, true>), kv_rows_grid(a), dim3(256), 0, st, a); \
                           else hipLaunchKernelGGL((kr_kv_read_kernel<F, false>), kv_rows_grid(a), dim3(256), 0, st, a); break
        KV_CASE(KR_KV_BF16); KV_CASE(KR_KV_F16); KV_CASE(KR_KV_E4M3); KV_CASE(KR_KV_MX8); KV_CASE(KR_KV_MX4);
#undef KV_CASE
        default: return 1;
    }
    return 0;
}
int kr_launch_kv_move(const KvMoveArgs& a, hipStream_t st) {
    const int parts = a.row_bytes[2] ? 4 : 2, wide = (a.row_bytes[0] / 16 + 63) / 64, fine = (a.row_bytes[2] + 63) / 64;
    hipLaunchKernelGGL(kr_kv_move_kernel, dim3(wide > fine ? wide : fine, parts * a.layers, a.n_seq), dim3(64), 0, st, a);
    return 0;
}
