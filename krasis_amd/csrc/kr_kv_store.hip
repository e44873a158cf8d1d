// kr_kv_store.hip -- rows into a caller's cache pages, back out of them, and from slot to slot.
// Writing quantises: a microscaled block of 32 channels gets the smallest power of two 2^s with max|x| <= M 2^s (M = 448 for E4M3, 6 for E2M1; s >= -100), its elements are
// x / 2^s (exact) rounded to nearest even.  A block that holds a NaN or an infinity gets scale byte 255 and reads back as NaN.  All of it is bound by memory: a thread takes eight
// channels (16 bytes of a row) at a time, four threads a block, whose maximum they find among themselves.  49863 tokens of two heads of 256 channels read back from eight bits to f16 (155 MB)
// 24.3 us, 6.3 TB/s; three prompts of four heads of 128 stored at four bits 8.9 us and read back 7.5 (31 MB each).
#include "kr_kv_dev.h"

constexpr int KV_UNITS = 4;
__device__ __forceinline__ void kv_open8(const u32x4& w, int half, float* x) {
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

// Eight channels of a row: where they come from and where they go.  Units lie one after the other over rows, heads and channels; a thread takes KV_UNITS of them, 256 apart, so that as
// many loads are on their way together.
struct KvUnit { bool on; uint32_t row, head, c; size_t slot; };
__device__ __forceinline__ KvUnit kv_unit(const KvRowsArgs& a, int n) {
    KvUnit u;
    uint32_t in;
    u.row = kv_div(blockIdx.x * (256u * KV_UNITS) + 256u * n + threadIdx.x, a.per_row, in);
    u.on = u.row < (uint32_t)a.rows;
    u.head = kv_div(in, a.per_head, u.c);
    u.c *= 8;
    u.slot = u.on ? (uint32_t)a.slots[u.row] : 0;
    return u;
}

template <int FORMAT> __device__ __forceinline__ void kv_store(const KvRowsArgs& a, const KvUnit& u, bool key, float* x) {
    uint8_t* dst = (key ? a.p.k : a.p.v) + u.slot * a.p.row_bytes + (size_t)u.head * a.p.head_bytes;
    if constexpr (FORMAT == KR_KV_BF16 || FORMAT == KR_KV_F16) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = kv_pack<FORMAT == KR_KV_F16>(x[2 * e], x[2 * e + 1]);
        if (u.on) *reinterpret_cast<u32x4*>(dst + 2 * u.c) = w;
    } else if constexpr (FORMAT == KR_KV_E4M3) {
        if (u.on) *reinterpret_cast<u32x2*>(dst + u.c) = u32x2{kv_fp8x4(x), kv_fp8x4(x + 4)};
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
        if (u.on) {
            if constexpr (FORMAT == KR_KV_MX8) *reinterpret_cast<u32x2*>(dst + u.c) = u32x2{kv_fp8x4(x), kv_fp8x4(x + 4)};
            else {
                uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, x[0], x[1], 1.0f, 0);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], 1.0f, 1);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], 1.0f, 2);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], 1.0f, 3);
                *reinterpret_cast<uint32_t*>(dst + u.c / 2) = w;
            }
            if (!(u.c & 31)) (key ? a.p.ks : a.p.vs)[u.slot * a.p.srow_bytes + (size_t)u.head * a.p.shead_bytes + u.c / 32] = bad ? 255 : (uint8_t)(s + 127);
        }
    }
}
template <int FORMAT> __global__ void __launch_bounds__(256) kr_kv_write_kernel(const KvRowsArgs a) {
    const bool key = blockIdx.y == 0;
    const uint16_t* src = (const uint16_t*)(key ? a.k : a.v);
    const long tok = key ? a.k_tok : a.v_tok, head = key ? a.k_head : a.v_head;
    KvUnit u[KV_UNITS]; u32x4 w[KV_UNITS];
#pragma unroll
    for (int n = 0; n < KV_UNITS; n++) u[n] = kv_unit(a, n);
#pragma unroll
    for (int n = 0; n < KV_UNITS; n++) w[n] = u[n].on ? *reinterpret_cast<const u32x4*>(src + (size_t)u[n].row * tok + (size_t)u[n].head * head + u[n].c) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < KV_UNITS; n++) {
        float x[8];
        kv_open8(w[n], a.half, x);
        kv_store<FORMAT>(a, u[n], key, x);
    }
}

template <int FORMAT, bool H> __global__ void __launch_bounds__(256) kr_kv_read_kernel(const KvRowsArgs a) {
    constexpr int BYTES = FORMAT == KR_KV_MX4 ? 4 : FORMAT == KR_KV_E4M3 || FORMAT == KR_KV_MX8 ? 8 : 16;      // of a unit in the pages
    const bool key = blockIdx.y == 0;
    const uint8_t* pages = key ? a.p.k : a.p.v; const uint8_t* scales = key ? a.p.ks : a.p.vs;
    uint16_t* dst = (uint16_t*)(key ? a.k : a.v);
    const long tok = key ? a.k_tok : a.v_tok, head = key ? a.k_head : a.v_head;
    KvUnit u[KV_UNITS]; uint32_t w[KV_UNITS][BYTES / 4]; uint32_t byte[KV_UNITS];
#pragma unroll
    for (int n = 0; n < KV_UNITS; n++) u[n] = kv_unit(a, n);
#pragma unroll
    for (int n = 0; n < KV_UNITS; n++) {
        if (!u[n].on) continue;
        const uint8_t* src = pages + u[n].slot * a.p.row_bytes + (size_t)u[n].head * a.p.head_bytes + u[n].c * BYTES / 8;
        if constexpr (BYTES == 16) { const u32x4 x = *reinterpret_cast<const u32x4*>(src); w[n][0] = x.x; w[n][1] = x.y; w[n][2] = x.z; w[n][3] = x.w; }
        else if constexpr (BYTES == 8) { const u32x2 x = *reinterpret_cast<const u32x2*>(src); w[n][0] = x.x; w[n][1] = x.y; }
        else w[n][0] = *reinterpret_cast<const uint32_t*>(src);
        byte[n] = 127;
        if constexpr (FORMAT == KR_KV_MX8 || FORMAT == KR_KV_MX4) byte[n] = scales[u[n].slot * a.p.srow_bytes + (size_t)u[n].head * a.p.shead_bytes + u[n].c / 32];
    }
#pragma unroll
    for (int n = 0; n < KV_UNITS; n++) {
        if (!u[n].on) continue;
        u32x4 o;
        if constexpr (BYTES == 16) {
            o = u32x4{w[n][0], w[n][1], w[n][2], w[n][3]};
            if constexpr (H != (FORMAT == KR_KV_F16)) {
                float x[8];
                kv_open8(o, FORMAT == KR_KV_F16, x);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = kv_pack<H>(x[2 * e], x[2 * e + 1]);
            }
        } else {
            const float sc = kv_scale(byte[n]);
            if constexpr (BYTES == 4) o = u32x4{kv_pair<2, 0>(w[n][0], sc), kv_pair<2, 1>(w[n][0], sc), kv_pair<2, 2>(w[n][0], sc), kv_pair<2, 3>(w[n][0], sc)};
            else o = u32x4{kv_pair<1, 0>(w[n][0], sc), kv_pair<1, 1>(w[n][0], sc), kv_pair<1, 0>(w[n][BYTES / 4 - 1], sc), kv_pair<1, 1>(w[n][BYTES / 4 - 1], sc)};
            if constexpr (H) {                       // bf16 holds the value: one rounding
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = kv_pack<true>(kv_lo(o[e]), kv_hi(o[e]));
            }
        }
        *reinterpret_cast<u32x4*>(dst + (size_t)u[n].row * tok + (size_t)u[n].head * head + u[n].c) = o;
    }
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

static dim3 kv_rows_grid(const KvRowsArgs& a) { return dim3((unsigned)(((uint64_t)a.rows * a.per_row.d + 256 * KV_UNITS - 1) / (256 * KV_UNITS)), 2); }
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
