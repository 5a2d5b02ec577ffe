// AdamW over a list of tensors in one launch (gfx950): decoupled weight decay, moments in fp32 or in 8 bits.
//
//   m' = b1 m + (1 - b1) g        v' = b2 v + ((1 - b2) g) g        r = sqrt(v')
//   p' = c0 p - step (m' / (r root2 + eps))      c0 = 1 - lr wd, step = lr / (1 - b1^t), root2 = 1 / sqrt(1 - b2^t)
//
// 8 bits: VC_ADAMW_BLOCK = 256 consecutive elements share an fp32 scale top / 448 (top = the block's largest magnitude) and
// hold OCP e4m3 codes, round to nearest even.  The second moment is held by its ROOT r: a code's relative step of 2^-4 is
// then the step of the denominator itself, and the codes reach down to r = 2^-18 top instead of sqrt(2^-18) top.  A root
// that is not 0 gets the least code (2^-9) at least: rounded to 0 it would leave eps as the whole denominator of the next
// step.  The parameters move by the unrounded m' and r of this step; only what is kept for the next one is rounded.
// A block whose top is below 2^-100 is held as zeros (1 / top could leave the range; such a moment moves nothing).
// A gradient that is not finite reaches its block's scale, i.e. poisons the 256 elements that share it, as it poisons its
// own element with fp32 moments.
//
// Every product, sum, root and quotient rounds by itself (no contraction): the codes then do not depend on how a compiler
// fuses, and a step is reproducible bit for bit by elementary operations.
//
// Bound by HBM: 28 bytes per element (fp32, 32-bit moments), 16.06 (fp32, 8-bit), 10.06 (bf16, 8-bit); with 8-bit moments
// nearly as much by the VALU, so what is done once per block is shared by few lanes: a block belongs to 16 lanes of 16
// elements (its maximum is four DPP steps, its scales and reciprocals are 1/16 of a lane's work each), a wave has four.  A
// lane's elements lie in pieces of 16 bytes of p and g, neighbouring lanes' pieces beside each other.
// With 32-bit moments a lane has four elements of each of UNROLL stretches.
// Measured (copies reach 5.14 TB/s): 33.4 M fp32 parameters, 32-bit moments, 182 us = 5.14 TB/s; 357 M bf16 parameters, 8-bit
// moments, 664 us = 5.4 TB/s; 100 tensors of 42 thousand elements in all 21 us: two launches of 8 us, one behind the other, and the host.
// The tensors' addresses travel as kernel arguments (60 per launch): nothing on the device has to be written before the
// launch, so a captured step replays.
//
// Root and quotient are correctly rounded.  The compiler's sequences for that (33 issue slots together) cover every input; a
// wave whose values all lie in the middle of the range (v and |m'| in [2^-90, 2^20]) uses shorter ones (20).  With y = the correctly
// rounded reciprocal (root), q' = q + (a - b q) y is correctly rounded (P. Markstein, Computation of elementary functions on the IBM
// RISC System/6000 processor, 1990; a divisor whose mantissa is all ones is left out there).  That one Newton step makes such a y of
// the hardware's estimate does not follow: by arithmetic, an estimate one unit above the rounded reciprocal would miss it for 32
// mantissas, and one unit beside it for all ones.  It holds for this hardware's estimates (gfx950: off by one unit for 897 675 of the
// 2^23 mantissas): y compared for all 2^23, the root for all 2^24 of two octaves, the quotients by an all-ones divisor for all 2^23
// numerators.  tests/test_adamw_mantissas_gpu.py repeats the last two.
#include "common.h"
#include "kernels.h"

#pragma clang fp contract(off)

namespace {

constexpr int WAVES = 4, UNROLL = 4, BLK = VC_ADAMW_BLOCK;
constexpr int CHUNK = WAVES * UNROLL * BLK;  // elements of a workgroup

__device__ __forceinline__ f32x4 load4(const float* p, bool vec, int left) {
    if (vec && left >= 4) return *(const f32x4*)p;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) v[i] = p[i];
    return v;
}
__device__ __forceinline__ f32x4 load4(const bf16* p, bool vec, int left) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (vec && left >= 4) {
        const bf16x4 b = *(const bf16x4*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = bf2f(b[i]);
        return v;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) v[i] = bf2f(p[i]);
    return v;
}
__device__ __forceinline__ void store4(float* p, f32x4 v, bool vec, int left) {
    if (vec && left >= 4) {
        *(f32x4*)p = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) p[i] = v[i];
}
__device__ __forceinline__ void store4(bf16* p, f32x4 v, bool vec, int left) {
    if (vec && left >= 4) {
        bf16x4 b;
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = f2bf(v[i]);
        *(bf16x4*)p = b;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) p[i] = f2bf(v[i]);
}
__device__ __forceinline__ float root(float v) { return sqrtf(v); }
__device__ __forceinline__ float quotient(float a, float b) { return a / b; }
// v in [2^-90, 2^20]: s ~ sqrt v and h ~ 1 / (2 sqrt v) sharpened once, then the residual
__device__ __forceinline__ float root_mid(float v) {
    const float y = __builtin_amdgcn_rsqf(v);
    float s = v * y, h = 0.5f * y;
    const float e = __builtin_fmaf(-h, s, 0.5f);
    s = __builtin_fmaf(s, e, s);
    h = __builtin_fmaf(h, e, h);
    return __builtin_fmaf(__builtin_fmaf(-s, s, v), h, s);
}
// |a| in [2^-90, 2^20], b in [2^-45, 2^21]: nothing on the way leaves the normal numbers
__device__ __forceinline__ float quotient_mid(float a, float b) {
    float y = __builtin_amdgcn_rcpf(b);
    y = __builtin_fmaf(__builtin_fmaf(-b, y, 1.f), y, y);
    const float q = a * y;
    return __builtin_fmaf(__builtin_fmaf(-b, q, a), y, q);
}

// the tensor whose range of workgroups this one is in
__device__ __forceinline__ int tensor_of(const VcAdamwArgs& a) {
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first[mid] <= blockIdx.x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ---------------------------------------------------------------- moments in 8 bits
// largest of 16 lanes' values, as integers: of magnitudes' bits a NaN is above everything and so is kept
__device__ __forceinline__ unsigned top16(unsigned t) {
    auto step = [&](unsigned u) { t = u > t ? u : t; };
    step((unsigned)__builtin_amdgcn_update_dpp(0, (int)t, 0xB1, 0xF, 0xF, false));   // quad_perm 1 0 3 2
    step((unsigned)__builtin_amdgcn_update_dpp(0, (int)t, 0x4E, 0xF, 0xF, false));   // quad_perm 2 3 0 1
    step((unsigned)__builtin_amdgcn_update_dpp(0, (int)t, 0x141, 0xF, 0xF, false));  // row_half_mirror
    step((unsigned)__builtin_amdgcn_update_dpp(0, (int)t, 0x140, 0xF, 0xF, false));  // row_mirror
    return t;
}
// what a block's values are multiplied by for their codes, and what the codes are multiplied by
__device__ __forceinline__ float inverse(float top, float& scale) {
    const bool some = !(top < 0x1p-100f);  // (a NaN counts)
    scale = some ? top * (1.f / 448.f) : 0.f;
    return some ? (1.f / top) * 448.f : 0.f;
}
__device__ __forceinline__ unsigned encode(const float* c) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
}
__device__ __forceinline__ void decode(unsigned w, float scale, float* v) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo[0] * scale, v[1] = lo[1] * scale, v[2] = hi[0] * scale, v[3] = hi[1] * scale;
}

template <typename PT>
__global__ __launch_bounds__(WAVES * 64) void adamw8_kernel(const VcAdamwArgs a) {
    constexpr int E = 16, VE = 16 / sizeof(PT), PIECES = E / VE;  // elements of a lane, of a piece; pieces
    const int t_ = tensor_of(a);
    const VcAdamwTensor t = a.t[t_];
    const int lane = threadIdx.x & 63, l16 = lane & 15;
    const long long blk = (long long)(blockIdx.x - a.first[t_]) * (CHUNK / BLK) + (threadIdx.x >> 4);
    if (blk * BLK >= t.n) return;
    const long long base = blk * BLK + l16 * VE;  // the lane's first element; piece k is k * 16 * VE further on
    const long long rest = t.n - blk * BLK;
    PT* const P = (PT*)t.p + base;
    const PT* const G = (const PT*)t.g + base;
    uint8_t* const M = (uint8_t*)t.m + base;
    uint8_t* const V = (uint8_t*)t.v + base;
    const bool vec = rest >= BLK && (((uintptr_t)t.p | (uintptr_t)t.g) & 15) == 0 && (((uintptr_t)t.m | (uintptr_t)t.v) & (VE - 1)) == 0;
    const float gs = a.gscale != nullptr ? a.gscale_host * *a.gscale : a.gscale_host;
    float p[E], g[E], m[E], r[E];
    unsigned qm[E / 4], qv[E / 4];
    const float sm = t.ms[blk], sv = t.vs[blk];
    auto there = [&](int i) { return l16 * VE + i / VE * (16 * VE) + i % VE < rest; };
    if (vec) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int at = k * 16 * VE;
            if constexpr (sizeof(PT) == 2) {
                const bf16x8 x = *(const bf16x8*)(P + at), y = *(const bf16x8*)(G + at);
#pragma unroll
                for (int i = 0; i < 8; ++i) p[k * 8 + i] = bf2f(x[i]), g[k * 8 + i] = bf2f(y[i]);
                const uint2 x8 = *(const uint2*)(M + at), y8 = *(const uint2*)(V + at);
                qm[k * 2] = x8.x, qm[k * 2 + 1] = x8.y, qv[k * 2] = y8.x, qv[k * 2 + 1] = y8.y;
            } else {
                const f32x4 x = *(const f32x4*)(P + at), y = *(const f32x4*)(G + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[k * 4 + i] = x[i], g[k * 4 + i] = y[i];
                qm[k] = *(const unsigned*)(M + at), qv[k] = *(const unsigned*)(V + at);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) qm[i] = qv[i] = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int at = i / VE * (16 * VE) + i % VE;
            p[i] = g[i] = 0.f;
            if (there(i)) {
                p[i] = (float)P[at], g[i] = (float)G[at];
                qm[i / 4] |= (unsigned)M[at] << (i % 4 * 8), qv[i / 4] |= (unsigned)V[at] << (i % 4 * 8);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < E; i += 4) decode(qm[i / 4], sm, m + i), decode(qv[i / 4], sv, r + i);
    // r becomes v' and then its root
    constexpr unsigned LO = (127 - 90) << 23, HI = (127 + 20) << 23;
    unsigned out = 0;  // above HI - LO: some value is not in the middle of the range
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float gi = g[i] * gs;
        m[i] = m[i] * a.b1 + gi * a.one_b1;
        r[i] = (r[i] * r[i]) * a.b2 + (gi * a.one_b2) * gi;
        const unsigned x = (__float_as_uint(m[i]) & 0x7fffffffu) - LO, y = __float_as_uint(r[i]) - LO;
        out = out > x ? out : x;
        out = out > y ? out : y;
    }
    if (a.mid && __all(out <= HI - LO)) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            r[i] = root_mid(r[i]);
            p[i] = p[i] * a.c0 - quotient_mid(m[i], r[i] * a.root2 + a.eps) * a.step;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            r[i] = root(r[i]);
            p[i] = p[i] * a.c0 - quotient(m[i], r[i] * a.root2 + a.eps) * a.step;
        }
    }
    unsigned tm = 0, tr = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (!vec && !there(i)) m[i] = r[i] = 0.f;  // (behind the end: 0 whatever eps and a scale of no number made of it)
        const unsigned x = __float_as_uint(m[i]) & 0x7fffffffu, y = __float_as_uint(r[i]) & 0x7fffffffu;
        tm = tm > x ? tm : x;
        tr = tr > y ? tr : y;
    }
    float nm, nv;
    const float im = inverse(__uint_as_float(top16(tm)), nm), iv = inverse(__uint_as_float(top16(tr)), nv);
    const float least = iv > 0.f ? 0x1p-9f : 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        m[i] *= im;
        const float c = r[i] * iv;
        r[i] = c < least && r[i] > 0.f ? least : c;
    }
    if (vec) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int at = k * 16 * VE;
            if constexpr (sizeof(PT) == 2) {
                bf16x8 x;
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = f2bf(p[k * 8 + i]);
                *(bf16x8*)(P + at) = x;
                *(uint2*)(M + at) = make_uint2(encode(m + k * 8), encode(m + k * 8 + 4));
                *(uint2*)(V + at) = make_uint2(encode(r + k * 8), encode(r + k * 8 + 4));
            } else {
                *(f32x4*)(P + at) = (f32x4){p[k * 4], p[k * 4 + 1], p[k * 4 + 2], p[k * 4 + 3]};
                *(unsigned*)(M + at) = encode(m + k * 4);
                *(unsigned*)(V + at) = encode(r + k * 4);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const unsigned wm = encode(m + i), wv = encode(r + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = (i + j) / VE * (16 * VE) + (i + j) % VE;
                if (there(i + j)) {
                    P[at] = (PT)p[i + j];
                    M[at] = (uint8_t)(wm >> (8 * j)), V[at] = (uint8_t)(wv >> (8 * j));
                }
            }
        }
    }
    if (l16 == 0) t.ms[blk] = nm, t.vs[blk] = nv;
}

// ---------------------------------------------------------------- moments in 32 bits
template <typename PT>
__global__ __launch_bounds__(WAVES * 64) void adamw_kernel(const VcAdamwArgs a) {
    const int t_ = tensor_of(a);
    const VcAdamwTensor t = a.t[t_];
    PT* const P = (PT*)t.p;
    const PT* const G = (const PT*)t.g;
    float* const M = (float*)t.m;
    float* const V = (float*)t.v;
    const long long base = (long long)(blockIdx.x - a.first[t_]) * CHUNK + (threadIdx.x >> 6) * (UNROLL * BLK) + (threadIdx.x & 63) * 4;
    const bool vec = ((((uintptr_t)P | (uintptr_t)G) & (4 * sizeof(PT) - 1)) | (((uintptr_t)M | (uintptr_t)V) & 15)) == 0;
    const float gs = a.gscale != nullptr ? a.gscale_host * *a.gscale : a.gscale_host;
    f32x4 p[UNROLL], g[UNROLL], m[UNROLL], v[UNROLL];
    int left[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long long e = base + u * BLK, rest = t.n - e;
        left[u] = rest <= 0 ? 0 : rest < 4 ? (int)rest : 4;
        const long long at = left[u] > 0 ? e : 0;
        p[u] = load4(P + at, vec, left[u]);
        g[u] = load4(G + at, vec, left[u]);
        m[u] = load4(M + at, vec, left[u]);
        v[u] = load4(V + at, vec, left[u]);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        if (left[u] <= 0) break;
        const long long e = base + u * BLK;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float gi = g[u][i] * gs;
            m[u][i] = m[u][i] * a.b1 + gi * a.one_b1;
            v[u][i] = v[u][i] * a.b2 + (gi * a.one_b2) * gi;
            p[u][i] = p[u][i] * a.c0 - quotient(m[u][i], root(v[u][i]) * a.root2 + a.eps) * a.step;
        }
        store4(P + e, p[u], vec, left[u]);
        store4(M + e, m[u], vec, left[u]);
        store4(V + e, v[u], vec, left[u]);
    }
}

}  // namespace

int vc_adamw_launch(const VcAdamwTensor* t, int count, bool is_bf16, int bits, VcAdamwArgs& a, hipStream_t s) {
    a.mid = a.root2 <= 0x1p10f && a.eps <= 0x1p10f;
    for (int i = 0; i < count;) {
        a.count = 0;
        unsigned blocks = 0;
        // a launch takes up to VC_ADAMW_MAX_TENSORS tensors and fewer than 2^32 lanes (HIP's limit): 2^24 - 1 workgroups
        for (; i < count && a.count < VC_ADAMW_MAX_TENSORS; ++i) {
            if (t[i].n == 0) continue;
            const long long need = (t[i].n + CHUNK - 1) / CHUNK;
            if (a.count > 0 && blocks + need >= (1ll << 24)) break;
            a.t[a.count] = t[i];
            a.first[a.count++] = blocks;
            blocks += (unsigned)need;
        }
        if (a.count == 0) continue;
        (void)hipGetLastError();
        const dim3 grid(blocks), block(WAVES * 64);
        if (is_bf16 && bits == 8) hipLaunchKernelGGL((adamw8_kernel<bf16>), grid, block, 0, s, a);
        else if (is_bf16) hipLaunchKernelGGL((adamw_kernel<bf16>), grid, block, 0, s, a);
        else if (bits == 8) hipLaunchKernelGGL((adamw8_kernel<float>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((adamw_kernel<float>), grid, block, 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            vc_set_error("adamw launch failed: %s", hipGetErrorString(e));
            return -1;
        }
    }
    return 0;
}
