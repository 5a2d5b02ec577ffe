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
// Bound by HBM: 28 bytes per element (fp32, 32-bit moments), 16.06 (fp32, 8-bit), 10.06 (bf16, 8-bit).  One wave owns
// whole blocks of 256 elements, four per lane, so that a block's maximum is a butterfly over the wave and its codes are one
// dword per lane; UNROLL blocks per wave keep their loads in flight together.  The tensors' addresses travel as kernel
// arguments (64 per launch): nothing on the device has to be written before the launch, so a captured step replays.
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
// four e4m3 codes as one dword
__device__ __forceinline__ unsigned load_codes(const uint8_t* p, bool vec, int left) {
    if (vec && left >= 4) return *(const unsigned*)p;
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) w |= (unsigned)p[i] << (8 * i);
    return w;
}
__device__ __forceinline__ void store_codes(uint8_t* p, unsigned w, bool vec, int left) {
    if (vec && left >= 4) {
        *(unsigned*)p = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) p[i] = (uint8_t)(w >> (8 * i));
}
__device__ __forceinline__ f32x4 decode(unsigned w, float scale) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return (f32x4){lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
}
// largest magnitude of the wave's 256 values; compared as integers, where a NaN is above everything and so is kept
__device__ __forceinline__ float wave_top(f32x4 v) {
    unsigned t = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned b = __float_as_uint(v[i]) & 0x7fffffffu;
        t = b > t ? b : t;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const unsigned b = (unsigned)__shfl_xor((int)t, o, 64);
        t = b > t ? b : t;
    }
    return __uint_as_float(t);
}
template <bool ROOT>
__device__ __forceinline__ unsigned encode(f32x4 v, float& scale) {
    const float top = wave_top(v);
    const bool some = !(top < 0x1p-100f);  // (a NaN counts)
    const float inv = some ? (1.f / top) * 448.f : 0.f;
    scale = some ? top * (1.f / 448.f) : 0.f;
    f32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = v[i] * inv;
        if (ROOT && some && v[i] > 0.f) c[i] = c[i] < 0x1p-9f ? 0x1p-9f : c[i];
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
}

template <typename PT, int BITS>
__global__ __launch_bounds__(WAVES * 64) void adamw_kernel(const VcAdamwArgs a) {
    // the tensor whose range of workgroups this one is in
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first[mid] <= blockIdx.x) lo = mid;
        else hi = mid;
    }
    const VcAdamwTensor t = a.t[lo];
    PT* const P = (PT*)t.p;
    const PT* const G = (const PT*)t.g;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long base = (long long)(blockIdx.x - a.first[lo]) * CHUNK + wave * (UNROLL * BLK);
    const bool vec = ((((uintptr_t)P | (uintptr_t)G) & (4 * sizeof(PT) - 1)) | (((uintptr_t)t.m | (uintptr_t)t.v) & (BITS == 8 ? 3 : 15))) == 0;
    const float gs = a.gscale != nullptr ? a.gscale_host * *a.gscale : a.gscale_host;

    f32x4 p[UNROLL], g[UNROLL], m[UNROLL], v[UNROLL];
    unsigned qm[UNROLL], qv[UNROLL];
    float sm[UNROLL], sv[UNROLL];
    int left[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long long e = base + u * BLK + lane * 4;
        const long long rest = t.n - e;
        left[u] = rest <= 0 ? 0 : rest < 4 ? (int)rest : 4;
        const long long at = left[u] > 0 ? e : 0;
        p[u] = load4(P + at, vec, left[u]);
        g[u] = load4(G + at, vec, left[u]);
        if (BITS == 8) {
            const bool any = base + u * BLK < t.n;
            const long long blk = any ? (base + u * BLK) / BLK : 0;
            qm[u] = load_codes((const uint8_t*)t.m + at, vec, left[u]);
            qv[u] = load_codes((const uint8_t*)t.v + at, vec, left[u]);
            sm[u] = t.ms[blk], sv[u] = t.vs[blk];
        } else {
            m[u] = load4((const float*)t.m + at, vec, left[u]);
            v[u] = load4((const float*)t.v + at, vec, left[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long long e = base + u * BLK + lane * 4;
        if (base + u * BLK >= t.n) break;  // (uniform over the wave)
        if (BITS == 8) {
            m[u] = decode(qm[u], sm[u]);
            const f32x4 r = decode(qv[u], sv[u]);
            v[u] = r * r;
        }
        f32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float gi = g[u][i] * gs;
            const float mi = m[u][i] * a.b1 + gi * a.one_b1;
            const float vi = v[u][i] * a.b2 + (gi * a.one_b2) * gi;
            const float ri = sqrtf(vi);
            const float move = (mi / (ri * a.root2 + a.eps)) * a.step;
            p[u][i] = p[u][i] * a.c0 - move;
            m[u][i] = mi, v[u][i] = vi, r[i] = ri;
        }
        if (left[u] > 0) store4(P + e, p[u], vec, left[u]);
        if (BITS == 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i)  // (0 0 / eps = NaN with eps = 0: lanes behind the end must not reach the maximum)
                if (i >= left[u]) m[u][i] = 0.f, r[i] = 0.f;
            float nm, nv;
            const unsigned wm = encode<false>(m[u], nm), wv = encode<true>(r, nv);
            if (left[u] > 0) {
                store_codes((uint8_t*)t.m + e, wm, vec, left[u]);
                store_codes((uint8_t*)t.v + e, wv, vec, left[u]);
            }
            if (lane == 0) {
                const long long blk = (base + u * BLK) / BLK;
                t.ms[blk] = nm, t.vs[blk] = nv;
            }
        } else if (left[u] > 0) {
            store4((float*)t.m + e, m[u], vec, left[u]);
            store4((float*)t.v + e, v[u], vec, left[u]);
        }
    }
}

}  // namespace

int vc_adamw_launch(const VcAdamwTensor* t, int count, bool is_bf16, int bits, VcAdamwArgs& a, hipStream_t s) {
    for (int i = 0; i < count;) {
        a.count = 0;
        unsigned blocks = 0;
        // a launch takes up to VC_ADAMW_MAX_TENSORS tensors and 2^30 workgroups
        for (; i < count && a.count < VC_ADAMW_MAX_TENSORS; ++i) {
            if (t[i].n == 0) continue;
            const long long need = (t[i].n + CHUNK - 1) / CHUNK;
            if (a.count > 0 && blocks + need > (1ll << 30)) break;
            a.t[a.count] = t[i];
            a.first[a.count++] = blocks;
            blocks += (unsigned)need;
        }
        if (a.count == 0) continue;
        (void)hipGetLastError();
        const dim3 grid(blocks), block(WAVES * 64);
        if (is_bf16 && bits == 8) hipLaunchKernelGGL((adamw_kernel<bf16, 8>), grid, block, 0, s, a);
        else if (is_bf16) hipLaunchKernelGGL((adamw_kernel<bf16, 32>), grid, block, 0, s, a);
        else if (bits == 8) hipLaunchKernelGGL((adamw_kernel<float, 8>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((adamw_kernel<float, 32>), grid, block, 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            vc_set_error("adamw launch failed: %s", hipGetErrorString(e));
            return -1;
        }
    }
    return 0;
}
