// Gated linear recurrence over time (gfx950), forward, backward and the single step of serving.
//
//   f_t = sigmoid(z_t)      h_t = f_t h_(t-1) + (1 - f_t) v_t        gates[b][t] = (z | v), H values each
//   backward, from the last step down (mu = what the future hands to h_t; dlast behind the last step):
//     lam_t = dy_t + mu      dv_t = (1 - f_t) lam_t      dz_t = lam_t (h_(t-1) - v_t) f_t (1 - f_t)      mu <- f_t lam_t
//   dh0 = mu in front of the first step.
//
// A step is an affine map of the state, h -> a h + b, and maps compose: (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2).  So a
// workgroup takes a tile of steps at once: each wave composes the maps of its own SUB steps (two channels per lane, held in
// registers), the waves exchange their compositions through LDS, and with the state in front of its first step each wave
// runs its steps again and writes them.  gates are read from memory once, h is written once.  The backward pass needs
// h_(t-1) and does not read h: it recomputes the states from the gates, which it has to read anyway, starting at the fp32
// states that the forward saved every VC_SCAN_CHUNK steps (4 bytes per 64 steps and channel against 2-4 bytes per step,
// and without the rounding of a 16-bit h inside h_(t-1) - v_t).
//
// All arithmetic and the state are fp32; h and dgates round once, to their type.  1 - f is computed as its own quotient
// (sigmoid(-z)), so that a gate near 1 keeps its relative precision.
#include "common.h"
#include "kernels.h"

namespace {

// sigmoid(z) and 1 - sigmoid(z), both without cancellation or overflow: e = exp(-|z|) <= 1
__device__ __forceinline__ void gate(float z, float& f, float& q) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(z) * 1.44269504088896340736f);
    const float big = __builtin_amdgcn_rcpf(1.f + e), small = e * big;
    const bool pos = z >= 0.f;
    f = pos ? big : small;
    q = pos ? small : big;
}

struct f2 {
    float x, y;
};

// two neighbouring channels; `vec`: both exist and the address is a multiple of their size
__device__ __forceinline__ f2 load2(const float* p, bool vec, bool ok0, bool ok1) {
    if (vec) {
        const float2 v = *(const float2*)p;
        return {v.x, v.y};
    }
    return {ok0 ? p[0] : 0.f, ok1 ? p[1] : 0.f};
}
__device__ __forceinline__ f2 load2(const bf16* p, bool vec, bool ok0, bool ok1) {
    if (vec) {
        const unsigned w = *(const unsigned*)p;
        return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
    }
    return {ok0 ? bf2f(p[0]) : 0.f, ok1 ? bf2f(p[1]) : 0.f};
}
__device__ __forceinline__ void store2(float* p, f2 v, bool vec, bool ok0, bool ok1) {
    if (vec) {
        *(float2*)p = make_float2(v.x, v.y);
        return;
    }
    if (ok0) p[0] = v.x;
    if (ok1) p[1] = v.y;
}
__device__ __forceinline__ void store2(bf16* p, f2 v, bool vec, bool ok0, bool ok1) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    if (vec) {
        *(bf16x2*)p = (bf16x2){f2bf(v.x), f2bf(v.y)};
        return;
    }
    if (ok0) p[0] = f2bf(v.x);
    if (ok1) p[1] = f2bf(v.y);
}

template <typename T>
struct Lane {  // what a lane of a column tile works on
    int c, b, len;
    bool ok0, ok1, vin, vout;  // channels that exist; vector access to gates, to contiguous [..][H] rows
    __device__ Lane(const VcScanParams& p, int col, int batch, int lane) {
        c = col * 128 + lane * 2;
        b = batch;
        ok0 = c < p.H, ok1 = c + 1 < p.H;
        const bool even = ((p.H | p.sb | p.st) & 1) == 0 && ((uintptr_t)p.gates & (2 * sizeof(T) - 1)) == 0;
        vin = even && ok1;
        vout = (p.H & 1) == 0 && ok1;
        const int n = p.lengths != nullptr ? p.lengths[b] : p.T;
        len = n < 0 ? 0 : n > p.T ? p.T : n;
    }
};

template <typename T, int WAVES, int SUB>
__global__ __launch_bounds__(WAVES * 64) void scan_fwd_kernel(const VcScanParams p) {
    constexpr int TILE = WAVES * SUB;
    static_assert(TILE % VC_SCAN_CHUNK == 0 && VC_SCAN_CHUNK % SUB == 0, "saved states sit where a wave starts");
    __shared__ float4 agg[WAVES][64];
    __shared__ f2 carry[2][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Lane<T> L(p, blockIdx.x, blockIdx.y, lane);
    const T* const g = (const T*)p.gates + L.b * p.sb + L.c;
    T* const out = (T*)p.h + (size_t)L.b * p.T * p.H + L.c;
    const int nchunks = (p.T + VC_SCAN_CHUNK - 1) / VC_SCAN_CHUNK;
    const size_t sc = (size_t)L.b * p.H + L.c;
    if (wave == 0) carry[0][lane] = p.h0 != nullptr ? f2{L.ok0 ? p.h0[sc] : 0.f, L.ok1 ? p.h0[sc + 1] : 0.f} : f2{0.f, 0.f};
    int cur = 0;
    for (int s0 = 0; s0 < L.len; s0 += TILE, cur ^= 1) {
        f2 f[SUB], u[SUB];
        const int w0 = s0 + wave * SUB;
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            const int s = w0 + j;
            f[j] = {1.f, 1.f}, u[j] = {0.f, 0.f};
            if (s < L.len) {
                const T* row = g + (long long)(p.reverse ? L.len - 1 - s : s) * p.st;
                const f2 z = load2(row, L.vin, L.ok0, L.ok1), v = load2(row + p.H, L.vin, L.ok0, L.ok1);
                f2 q;
                gate(z.x, f[j].x, q.x);
                gate(z.y, f[j].y, q.y);
                u[j] = {q.x * v.x, q.y * v.y};
            }
        }
        f2 a = {1.f, 1.f}, b = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            a = {a.x * f[j].x, a.y * f[j].y};
            b = {f[j].x * b.x + u[j].x, f[j].y * b.y + u[j].y};
        }
        agg[wave][lane] = make_float4(a.x, a.y, b.x, b.y);
        __syncthreads();
        f2 h = carry[cur][lane];
        for (int w = 0; w < wave; ++w) {
            const float4 m = agg[w][lane];
            h = {m.x * h.x + m.z, m.y * h.y + m.w};
        }
        if (p.states != nullptr && w0 % VC_SCAN_CHUNK == 0 && w0 < L.len) {
            float* q = p.states + ((size_t)L.b * nchunks + w0 / VC_SCAN_CHUNK) * p.H + L.c;
            if (L.ok0) q[0] = h.x;
            if (L.ok1) q[1] = h.y;
        }
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            const int s = w0 + j;
            h = {f[j].x * h.x + u[j].x, f[j].y * h.y + u[j].y};
            if (s < L.len) store2(out + (size_t)(p.reverse ? L.len - 1 - s : s) * p.H, h, L.vout, L.ok0, L.ok1);
        }
        if (wave == WAVES - 1) carry[cur ^ 1][lane] = h;
        __syncthreads();
    }
    __syncthreads();
    if (wave == 0 && p.last != nullptr) {
        const f2 h = carry[cur][lane];
        if (L.ok0) p.last[sc] = h.x;
        if (L.ok1) p.last[sc + 1] = h.y;
    }
    for (int t = L.len + wave; t < p.T; t += WAVES) store2(out + (size_t)t * p.H, {0.f, 0.f}, L.vout, L.ok0, L.ok1);
}

template <typename T, int WAVES, int SUB>
__global__ __launch_bounds__(WAVES * 64) void scan_bwd_kernel(const VcScanParams p) {
    constexpr int TILE = WAVES * SUB;
    static_assert(TILE == VC_SCAN_CHUNK, "a tile starts at a saved state");
    __shared__ float4 agg[WAVES][64];  // forward maps
    __shared__ f2 back[WAVES][64];     // constant part of the backward maps (their factor is the forward's)
    __shared__ f2 carry[2][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Lane<T> L(p, blockIdx.x, blockIdx.y, lane);
    const T* const g = (const T*)p.gates + L.b * p.sb + L.c;
    const T* const dy = p.dy != nullptr ? (const T*)p.dy + (size_t)L.b * p.T * p.H + L.c : nullptr;
    T* const out = (T*)p.dgates + (size_t)L.b * p.T * 2 * p.H + L.c;
    const int nchunks = (p.T + VC_SCAN_CHUNK - 1) / VC_SCAN_CHUNK;
    const size_t sc = (size_t)L.b * p.H + L.c;
    if (wave == 0) carry[0][lane] = p.dlast != nullptr ? f2{L.ok0 ? p.dlast[sc] : 0.f, L.ok1 ? p.dlast[sc + 1] : 0.f} : f2{0.f, 0.f};
    int cur = 0;
    for (int k = (L.len + TILE - 1) / TILE - 1; k >= 0; --k, cur ^= 1) {
        const int w0 = k * TILE + wave * SUB;
        f2 f[SUB], q[SUB], v[SUB], d[SUB], before[SUB];
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            const int s = w0 + j;
            f[j] = {1.f, 1.f}, q[j] = v[j] = d[j] = {0.f, 0.f};
            if (s < L.len) {
                const long long t = p.reverse ? L.len - 1 - s : s;
                const T* row = g + t * p.st;
                const f2 z = load2(row, L.vin, L.ok0, L.ok1);
                v[j] = load2(row + p.H, L.vin, L.ok0, L.ok1);
                if (dy != nullptr) d[j] = load2(dy + t * p.H, L.vout, L.ok0, L.ok1);
                gate(z.x, f[j].x, q[j].x);
                gate(z.y, f[j].y, q[j].y);
            }
        }
        f2 a = {1.f, 1.f}, b = {0.f, 0.f}, c = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            a = {a.x * f[j].x, a.y * f[j].y};
            b = {f[j].x * b.x + q[j].x * v[j].x, f[j].y * b.y + q[j].y * v[j].y};
        }
#pragma unroll
        for (int j = SUB - 1; j >= 0; --j) c = {f[j].x * (d[j].x + c.x), f[j].y * (d[j].y + c.y)};
        agg[wave][lane] = make_float4(a.x, a.y, b.x, b.y);
        back[wave][lane] = c;
        __syncthreads();
        const float* st = p.states + ((size_t)L.b * nchunks + k) * p.H + L.c;
        f2 h = {L.ok0 ? st[0] : 0.f, L.ok1 ? st[1] : 0.f}, mu = carry[cur][lane];
        for (int w = 0; w < wave; ++w) {
            const float4 m = agg[w][lane];
            h = {m.x * h.x + m.z, m.y * h.y + m.w};
        }
        for (int w = WAVES - 1; w > wave; --w) {
            const float4 m = agg[w][lane];
            const f2 n = back[w][lane];
            mu = {m.x * mu.x + n.x, m.y * mu.y + n.y};
        }
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            before[j] = h;
            h = {f[j].x * h.x + q[j].x * v[j].x, f[j].y * h.y + q[j].y * v[j].y};
        }
#pragma unroll
        for (int j = SUB - 1; j >= 0; --j) {
            const int s = w0 + j;
            const f2 lam = {d[j].x + mu.x, d[j].y + mu.y};
            mu = {f[j].x * lam.x, f[j].y * lam.y};
            if (s < L.len) {
                T* row = out + (size_t)(p.reverse ? L.len - 1 - s : s) * 2 * p.H;
                store2(row, {mu.x * q[j].x * (before[j].x - v[j].x), mu.y * q[j].y * (before[j].y - v[j].y)}, L.vout, L.ok0, L.ok1);
                store2(row + p.H, {q[j].x * lam.x, q[j].y * lam.y}, L.vout, L.ok0, L.ok1);
            }
        }
        if (wave == 0) carry[cur ^ 1][lane] = mu;
        __syncthreads();
    }
    __syncthreads();
    if (wave == 0 && p.dh0 != nullptr) {
        const f2 mu = carry[cur][lane];
        if (L.ok0) p.dh0[sc] = mu.x;
        if (L.ok1) p.dh0[sc + 1] = mu.y;
    }
    for (int t = L.len + wave; t < p.T; t += WAVES) {
        T* row = out + (size_t)t * 2 * p.H;
        store2(row, {0.f, 0.f}, L.vout, L.ok0, L.ok1);
        store2(row + p.H, {0.f, 0.f}, L.vout, L.ok0, L.ok1);
    }
}

// one step for every sequence, the state updated in place
template <typename T>
__global__ __launch_bounds__(256) void scan_step_kernel(const T* gates, long long sb, float* state, T* h, int B, int H) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= H) return;
    for (int b = blockIdx.y; b < B; b += gridDim.y) {
        const T* row = gates + b * sb + c;
        const size_t e = (size_t)b * H + c;
        float f, q;
        gate((float)row[0], f, q);
        const float n = f * state[e] + q * (float)row[H];
        state[e] = n;
        h[e] = (T)n;
    }
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        vc_set_error("%s launch failed: %s", what, hipGetErrorString(e));
        return -1;
    }
    return 0;
}

}  // namespace

int vc_scan_launch_fwd(const VcScanParams& p, bool is_bf16, hipStream_t s) {
    const dim3 grid((p.H + 127) / 128, p.B);
    (void)hipGetLastError();
    if (is_bf16) hipLaunchKernelGGL((scan_fwd_kernel<bf16, 8, 16>), grid, dim3(512), 0, s, p);
    else hipLaunchKernelGGL((scan_fwd_kernel<float, 8, 16>), grid, dim3(512), 0, s, p);
    return launched("gated_scan_fwd");
}
int vc_scan_launch_bwd(const VcScanParams& p, bool is_bf16, hipStream_t s) {
    const dim3 grid((p.H + 127) / 128, p.B);
    (void)hipGetLastError();
    if (is_bf16) hipLaunchKernelGGL((scan_bwd_kernel<bf16, 8, 8>), grid, dim3(512), 0, s, p);
    else hipLaunchKernelGGL((scan_bwd_kernel<float, 8, 8>), grid, dim3(512), 0, s, p);
    return launched("gated_scan_bwd");
}
int vc_scan_launch_step(const void* gates, long long sb, float* state, void* h, int B, int H, bool is_bf16, hipStream_t s) {
    const dim3 grid((H + 255) / 256, B < 4096 ? B : 4096);
    (void)hipGetLastError();
    if (is_bf16) hipLaunchKernelGGL((scan_step_kernel<bf16>), grid, dim3(256), 0, s, (const bf16*)gates, sb, state, (bf16*)h, B, H);
    else hipLaunchKernelGGL((scan_step_kernel<float>), grid, dim3(256), 0, s, (const float*)gates, sb, state, (float*)h, B, H);
    return launched("gated_scan_step");
}
