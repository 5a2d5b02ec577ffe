// Gated linear recurrence over time (gfx950), forward, backward and the single step of serving.
//
//   f_t = sigmoid(z_t)      h_t = f_t h_(t-1) + (1 - f_t) v_t        gates[b][t] = (z | v), H values each
//   backward, from the last step down (mu = what the future hands to h_t; dlast behind the last step):
//     lam_t = dy_t + mu      dv_t = (1 - f_t) lam_t      dz_t = lam_t (h_(t-1) - v_t) f_t (1 - f_t)      mu <- f_t lam_t
//   dh0 = mu in front of the first step.
//
// A step is an affine map of the state, h -> a h + b, and maps compose: (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2).  So a
// workgroup takes a tile of steps x 128 channels at once: each wave composes the maps of its own SUB steps (two channels per
// lane, held in registers), the waves exchange their compositions through LDS, and with the state in front of its first step
// each wave runs its steps again and writes them.  gates are read from memory once, h is written once.  The backward pass
// needs h_(t-1) and does not read h: it recomputes the states from the gates, which it has to read anyway, starting at the
// fp32 states that the forward saved every VC_SCAN_CHUNK steps (4 bytes per 64 steps and channel against 2-4 bytes per step,
// and without the rounding of a 16-bit h inside h_(t-1) - v_t).
//
// The tiles of one sequence run at the same time (one sequence of 1024 channels is 8 workgroups otherwise).  A tile publishes
// its composition as soon as it has it; the state in front of a tile is the nearest state that an earlier tile has published,
// carried through the compositions in between, always from the earlier to the later tile: the same operations on the same
// numbers whichever state was found, so results do not depend on timing.  Every published word is 64 bits with its own
// ready mark (words are 0 before), written and read by relaxed device-scope atomics: no fence, no L2 write-back.  Tiles take
// their number from a counter, earlier steps first, so a tile only ever waits for tiles that run already, and every wait ends.
//
// Measured (copies on this card reach 5.14 TB/s): 8 x 2048 x 2048 bf16 forward 44 us = 4.6 TB/s, backward 82 us = 4.1; one
// sequence of 131072 x 1024 193 us = 4.2 TB/s.
//
// All arithmetic and the state are fp32; h and dgates round once, to their type.  1 - f is computed as its own quotient
// (sigmoid(-z)), so that a gate near 1 keeps its relative precision.
#include <type_traits>

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

// two neighbouring channels as they lie in memory.  VEC: at a multiple of their size; otherwise one by one (d: elements from
// the first to the second, 0 where there is no second).
template <typename T>
struct Raw;
template <>
struct Raw<bf16> {
    unsigned w;
    template <bool VEC>
    __device__ __forceinline__ void load(const bf16* p, int d) {
        if (VEC) w = *(const unsigned*)p;
        else w = (unsigned)*(const unsigned short*)p | (unsigned)*(const unsigned short*)(p + d) << 16;
    }
    __device__ __forceinline__ f2 get() const { return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }
};
template <>
struct Raw<float> {
    float a, b;
    template <bool VEC>
    __device__ __forceinline__ void load(const float* p, int d) {
        if (VEC) {
            const float2 v = *(const float2*)p;
            a = v.x, b = v.y;
        } else
            a = p[0], b = p[d];
    }
    __device__ __forceinline__ f2 get() const { return {a, b}; }
};
// two neighbouring values as they lie in memory
template <typename T>
struct Pair;
template <>
struct Pair<float> {
    typedef float2 type;
    static __device__ __forceinline__ type make(f2 v) { return make_float2(v.x, v.y); }
};
template <>
struct Pair<bf16> {
    typedef __attribute__((ext_vector_type(2))) __bf16 type;
    static __device__ __forceinline__ type make(f2 v) { return (type){f2bf(v.x), f2bf(v.y)}; }
};
template <typename T>
__device__ __forceinline__ typename Pair<T>::type pair(f2 v) {
    return Pair<T>::make(v);
}
template <bool VEC>
__device__ __forceinline__ void store2(float* p, f2 v, int n) {
    if (VEC && n == 2) *(float2*)p = pair<float>(v);
    else {
        if (n > 0) p[0] = v.x;
        if (n > 1) p[1] = v.y;
    }
}
template <bool VEC>
__device__ __forceinline__ void store2(bf16* p, f2 v, int n) {
    if (VEC && n == 2) *(Pair<bf16>::type*)p = pair<bf16>(v);
    else {
        if (n > 0) p[0] = f2bf(v.x);
        if (n > 1) p[1] = f2bf(v.y);
    }
}

// ---------------------------------------------------------------- states between tiles
// workspace: a counter (256 bytes), then for each sequence and tile two words of 64 bits per channel: the tile's composition
// (a with its sign bit set, as a is never negative; b) and the state behind it (1; h)
typedef unsigned long long u64;
__device__ __forceinline__ u64 word(unsigned hi, float lo) { return (u64)hi << 32 | __float_as_uint(lo); }
__device__ __forceinline__ void put(u64* p, u64 v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ u64 get(const u64* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float low(u64 w) { return __uint_as_float((unsigned)w); }

struct Between {
    u64 *maps, *states;  // this lane's first channel, tile 0 of its sequence (tiles counted in the order of processing)
    long long stride;    // words from tile to tile
    int d;               // 1, or 0 where there is no second channel

    // the state in front of tile `tile` > 0
    __device__ __forceinline__ f2 before(int tile) const {
        constexpr int W = 4;  // (2: the same within 1 %; 8: 30 % slower, its registers spill)
        // the nearest tile whose state is there for all lanes, the latest W tiles first; the first tile's always comes
        int from = -1;
        while (from < 0) {
            for (int top = tile - 1; top >= 0 && from < 0; top -= W) {
                u64 x[W], y[W];
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const u64* q = states + (top - i > 0 ? top - i : 0) * stride;
                    x[i] = get(q), y[i] = get(q + d);
                }
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (from < 0 && top - i >= 0 && __all(x[i] != 0 && y[i] != 0)) from = top - i;
            }
        }
        const u64* q = states + from * stride;
        f2 h = {low(get(q)), low(get(q + d))};
        for (int k = from + 1; k < tile; k += W) {
            u64 x[W], y[W];
            bool ready;
            do {
                ready = true;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const u64* m = maps + (k + i < tile ? k + i : tile - 1) * stride;
                    x[i] = get(m), y[i] = get(m + d);
                }
#pragma unroll
                for (int i = 0; i < W; ++i) ready = ready && x[i] != 0 && y[i] != 0;
            } while (!__all(ready));
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (k + i < tile)
                    h = {__uint_as_float((unsigned)(x[i] >> 32) & 0x7fffffffu) * h.x + low(x[i]),
                         __uint_as_float((unsigned)(y[i] >> 32) & 0x7fffffffu) * h.y + low(y[i])};
        }
        return h;
    }
    __device__ __forceinline__ void put_map(int tile, f2 a, f2 b, int n) const {
        u64* q = maps + tile * stride;
        if (n > 0) put(q, word(__float_as_uint(a.x) | 0x80000000u, b.x));
        if (n > 1) put(q + 1, word(__float_as_uint(a.y) | 0x80000000u, b.y));
    }
    __device__ __forceinline__ void put_state(int tile, f2 h, int n) const {
        u64* q = states + tile * stride;
        if (n > 0) put(q, word(1u, h.x));
        if (n > 1) put(q + 1, word(1u, h.y));
    }
};

__global__ __launch_bounds__(256) void scan_clear_kernel(uint4* p, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = make_uint4(0, 0, 0, 0);
}

// what a workgroup and a lane of it work on
template <typename T>
struct Place {
    int tile, ntiles, c, n, d, b, len;  // c: first of the lane's n (0, 1, 2) channels (0 if it has none); d: to its second
    Between between;
    __device__ Place(const VcScanParams& p, int steps, int lane, int* shared) {
        const int cols = (p.H + 127) >> 7;
        ntiles = (p.T + steps - 1) / steps;
        int id = blockIdx.x;
        if (ntiles > 1) {
            if (threadIdx.x == 0) *shared = (int)atomicAdd((unsigned*)p.ws, 1u);
            __syncthreads();
            id = *shared;
        }
        const int per = cols * p.B;
        tile = id / per;
        id -= tile * per;
        b = id / cols;
        c = (id - b * cols) * 128 + lane * 2;
        n = p.H - c >= 2 ? 2 : p.H - c > 0 ? p.H - c : 0;
        c = n > 0 ? c : 0;
        d = c + 1 < p.H ? 1 : 0;
        const int l = p.lengths != nullptr ? p.lengths[b] : p.T;
        len = l < 0 ? 0 : l > p.T ? p.T : l;
        between.stride = p.H;
        between.maps = (u64*)(p.ws + 256) + (long long)b * ntiles * p.H + c;
        between.states = between.maps + (long long)p.B * ntiles * p.H;
        between.d = d;
    }
};

template <typename T, int WAVES, int SUB, bool VEC>
__global__ __launch_bounds__(WAVES * 64, 4) void scan_fwd_kernel(const VcScanParams p) {
    constexpr int TILE = WAVES * SUB;
    static_assert(TILE % VC_SCAN_CHUNK == 0 && VC_SCAN_CHUNK % SUB == 0, "saved states sit where a wave starts");
    __shared__ float4 agg[WAVES][64];
    __shared__ f2 carry[64];
    __shared__ int shared;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    typedef typename Pair<T>::type P2;
    const Place<T> L(p, TILE, lane, &shared);
    T* const out = (T*)p.h + (long long)L.b * p.T * p.H + L.c;
    const int w0 = L.tile * TILE + wave * SUB;  // the wave's first step
    const int left = L.len - w0;                // steps that are there from it on
    // step w0 + j is at time t0 + j dt
    const int dt = p.reverse ? -1 : 1;
    const long long t0 = p.reverse ? L.len - 1 - w0 : w0;
    const long long sc = (long long)L.b * p.H + L.c;
    if (L.tile * TILE < L.len) {
        Raw<T> z[SUB], v[SUB];
        if (left > 0) {
            const T* const g = (const T*)p.gates + L.b * p.sb + L.c + t0 * p.st;
            const long long st = p.st * dt;
            if (left >= SUB) {
#pragma unroll
                for (int j = 0; j < SUB; ++j) {
                    z[j].template load<VEC>(g + j * st, L.d);
                    v[j].template load<VEC>(g + j * st + p.H, L.d);
                }
            } else {
#pragma unroll
                for (int j = 0; j < SUB; ++j) {
                    const long long at = (j < left ? j : left - 1) * st;  // (read again, not used)
                    z[j].template load<VEC>(g + at, L.d);
                    v[j].template load<VEC>(g + at + p.H, L.d);
                }
            }
        }
        f2 f[SUB], u[SUB], a = {1.f, 1.f}, b = {0.f, 0.f};
        auto compose = [&](auto whole) {  // (a wave whose steps are all there tests none of them)
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                f[j] = {1.f, 1.f}, u[j] = {0.f, 0.f};
                if (decltype(whole)::value || j < left) {
                    const f2 zz = z[j].get(), vv = v[j].get();
                    f2 q;
                    gate(zz.x, f[j].x, q.x);
                    gate(zz.y, f[j].y, q.y);
                    u[j] = {q.x * vv.x, q.y * vv.y};
                }
                a = {a.x * f[j].x, a.y * f[j].y};
                b = {f[j].x * b.x + u[j].x, f[j].y * b.y + u[j].y};
            }
        };
        if (left >= SUB) compose(std::true_type());
        else compose(std::false_type());
        agg[wave][lane] = make_float4(a.x, a.y, b.x, b.y);
        __syncthreads();
        if (wave == 0) {
            f2 h;
            if (L.tile == 0) h = p.h0 != nullptr ? f2{p.h0[sc], p.h0[sc + L.d]} : f2{0.f, 0.f};
            a = {1.f, 1.f}, b = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float4 m = agg[w][lane];
                a = {a.x * m.x, a.y * m.y};
                b = {m.x * b.x + m.z, m.y * b.y + m.w};
            }
            const bool more = (L.tile + 1) * TILE < L.len;
            if (L.tile > 0) {
                if (more) L.between.put_map(L.tile, a, b, L.n);
                h = L.between.before(L.tile);
            }
            carry[lane] = h;
            h = {a.x * h.x + b.x, a.y * h.y + b.y};
            if (more) L.between.put_state(L.tile, h, L.n);
            else store2<false>(p.last + sc, h, L.n);
        }
        __syncthreads();
        f2 h = carry[lane];
        for (int w = 0; w < wave; ++w) {
            const float4 m = agg[w][lane];
            h = {m.x * h.x + m.z, m.y * h.y + m.w};
        }
        if (p.states != nullptr && w0 % VC_SCAN_CHUNK == 0 && left > 0) {
            const long long chunks = (p.T + VC_SCAN_CHUNK - 1) / VC_SCAN_CHUNK;
            store2<false>(p.states + (L.b * chunks + w0 / VC_SCAN_CHUNK) * p.H + L.c, h, L.n);
        }
        T* const o = out + t0 * p.H;
        const long long so = (long long)p.H * dt;
        auto write = [&](auto whole) {
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                h = {f[j].x * h.x + u[j].x, f[j].y * h.y + u[j].y};
                if (decltype(whole)::value) *(P2*)(o + j * so) = pair<T>(h);
                else if (j < left) store2<VEC>(o + j * so, h, L.n);
            }
        };
        if (VEC && left >= SUB && __all(L.n == 2)) write(std::true_type());
        else write(std::false_type());
    } else if (L.len == 0 && L.tile == 0 && wave == 0)
        store2<false>(p.last + sc, p.h0 != nullptr ? f2{p.h0[sc], p.h0[sc + L.d]} : f2{0.f, 0.f}, L.n);
    if (left < SUB)  // behind the end: zeros
        for (int t = left > 0 ? L.len : w0; t < w0 + SUB && t < p.T; ++t) store2<VEC>(out + (long long)t * p.H, {0.f, 0.f}, L.n);
}

template <typename T, int WAVES, int SUB, bool VEC>
__global__ __launch_bounds__(WAVES * 64, 4) void scan_bwd_kernel(const VcScanParams p) {
    constexpr int TILE = WAVES * SUB;
    static_assert(TILE % VC_SCAN_CHUNK == 0, "a tile starts at a saved state");
    __shared__ float4 agg[WAVES][64];  // forward maps
    __shared__ f2 back[WAVES][64];     // constant part of the backward maps (their factor is the forward's)
    __shared__ f2 carry[64];
    __shared__ int shared;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    typedef typename Pair<T>::type P2;
    const Place<T> L(p, TILE, lane, &shared);
    const int tile = L.ntiles - 1 - L.tile;                  // the last steps come first
    const int first = (L.len + TILE - 1) / TILE - 1 - tile;  // tiles of this sequence that come before
    T* const out = (T*)p.dgates + (long long)L.b * p.T * 2 * p.H + L.c;
    const int w0 = tile * TILE + wave * SUB, left = L.len - w0;
    const int dt = p.reverse ? -1 : 1;
    const long long t0 = p.reverse ? L.len - 1 - w0 : w0;
    const long long sc = (long long)L.b * p.H + L.c;
    if (first >= 0) {
        Raw<T> z[SUB], v[SUB], d[SUB];
        if (left > 0) {
            const T* const g = (const T*)p.gates + L.b * p.sb + L.c + t0 * p.st;
            const long long st = p.st * dt;
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                const long long at = (j < left ? j : left - 1) * st;  // (behind the end: read again, not used)
                z[j].template load<VEC>(g + at, L.d);
                v[j].template load<VEC>(g + at + p.H, L.d);
            }
            if (p.dy != nullptr) {
                const T* const y = (const T*)p.dy + ((long long)L.b * p.T + t0) * p.H + L.c;
                const long long so = (long long)p.H * dt;
#pragma unroll
                for (int j = 0; j < SUB; ++j) d[j].template load<VEC>(y + (j < left ? j : left - 1) * so, L.d);
            }
        }
        f2 f[SUB], q[SUB], a = {1.f, 1.f}, b = {0.f, 0.f}, c = {0.f, 0.f};
        const bool has_dy = p.dy != nullptr;
        auto dy = [&](int j, auto whole) { return decltype(whole)::value || has_dy && j < left ? d[j].get() : f2{0.f, 0.f}; };
        auto compose = [&](auto whole) {  // (a wave whose steps are all there tests none of them)
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                f[j] = {1.f, 1.f}, q[j] = {0.f, 0.f};
                if (decltype(whole)::value || j < left) {
                    const f2 zz = z[j].get();
                    gate(zz.x, f[j].x, q[j].x);
                    gate(zz.y, f[j].y, q[j].y);
                    const f2 vv = v[j].get();
                    b = {f[j].x * b.x + q[j].x * vv.x, f[j].y * b.y + q[j].y * vv.y};
                }
                a = {a.x * f[j].x, a.y * f[j].y};
            }
#pragma unroll
            for (int j = SUB - 1; j >= 0; --j) {
                const f2 e = dy(j, whole);
                c = {f[j].x * (e.x + c.x), f[j].y * (e.y + c.y)};
            }
        };
        if (left >= SUB && has_dy) compose(std::true_type());
        else compose(std::false_type());
        agg[wave][lane] = make_float4(a.x, a.y, b.x, b.y);
        back[wave][lane] = c;
        __syncthreads();
        if (wave == 0) {
            f2 mu;
            if (first == 0) mu = p.dlast != nullptr ? f2{p.dlast[sc], p.dlast[sc + L.d]} : f2{0.f, 0.f};
            a = {1.f, 1.f}, c = {0.f, 0.f};
#pragma unroll
            for (int w = WAVES - 1; w >= 0; --w) {
                const float4 m = agg[w][lane];
                const f2 n = back[w][lane];
                a = {a.x * m.x, a.y * m.y};
                c = {m.x * c.x + n.x, m.y * c.y + n.y};
            }
            if (first > 0) {
                if (tile > 0) L.between.put_map(first, a, c, L.n);
                mu = L.between.before(first);
            }
            carry[lane] = mu;
            mu = {a.x * mu.x + c.x, a.y * mu.y + c.y};
            if (tile > 0) L.between.put_state(first, mu, L.n);
            else if (p.dh0 != nullptr) store2<false>(p.dh0 + sc, mu, L.n);
        }
        const long long chunks = (p.T + VC_SCAN_CHUNK - 1) / VC_SCAN_CHUNK;
        const float* st = p.states + (L.b * chunks + tile * (TILE / VC_SCAN_CHUNK)) * p.H + L.c;
        f2 h = {st[0], st[L.d]};
        for (int w = 0; w < wave; ++w) {
            const float4 m = agg[w][lane];
            h = {m.x * h.x + m.z, m.y * h.y + m.w};
        }
        __syncthreads();
        f2 mu = carry[lane];
        for (int w = WAVES - 1; w > wave; --w) {
            const float4 m = agg[w][lane];
            const f2 n = back[w][lane];
            mu = {m.x * mu.x + n.x, m.y * mu.y + n.y};
        }
        f2 before[SUB];
        T* const o = out + t0 * 2 * p.H;
        const long long so = 2ll * p.H * dt;
        auto write = [&](auto whole) {
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                const f2 vv = v[j].get();
                before[j] = h;
                if (decltype(whole)::value || j < left) h = {f[j].x * h.x + q[j].x * vv.x, f[j].y * h.y + q[j].y * vv.y};
            }
#pragma unroll
            for (int j = SUB - 1; j >= 0; --j) {
                const f2 e = dy(j, whole), lam = {e.x + mu.x, e.y + mu.y}, vv = v[j].get();
                mu = {f[j].x * lam.x, f[j].y * lam.y};
                const f2 dv = {q[j].x * lam.x, q[j].y * lam.y};
                const f2 dz = {mu.x * q[j].x * (before[j].x - vv.x), mu.y * q[j].y * (before[j].y - vv.y)};
                if (decltype(whole)::value) {
                    *(P2*)(o + j * so) = pair<T>(dz);
                    *(P2*)(o + j * so + p.H) = pair<T>(dv);
                } else if (j < left) {
                    store2<VEC>(o + j * so, dz, L.n);
                    store2<VEC>(o + j * so + p.H, dv, L.n);
                }
            }
        };
        if (VEC && has_dy && left >= SUB && __all(L.n == 2)) write(std::true_type());
        else write(std::false_type());
    } else if (L.len == 0 && tile == 0 && wave == 0 && p.dh0 != nullptr)
        store2<false>(p.dh0 + sc, p.dlast != nullptr ? f2{p.dlast[sc], p.dlast[sc + L.d]} : f2{0.f, 0.f}, L.n);
    if (left < SUB)  // behind the end: zeros
        for (int t = left > 0 ? L.len : w0; t < w0 + SUB && t < p.T; ++t) {
            store2<VEC>(out + (long long)t * 2 * p.H, {0.f, 0.f}, L.n);
            store2<VEC>(out + (long long)t * 2 * p.H + p.H, {0.f, 0.f}, L.n);
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

namespace {

// Forward: 16 waves of 16 steps, one workgroup a CU.  Half as many waves or steps: 8 .. 30 % slower (a sequence is more tiles,
// whose states wait for each other, and a wave has fewer loads in flight); 32 steps spill.  Backward: its three inputs and h
// in registers leave room for 8 steps; 16 waves against 8: one sequence of 131072 x 512 320 against 433 us, 32 sequences
// of 2048 x 1024 262 against 258.  Workgroups that stay and ask for their next tile's gates while they finish one measured 20 %
// slower in both directions (more registers, fewer loads in flight).
constexpr int FWD_WAVES = 16, FWD_SUB = 16, BWD_WAVES = 16, BWD_SUB = 8;

// whether every pair of channels begins at a multiple of two elements
bool pairs(const VcScanParams& p, int elem) {
    return ((p.H | p.sb | p.st) & 1) == 0 && ((uintptr_t)p.gates & (2 * elem - 1)) == 0;
}
// the workgroups of a launch; clears what they exchange their states through
unsigned begin(const VcScanParams& p, int steps, size_t bytes, hipStream_t s) {
    const long long tiles = (p.T + steps - 1) / steps;
    if (bytes > 0) {
        const long long n = (long long)bytes / 16, blocks = (n + 255) / 256;
        hipLaunchKernelGGL(scan_clear_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, (uint4*)p.ws, n);
    }
    return (unsigned)(tiles * ((p.H + 127) / 128) * p.B);
}

template <typename T>
int fwd(const VcScanParams& p, hipStream_t s) {
    (void)hipGetLastError();
    const dim3 grid(begin(p, FWD_WAVES * FWD_SUB, vc_scan_workspace(p.B, p.T, p.H, 0), s)), block(FWD_WAVES * 64);
    if (pairs(p, sizeof(T))) hipLaunchKernelGGL((scan_fwd_kernel<T, FWD_WAVES, FWD_SUB, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((scan_fwd_kernel<T, FWD_WAVES, FWD_SUB, false>), grid, block, 0, s, p);
    return launched("gated_scan_fwd");
}
template <typename T>
int bwd(const VcScanParams& p, hipStream_t s) {
    (void)hipGetLastError();
    const dim3 grid(begin(p, BWD_WAVES * BWD_SUB, vc_scan_workspace(p.B, p.T, p.H, 1), s)), block(BWD_WAVES * 64);
    if (pairs(p, sizeof(T))) hipLaunchKernelGGL((scan_bwd_kernel<T, BWD_WAVES, BWD_SUB, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((scan_bwd_kernel<T, BWD_WAVES, BWD_SUB, false>), grid, block, 0, s, p);
    return launched("gated_scan_bwd");
}

}  // namespace

// what the tiles of a sequence exchange: 0 where a sequence is one tile
size_t vc_scan_workspace(int B, int T, int H, int op) {
    const int steps = op == 0 ? FWD_WAVES * FWD_SUB : BWD_WAVES * BWD_SUB;
    const long long tiles = ((long long)T + steps - 1) / steps;
    return tiles > 1 ? (size_t)(256 + 2 * 8 * tiles * B * H) : 0;
}
int vc_scan_launch_fwd(const VcScanParams& p, bool is_bf16, hipStream_t s) { return is_bf16 ? fwd<bf16>(p, s) : fwd<float>(p, s); }
int vc_scan_launch_bwd(const VcScanParams& p, bool is_bf16, hipStream_t s) { return is_bf16 ? bwd<bf16>(p, s) : bwd<float>(p, s); }
int vc_scan_launch_step(const void* gates, long long sb, float* state, void* h, int B, int H, bool is_bf16, hipStream_t s) {
    const dim3 grid((H + 255) / 256, B < 4096 ? B : 4096);
    (void)hipGetLastError();
    if (is_bf16) hipLaunchKernelGGL((scan_step_kernel<bf16>), grid, dim3(256), 0, s, (const bf16*)gates, sb, state, (bf16*)h, B, H);
    else hipLaunchKernelGGL((scan_step_kernel<float>), grid, dim3(256), 0, s, (const float*)gates, sb, state, (float*)h, B, H);
    return launched("gated_scan_step");
}
