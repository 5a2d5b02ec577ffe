// Gated linear recurrence over time (gfx950), forward, backward and the single step of serving.
//
//   f_t = sigmoid(z_t)      h_t = f_t h_(t-1) + (1 - f_t) v_t        gates[b][t] = (z | v), H values each
//   backward, from the last step down (mu = what the future hands to h_t; dlast behind the last step):
//     lam_t = dy_t + mu      dv_t = (1 - f_t) lam_t      dz_t = lam_t (h_(t-1) - v_t) f_t (1 - f_t)      mu <- f_t lam_t
//   dh0 = mu in front of the first step.
//
// A step is an affine map of the state, h -> a h + b, and maps compose: (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2).  So a
// workgroup takes a tile of steps x 128 channels at once (64, 32 or 16 where there are no more, and more steps): each wave composes
// the maps of its own SUB steps (two channels per lane, held in registers), the waves exchange their compositions through LDS,
// and with the state in front of its first step each wave runs its steps again and writes them.  gates are read from memory once, h is written once.  The backward pass
// needs h_(t-1) and does not read h: it recomputes the states from the gates, which it has to read anyway, starting at the
// fp32 states that the forward saved every VC_SCAN_CHUNK steps (4 bytes per 64 steps and channel against 2-4 bytes per step,
// and without the rounding of a 16-bit h inside h_(t-1) - v_t).
//
// The tiles of one sequence run at the same time (one sequence of 1024 channels is 8 workgroups otherwise), and hand their states on
// as D. Merrill and M. Garland describe for sums (Single-pass parallel prefix scan with decoupled look-back, 2016).  A tile publishes
// its composition as soon as it has it; the state in front of a tile is the nearest state that an earlier tile has published,
// carried through the compositions in between, always from the earlier to the later tile: the same operations on the same
// numbers whichever state was found, so results do not depend on timing.  Every published word is 64 bits with its own
// ready mark (words are 0 before), written and read by relaxed device-scope atomics: no fence, no L2 write-back.  Tiles take
// their number from a counter, earlier steps first, so a tile only ever waits for tiles that run already, and every wait ends.
//
// Measured (copies on this card reach 5.14 TB/s): 8 x 2048 x 2048 bf16 forward 44 us = 4.6 TB/s, backward 82 us = 4.1; one
// sequence of 131072 x 1024 181 us = 4.45 TB/s.
//
// All arithmetic and the state are fp32; h and dgates round once, to their type.  1 - f is computed as its own quotient
// (sigmoid(-z)), so that a gate near 1 keeps its relative precision.
#include <type_traits>

#include "common.h"
#include "kernels.h"

// every product and sum as written: the paths below (whole waves or not, dy there or not) give the same bits
#pragma clang fp contract(off)

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
// a b + c
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { return {__builtin_fmaf(a.x, b.x, c.x), __builtin_fmaf(a.y, b.y, c.y)}; }

// Two neighbouring channels as they lie in memory, one load or store for both, at any multiple of an element (the hardware takes
// addresses of any alignment; one by one, 8 x 2048 x 2047 bf16, forward and backward, took 250 us instead of 177).  What a lane of the last
// column does with H odd: it loads the channel in front of its own beside it, so that nothing behind the row is read, and stores
// one value.  H = 1 has none in front: values one by one.
enum Channels { EVEN, ODD, ONE };
template <typename T>
struct Raw;
template <>
struct Raw<bf16> {
    typedef unsigned any_t __attribute__((aligned(2)));
    unsigned w;
    template <Channels C>
    __device__ __forceinline__ void load(const bf16* p, int d) {
        if (C == EVEN) w = *(const any_t*)p;
        else if (C == ODD) {
            w = *(const any_t*)(p - 1 + d);
            w = d ? w : w >> 16;
        } else
            w = *(const unsigned short*)p;
    }
    __device__ __forceinline__ f2 get() const { return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }
};
template <>
struct Raw<float> {
    float a, b;
    template <Channels C>
    __device__ __forceinline__ void load(const float* p, int d) {
        if (C == ONE) a = b = p[0];
        else {
            float v[2];
            __builtin_memcpy(v, C == ODD ? p - 1 + d : p, 8);
            a = C == ODD && !d ? v[1] : v[0], b = v[1];
        }
    }
    __device__ __forceinline__ f2 get() const { return {a, b}; }
};
__device__ __forceinline__ void put2(float* p, f2 v) { __builtin_memcpy(p, &v, 8); }
__device__ __forceinline__ void put2(bf16* p, f2 v) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    *(Raw<bf16>::any_t*)p = __builtin_bit_cast(unsigned, (bf16x2){f2bf(v.x), f2bf(v.y)});
}
// n: 0, 1 or 2 channels
template <typename T>
__device__ __forceinline__ void store2(T* p, f2 v, int n) {
    if (n == 2) put2(p, v);
    else if (n == 1) p[0] = (T)v.x;
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
                    h = fma2({__uint_as_float((unsigned)(x[i] >> 32) & 0x7fffffffu), __uint_as_float((unsigned)(y[i] >> 32) & 0x7fffffffu)}, h,
                             {low(x[i]), low(y[i])});
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

// (a later map behind an earlier one)
struct Map {
    f2 a, b;
};
__device__ __forceinline__ Map after(Map later, Map earlier) {
    return {{later.a.x * earlier.a.x, later.a.y * earlier.a.y}, fma2(later.a, earlier.b, later.b)};
}
__device__ __forceinline__ f2 apply(Map m, f2 h) { return fma2(m.a, h, m.b); }
// Few channels: LANES of a wave's lanes hold the channels (two each), the next LANES the following steps, and so on.
// Compositions over a wave's groups of lanes: `m` becomes that of all groups up to and with the own (DOWN: from the own on, in
// the backward's order); returns that of the groups in front of the own.
template <int LANES, bool DOWN>
__device__ __forceinline__ Map over_groups(Map& m, int lane) {
    Map e = {{1.f, 1.f}, {0.f, 0.f}};
    if constexpr (LANES < 64) {
        auto from = [&](Map v, int by) {
            const int src = DOWN ? lane + by : lane - by;
            return Map{{__shfl(v.a.x, src, 64), __shfl(v.a.y, src, 64)}, {__shfl(v.b.x, src, 64), __shfl(v.b.y, src, 64)}};
        };
        auto has = [&](int by) { return DOWN ? lane + by < 64 : lane >= by; };
#pragma unroll
        for (int by = LANES; by < 64; by *= 2) {
            const Map o = from(m, by);
            if (has(by)) m = after(m, o);
        }
        const Map o = from(m, LANES);
        if (has(LANES)) e = o;
    }
    return e;
}

// what a workgroup and a lane of it work on
template <typename T, int LANES>
struct Place {
    int tile, ntiles, c, n, d, b, len;  // c: first of the lane's n (0, 1, 2) channels (0 if it has none); d: to its second
    Between between;
    __device__ Place(const VcScanParams& p, int steps, int lane, int* shared) {
        const int cols = (p.H + 2 * LANES - 1) / (2 * LANES);
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
        c = (id - b * cols) * (2 * LANES) + (lane & (LANES - 1)) * 2;
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

template <typename T, int WAVES, int SUB, Channels C, int LANES>
__global__ __launch_bounds__(WAVES * 64, 4) void scan_fwd_kernel(const VcScanParams p) {
    constexpr int GROUPS = 64 / LANES, TILE = WAVES * GROUPS * SUB;
    static_assert(TILE % VC_SCAN_CHUNK == 0 && VC_SCAN_CHUNK % SUB == 0, "saved states sit where a wave starts");
    __shared__ float4 agg[WAVES][LANES];
    __shared__ f2 carry[LANES];
    __shared__ int shared;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int cl = lane & (LANES - 1), group = LANES < 64 ? lane / LANES : 0;
    const Place<T, LANES> L(p, TILE, lane, &shared);
    T* const out = (T*)p.h + (long long)L.b * p.T * p.H + L.c;
    const int w0 = L.tile * TILE + (wave * GROUPS + group) * SUB;  // the lane's first step (the wave's, with one group)
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
                    z[j].template load<C>(g + j * st, L.d);
                    v[j].template load<C>(g + j * st + p.H, L.d);
                }
            } else {
#pragma unroll
                for (int j = 0; j < SUB; ++j) {
                    const long long at = (j < left ? j : left - 1) * st;  // (read again, not used)
                    z[j].template load<C>(g + at, L.d);
                    v[j].template load<C>(g + at + p.H, L.d);
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
                b = fma2(f[j], b, u[j]);
            }
        };
        if (LANES == 64 ? left >= SUB : __all(left >= SUB)) compose(std::true_type());
        else compose(std::false_type());
        Map own = {a, b};
        const Map front = over_groups<LANES, false>(own, lane);
        if (group == GROUPS - 1) agg[wave][cl] = make_float4(own.a.x, own.a.y, own.b.x, own.b.y);
        __syncthreads();
        if (wave == 0) {
            const int n = group == 0 ? L.n : 0;
            f2 h;
            if (L.tile == 0) h = p.h0 != nullptr ? f2{p.h0[sc], p.h0[sc + L.d]} : f2{0.f, 0.f};
            a = {1.f, 1.f}, b = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float4 m = agg[w][cl];
                a = {a.x * m.x, a.y * m.y};
                b = fma2({m.x, m.y}, b, {m.z, m.w});
            }
            const bool more = (L.tile + 1) * TILE < L.len;
            if (L.tile > 0) {
                if (more) L.between.put_map(L.tile, a, b, n);
                h = L.between.before(L.tile);
            }
            if (group == 0) carry[cl] = h;
            h = fma2(a, h, b);
            if (more) L.between.put_state(L.tile, h, n);
            else store2(p.last + sc, h, n);
        }
        __syncthreads();
        f2 h = carry[cl];
        for (int w = 0; w < wave; ++w) {
            const float4 m = agg[w][cl];
            h = fma2({m.x, m.y}, h, {m.z, m.w});
        }
        if (LANES < 64) h = apply(front, h);
        if (p.states != nullptr && w0 % VC_SCAN_CHUNK == 0 && left > 0) {
            const long long chunks = (p.T + VC_SCAN_CHUNK - 1) / VC_SCAN_CHUNK;
            store2(p.states + (L.b * chunks + w0 / VC_SCAN_CHUNK) * p.H + L.c, h, L.n);
        }
        T* const o = out + t0 * p.H;
        const long long so = (long long)p.H * dt;
        auto write = [&](auto whole) {
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                h = fma2(f[j], h, u[j]);
                if (decltype(whole)::value) put2(o + j * so, h);
                else if (j < left) store2(o + j * so, h, L.n);
            }
        };
        if (C == EVEN && __all(left >= SUB && L.n == 2)) write(std::true_type());
        else write(std::false_type());
    } else if (L.len == 0 && L.tile == 0 && wave == 0)
        store2(p.last + sc, p.h0 != nullptr ? f2{p.h0[sc], p.h0[sc + L.d]} : f2{0.f, 0.f}, L.n);
    if (left < SUB)  // behind the end: zeros
        for (int t = left > 0 ? L.len : w0; t < w0 + SUB && t < p.T; ++t) store2(out + (long long)t * p.H, {0.f, 0.f}, L.n);
}

template <typename T, int WAVES, int SUB, Channels C, int LANES>
__global__ __launch_bounds__(WAVES * 64, 4) void scan_bwd_kernel(const VcScanParams p) {
    constexpr int GROUPS = 64 / LANES, TILE = WAVES * GROUPS * SUB;
    static_assert(TILE % VC_SCAN_CHUNK == 0, "a tile starts at a saved state");
    __shared__ float4 agg[WAVES][LANES];  // forward maps
    __shared__ f2 back[WAVES][LANES];     // constant part of the backward maps (their factor is the forward's)
    __shared__ f2 carry[LANES];
    __shared__ int shared;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int cl = lane & (LANES - 1), group = LANES < 64 ? lane / LANES : 0;
    const Place<T, LANES> L(p, TILE, lane, &shared);
    const int tile = L.ntiles - 1 - L.tile;                  // the last steps come first
    const int first = (L.len + TILE - 1) / TILE - 1 - tile;  // tiles of this sequence that come before
    T* const out = (T*)p.dgates + (long long)L.b * p.T * 2 * p.H + L.c;
    const int w0 = tile * TILE + (wave * GROUPS + group) * SUB, left = L.len - w0;
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
                z[j].template load<C>(g + at, L.d);
                v[j].template load<C>(g + at + p.H, L.d);
            }
            if (p.dy != nullptr) {
                const T* const y = (const T*)p.dy + ((long long)L.b * p.T + t0) * p.H + L.c;
                const long long so = (long long)p.H * dt;
#pragma unroll
                for (int j = 0; j < SUB; ++j) d[j].template load<C>(y + (j < left ? j : left - 1) * so, L.d);
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
                    b = fma2(f[j], b, {q[j].x * vv.x, q[j].y * vv.y});
                }
                a = {a.x * f[j].x, a.y * f[j].y};
            }
#pragma unroll
            for (int j = SUB - 1; j >= 0; --j) {
                const f2 e = dy(j, whole);
                c = {f[j].x * (e.x + c.x), f[j].y * (e.y + c.y)};
            }
        };
        if (has_dy && (LANES == 64 ? left >= SUB : __all(left >= SUB))) compose(std::true_type());
        else compose(std::false_type());
        Map own = {a, b}, future = {a, c};
        const Map front = over_groups<LANES, false>(own, lane), behind = over_groups<LANES, true>(future, lane);
        if (group == GROUPS - 1) agg[wave][cl] = make_float4(own.a.x, own.a.y, own.b.x, own.b.y);
        if (group == 0) back[wave][cl] = future.b;
        __syncthreads();
        if (wave == 0) {
            const int n = group == 0 ? L.n : 0;
            f2 mu;
            if (first == 0) mu = p.dlast != nullptr ? f2{p.dlast[sc], p.dlast[sc + L.d]} : f2{0.f, 0.f};
            a = {1.f, 1.f}, c = {0.f, 0.f};
#pragma unroll
            for (int w = WAVES - 1; w >= 0; --w) {
                const float4 m = agg[w][cl];
                const f2 k = back[w][cl];
                a = {a.x * m.x, a.y * m.y};
                c = fma2({m.x, m.y}, c, k);
            }
            if (first > 0) {
                if (tile > 0) L.between.put_map(first, a, c, n);
                mu = L.between.before(first);
            }
            if (group == 0) carry[cl] = mu;
            mu = fma2(a, mu, c);
            if (tile > 0) L.between.put_state(first, mu, n);
            else if (p.dh0 != nullptr) store2(p.dh0 + sc, mu, n);
        }
        const long long chunks = (p.T + VC_SCAN_CHUNK - 1) / VC_SCAN_CHUNK;
        const float* st = p.states + (L.b * chunks + tile * (TILE / VC_SCAN_CHUNK)) * p.H + L.c;
        f2 h = {st[0], st[L.d]};
        for (int w = 0; w < wave; ++w) {
            const float4 m = agg[w][cl];
            h = fma2({m.x, m.y}, h, {m.z, m.w});
        }
        if (LANES < 64) h = apply(front, h);
        __syncthreads();
        f2 mu = carry[cl];
        for (int w = WAVES - 1; w > wave; --w) {
            const float4 m = agg[w][cl];
            const f2 k = back[w][cl];
            mu = fma2({m.x, m.y}, mu, k);
        }
        if (LANES < 64) mu = apply(behind, mu);
        f2 before[SUB];
        T* const o = out + t0 * 2 * p.H;
        const long long so = 2ll * p.H * dt;
        auto write = [&](auto whole) {
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                const f2 vv = v[j].get();
                before[j] = h;
                if (decltype(whole)::value || j < left) h = fma2(f[j], h, {q[j].x * vv.x, q[j].y * vv.y});
            }
#pragma unroll
            for (int j = SUB - 1; j >= 0; --j) {
                const f2 e = dy(j, whole), lam = {e.x + mu.x, e.y + mu.y}, vv = v[j].get();
                mu = {f[j].x * lam.x, f[j].y * lam.y};
                const f2 dv = {q[j].x * lam.x, q[j].y * lam.y};
                const f2 dz = {mu.x * q[j].x * (before[j].x - vv.x), mu.y * q[j].y * (before[j].y - vv.y)};
                if (decltype(whole)::value) {
                    put2(o + j * so, dz);
                    put2(o + j * so + p.H, dv);
                } else if (j < left) {
                    store2(o + j * so, dz, L.n);
                    store2(o + j * so + p.H, dv, L.n);
                }
            }
        };
        if (C == EVEN && has_dy && __all(left >= SUB && L.n == 2)) write(std::true_type());
        else write(std::false_type());
    } else if (L.len == 0 && tile == 0 && wave == 0 && p.dh0 != nullptr)
        store2(p.dh0 + sc, p.dlast != nullptr ? f2{p.dlast[sc], p.dlast[sc + L.d]} : f2{0.f, 0.f}, L.n);
    if (left < SUB)  // behind the end: zeros
        for (int t = left > 0 ? L.len : w0; t < w0 + SUB && t < p.T; ++t) {
            store2(out + (long long)t * 2 * p.H, {0.f, 0.f}, L.n);
            store2(out + (long long)t * 2 * p.H + p.H, {0.f, 0.f}, L.n);
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
        const float n = __builtin_fmaf(f, state[e], q * (float)row[H]);
        state[e] = n;
        h[e] = (T)n;
    }
}

// Rows of D values with 64 more columns behind each, for a product that is to add a bias: 1 1 1 0 ... behind the rows of x, and behind
// those of W the bias as three numbers of 8 bits, whose sum it is: the product's fp32 sums then hold x W^T + b, and round once.  A wave
// per row, four values a lane at a time.  Bound by HBM: 16384 x 2048 to bf16 36 us = 5.6
// TB/s; a weight of 4096 x 2048 12 us.
template <typename T>
__global__ __launch_bounds__(256) void bias_columns_kernel(const float* in, const float* bias, T* out, long long rows, int D) {
    const int lane = threadIdx.x & 63, width = D + 64;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (long long)gridDim.x * 4) {
        const float* const from = in + r * D;
        T* const to = out + r * width;
        for (int c = lane * 4; c < width; c += 256) {
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (c < D) __builtin_memcpy(&v, from + c, 16);
            else if (c == D && bias == nullptr) v = (f32x4){1.f, 1.f, 1.f, 0.f};
            else if (c == D) {
                float rest = bias[r];
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    v[k] = bf2f(f2bf(rest));
                    rest = fabsf(v[k]) < INFINITY ? rest - v[k] : 0.f;
                }
            }
            if constexpr (sizeof(T) == 2) {
                const bf16x4 o = {f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])};
                __builtin_memcpy(to + c, &o, 8);
            } else
                __builtin_memcpy(to + c, &v, 16);
        }
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

// Forward, bf16: 16 waves of 16 steps, one workgroup a CU.  Half as many waves or steps: 8 .. 30 % slower (a sequence is more
// tiles, whose states wait for each other, and a wave has fewer loads in flight); 32 steps spill.  fp32: 8 steps (its 16 spill: 8 x
// 2048 x 2048 forward and backward 240 against 228 us, 32 x 23 x 3686 forward 22.7 against 15.2).  Backward: its three inputs and
// h in registers leave room for 8 steps; 16 waves against 8: one sequence of 131072 x 512 320 against 433 us, 32 sequences
// of 2048 x 1024 262 against 258.  Workgroups that stay and ask for their next tile's gates while they finish one measured 20 %
// slower in both directions (more registers, fewer loads in flight).
constexpr int WAVES = 16, BWD_SUB = 8;
constexpr int fwd_sub(bool is_bf16) { return is_bf16 ? 16 : 8; }

// lanes of a wave that hold channels: the fewest that hold all of them (bf16, forward and backward: 45 x 8291 x 32 147 us
// with 64, 76 with 16; 1 x 131072 x 16 205 with 64, 78 with 8)
int lanes(int H) { return H > 64 ? 64 : H > 32 ? 32 : H > 16 ? 16 : 8; }
int tile_steps(int H, bool is_bf16, int op) { return WAVES * (op == 0 ? fwd_sub(is_bf16) : BWD_SUB) * (64 / lanes(H)); }
// the workgroups of one sequence
long long workgroups(int T, int H, bool is_bf16, int op) {
    const int steps = tile_steps(H, is_bf16, op), channels = 2 * lanes(H);
    return ((long long)T + steps - 1) / steps * ((H + channels - 1) / channels);
}
// a launch has fewer than 2^32 lanes (HIP's limit for a dimension of the grid)
constexpr long long MOST_WORKGROUPS = ((1ll << 32) - 1) / (WAVES * 64);

// the sequences from b on, n of them
VcScanParams part(const VcScanParams& p, bool is_bf16, int b, int n) {
    const long long elem = is_bf16 ? 2 : 4, row = (long long)b * p.H, steps = row * p.T;
    const auto at = [](const void* q, long long bytes) { return q != nullptr ? (char*)q + bytes : nullptr; };
    VcScanParams q = p;
    q.B = n;
    q.gates = at(p.gates, b * p.sb * elem);
    q.lengths = (const int*)at(p.lengths, b * 4ll);
    q.h0 = (const float*)at(p.h0, row * 4), q.last = (float*)at(p.last, row * 4);
    q.dlast = (const float*)at(p.dlast, row * 4), q.dh0 = (float*)at(p.dh0, row * 4);
    q.states = (float*)at(p.states, row * ((p.T + VC_SCAN_CHUNK - 1) / VC_SCAN_CHUNK) * 4);
    q.h = at(p.h, steps * elem), q.dy = at(p.dy, steps * elem), q.dgates = at(p.dgates, 2 * steps * elem);
    return q;
}

template <typename T, Channels C, int LANES>
void launch(const VcScanParams& all, int op, hipStream_t s) {
    constexpr bool is_bf16 = sizeof(T) == 2;
    const long long each = workgroups(all.T, all.H, is_bf16, op), most = MOST_WORKGROUPS / each;
    for (long long b = 0; b < all.B; b += most) {  // (all sequences in one launch up to some 4 million workgroups)
        const VcScanParams p = part(all, is_bf16, (int)b, (int)(all.B - b < most ? all.B - b : most));
        // what the tiles exchange their states through
        const long long n = (long long)vc_scan_workspace(p.B, p.T, p.H, is_bf16, op) / 16, blocks = (n + 255) / 256;
        if (n > 0) hipLaunchKernelGGL(scan_clear_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, (uint4*)p.ws, n);
        const dim3 grid((unsigned)(each * p.B)), block(WAVES * 64);
        if (op == 0) hipLaunchKernelGGL((scan_fwd_kernel<T, WAVES, fwd_sub(is_bf16), C, LANES>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((scan_bwd_kernel<T, WAVES, BWD_SUB, C, LANES>), grid, block, 0, s, p);
    }
}
template <typename T, Channels C>
void launch(const VcScanParams& p, int op, hipStream_t s) {
    switch (lanes(p.H)) {
        case 64: return launch<T, C, 64>(p, op, s);
        case 32: return launch<T, C, 32>(p, op, s);
        case 16: return launch<T, C, 16>(p, op, s);
        default: return launch<T, C, 8>(p, op, s);
    }
}
template <typename T>
void launch(const VcScanParams& p, int op, hipStream_t s) {
    if (p.H % 2 == 0) launch<T, EVEN>(p, op, s);
    else if (p.H > 1) launch<T, ODD>(p, op, s);
    else launch<T, ONE, 8>(p, op, s);
}

}  // namespace

bool vc_scan_fits(int T, int H, bool is_bf16) { return workgroups(T, H, is_bf16, 0) <= MOST_WORKGROUPS && workgroups(T, H, is_bf16, 1) <= MOST_WORKGROUPS; }
// what the tiles of a sequence exchange: 0 where a sequence is one tile
size_t vc_scan_workspace(int B, int T, int H, bool is_bf16, int op) {
    const int steps = tile_steps(H, is_bf16, op);
    const long long tiles = ((long long)T + steps - 1) / steps;
    return tiles > 1 ? (size_t)(256 + 2 * 8 * tiles * B * H) : 0;
}
int vc_scan_launch_fwd(const VcScanParams& p, bool is_bf16, hipStream_t s) {
    (void)hipGetLastError();
    if (is_bf16) launch<bf16>(p, 0, s);
    else launch<float>(p, 0, s);
    return launched("gated_scan_fwd");
}
int vc_scan_launch_bwd(const VcScanParams& p, bool is_bf16, hipStream_t s) {
    (void)hipGetLastError();
    if (is_bf16) launch<bf16>(p, 1, s);
    else launch<float>(p, 1, s);
    return launched("gated_scan_bwd");
}
int vc_scan_launch_step(const void* gates, long long sb, float* state, void* h, int B, int H, bool is_bf16, hipStream_t s) {
    const dim3 grid((H + 255) / 256, B < 4096 ? B : 4096);
    (void)hipGetLastError();
    if (is_bf16) hipLaunchKernelGGL((scan_step_kernel<bf16>), grid, dim3(256), 0, s, (const bf16*)gates, sb, state, (bf16*)h, B, H);
    else hipLaunchKernelGGL((scan_step_kernel<float>), grid, dim3(256), 0, s, (const float*)gates, sb, state, (float*)h, B, H);
    return launched("gated_scan_step");
}
int vc_bias_columns_launch(const float* in, const float* bias, void* out, bool to_bf16, long long rows, int D, hipStream_t s) {
    const dim3 grid((unsigned)(rows < 4 * 65536 ? (rows + 3) / 4 : 65536));
    (void)hipGetLastError();
    if (to_bf16) hipLaunchKernelGGL((bias_columns_kernel<bf16>), grid, dim3(256), 0, s, in, bias, (bf16*)out, rows, D);
    else hipLaunchKernelGGL((bias_columns_kernel<float>), grid, dim3(256), 0, s, in, bias, (float*)out, rows, D);
    return launched("bias_columns");
}
