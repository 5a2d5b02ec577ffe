// Linear classifier and cross-entropy in one operator (gfx950), for vocabularies whose logits are not worth keeping.
//
//   z = x w^T + b      loss_n = lse_n - z[n][label_n]      lse_n = log sum_v exp z[n][v]
//   P[n][v] = exp(z[n][v] - lse_n) - [v = label_n]      dx = g P w      dw = g P^T x      db = g sum_n P[n]
//   g = upstream / count (mean), upstream (sum); with reduction 0 each row's own g_n multiplies its row of P instead
//
// Forward: every tile of the product x w^T ends in its registers as a (maximum, sum of exponentials) pair for each of its
// rows; a second launch joins a row's pairs.  Backward: the vocabulary goes by in pieces; a piece's logits are computed
// again, turned into P (rounded once, to the operands' type, for the two matrix products that read it) and multiplied into
// dx and dw.  A factor g common to all rows stays out of P: P at the label is close to -1 in every row, and g times that would
// round by the same amount in all of them, an error that adds up (measured: 3.5e-3 of dw instead of 2.3e-3 with bf16).  N x V is
// not held.
// Where memory allows and it is quicker (vc_lce_keep), the forward keeps more: tiles store exp(z - ref) with ref = the logit of
// the row's own label, which is known beforehand (EPI_KEEP); once the row's sum is known a pass over them makes P of them, where
// they lie, and the backward is its two products.  ref is at most the row's maximum, so nothing of weight underflows; where some
// exp(z - ref) passes 2^64 the forward computes P as the backward would have.
//
// Rows whose label is ignore_index take no part: the rows that count are listed first (rows_kernel) and all products run
// over that list, so that an ignored row costs nothing and whatever it holds (NaN included) reaches nothing.
#include <type_traits>

#include "common.h"
#include "kernels.h"


namespace {

// ---------------------------------------------------------------- the list of rows
// rows[0 .. count) = the rows that count, ascending; rows[N - 1 - j] = the j-th row that does not; rows[N] = count
__global__ __launch_bounds__(1024) void rows_kernel(const long long* labels, long long ignore, int N, int* rows) {
    __shared__ int part[16], base_sh;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    int base = 0;
    for (int n0 = 0; n0 < N; n0 += 1024) {
        const int n = n0 + tid;
        const bool in = n < N, keep = in && labels[n] != ignore;
        const unsigned long long mask = __ballot(keep);
        if (lane == 0) part[wave] = __popcll(mask);
        __syncthreads();
        int before = base;
        for (int w = 0; w < wave; ++w) before += part[w];
        const int k = before + __popcll(mask & ((1ull << lane) - 1));  // rows that count before n
        if (keep) rows[k] = n;
        else if (in) rows[N - 1 - (n - k)] = n;
        if (tid == 1023) base_sh = k + (keep ? 1 : 0);
        __syncthreads();
        base = base_sh;
    }
    if (tid == 0) rows[N] = base, rows[N + 1] = 0, rows[N + 2] = 0;  // (their number; workgroups of lce_rows_kernel that are done; EPI_KEEP gave up)
}

// ---------------------------------------------------------------- matrix products
// out[s][r] = sum_k S(s, k) R(r, k).  A workgroup of WR x WS waves makes a BR x BS tile (256, 128 or 64 square), a wave BR/WR x
// BS/WS of it, in steps of one or two fragments of k (a fragment: 32 bf16 or 16 fp32, 64 bytes; Feed says which).  The operands'
// tiles come in by DMA (global_load_lds, 16 bytes a lane) into a ring of two or four buffers, one or three steps ahead of their
// use.  An operand lies in memory with k contiguous (rows of x, w; P for dx) or with its rows contiguous and k across (w for dx;
// x and P for dw: nothing is transposed in memory):
//   k contiguous: LDS rows of 64 or 128 bytes; a fragment is one ds_read_b128.  The 16-byte chunk c of row r lies at slot
//     c ^ turn(r): of the sixteen lanes that one cycle pair serves, whether they are rows 0-15 of one chunk or rows 0-3,
//     12-15 of one and 4-11 of the next, no two meet in a bank (measured: 0 conflicts).
//   k across: LDS rows of one k each.  bf16: fragments come through ds_read_b64_tr_b16, which hands lane i of 16 the i-th
//     column of four rows; a lane group reads four rows x 32 bytes, so the 32-byte unit u of row k lies at u ^ f(k) with f
//     different for the eight rows that half a wave reads at once.  fp32: one ds_read_b32 a value, units of 64 bytes at u ^ (k / 4 % 4).
// The swizzles act on the DMA's source address: what a lane fetches, not where it lands.
// Bound by the matrix cores' issue: the loops of 256 x 256 tiles run at some 1.25 PFLOP/s (59 % of the cycles issue a matrix
// instruction, at 2.1 GHz), near what a large library product reaches here (1.33).  1843 rows x 1024 of 32768, us: EPI_STATS 133,
// EPI_KEEP 156, EPI_PROB 156, EPI_DX 133, EPI_DW 120 (123.7 GFLOP each); 7373 x 2048 of 65536: 1555, 1791, 1898, 1734, 1573 (1979
// GFLOP each).  The difference of the first three is the epilogue's stores.  What did not help: fragments read four slots ahead
// or raised wave priority (within 1 %), tiles of 256 x 128 in three buffers, two workgroups a CU (+2 .. +20 %), rows of 64 bytes
// of k for the forward (+15 %), touching the next lines early (+10 %), workgroups that stay and fetch their next tile during the epilogue (+33 %: registers spill).
// Nothing is read outside the operands: rows and columns behind the end are read from a row or column inside (what they make
// is not stored), k behind the end from a page of zeros (k contiguous) or, with k across, from a k inside, where the other
// operand, P, is 0 (EPI_PROB writes whole tiles of P, zeros behind the last row and the last word).
struct Operand {
    const char* p;
    long long ld;  // bytes from row to row (k contiguous) or from k to k (k across), below 2^32
};

enum { EPI_STATS, EPI_KEEP, EPI_PROB, EPI_DX, EPI_DW };

// the factor common to all rows
struct Factor {
    const float* dloss;
    const int* count;
    int reduction;
    __device__ __forceinline__ float get() const {
        if (reduction == 0) return 1.f;
        const int n = *count;
        return reduction == 1 ? dloss[0] / (float)(n > 0 ? n : 1) : dloss[0];
    }
};

// The product for dx has few tiles and a long k: k is split, each split into sums of its own, so that all tiles make one round on
// the chip (`slots` workgroups at once).  The tiles that there are decide, not those that the launch allows for (1777 rows of
// which 1244 count: 4 splits by the former, 6 by the latter, 232 against 178 us).
struct Splits {
    int slots, most, rtiles, bs;
    __device__ __forceinline__ int of(int ns) const {
        const int t = rtiles * ((ns + bs - 1) / bs), z = t > 0 ? slots / t : 1;
        return z < 1 ? 1 : z > most ? most : z;
    }
};

struct Gemm {
    Operand R, S;
    int nr, ns, K;      // K: where k is contiguous in an operand, a multiple of its 16-byte chunk
    const int* ns_dev;  // nullable: ns is *ns_dev
    const int* k_dev;   // nullable: K is *k_dev
    int rtiles;
    Splits splits;  // EPI_DX
    const int* when;  // nullable: nothing is done where *when is 0
    // EPI_STATS / EPI_KEEP / EPI_PROB: r = word v0 + r, s = listed row
    const void* bias;
    const long long* labels;
    const int* rows;
    int v0;
    float2* part;  // [s][part_ld], this launch's tiles from part0 on
    int part_ld, part0;
    float* zlab;   // [s]: logit of the row's label
    const float* ref;  // EPI_KEEP: [s], what a row's exponentials are taken relative to
    int* gave_up;      // EPI_KEEP
    const float* lse;
    const float* scale;  // nullable: [N], each row's own factor
    void* P;
    long long ldp;
    float* dbpart;   // nullable: [s tile][ldp]
    float* acc;      // EPI_DX: [split][s][nr]
    long long acc_split;
    int add;
    void* out;       // EPI_DW: [s][nr]
    Factor factor;   // EPI_DW
};

typedef __attribute__((address_space(3))) void* lptr_t;
typedef __attribute__((address_space(3))) s16x4* ltr_t;

__device__ __attribute__((aligned(128))) unsigned int vc_lce_zero_page[32];

template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    static constexpr int KF = 32, PER = 8;  // k of a fragment, of a 16-byte chunk
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<float> {
    static constexpr int KF = 16, PER = 4;
    typedef f32x4 frag;
    // four instructions of k = 4; k is dealt to the lane groups in fours, alike for both operands
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// 16 bytes per lane from `src` to LDS at the wave-uniform `lds` + 16 * lane.  Written out, not the builtin: the compiler knows
// which LDS the builtin writes only as "some", and waits for every such load before any transposed read (measured: the products
// with k across 1.9x slower); here the waits at the end of a step are all there are.  It has no result register; the address
// registers are read when it issues.
__device__ __forceinline__ void dma(unsigned lds, const char* src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "m0");
}

// one operand of a tile: ROWS rows by the k of SUBS fragments, KACROSS = k across
template <typename T, int ROWS, int SUBS, int NTHR, bool KACROSS>
struct Tile {
    static constexpr int STEP = Mma<T>::KF * SUBS, PER = Mma<T>::PER, ROWB = 64 * SUBS, BYTES = ROWS * ROWB;
    static constexpr int PIECES = BYTES / 16 / NTHR;      // 16-byte pieces of a thread
    static constexpr int CPR = KACROSS ? ROWS / PER : 4 * SUBS;  // chunks of an LDS row
    static constexpr int RPP = NTHR / CPR;                // LDS rows of one pass of the workgroup
    const char* p[PIECES];  // k contiguous: a piece at k = 0; k across: its column at k = 0
    int tid;
    // k across: what a piece's chunk of a row of one k is moved by
    // (64 columns of bf16 are four units only: two rows then share a bank)
    static __device__ __forceinline__ int swz(int k) { return sizeof(T) == 2 ? ((k & 3) | (ROWS > 64 ? (k >> 3) & 1 : 0) << 2) << 1 : ((k >> 2) & 3) << 2; }
    // k contiguous: what a chunk of row r is moved by
    static __device__ __forceinline__ int turn(int r) {
        const int h = (r >> 2) & 3;
        return SUBS == 2 ? (r >> 1) & 7 : (h >> 1) | ((h ^ (h >> 1)) & 1) << 1;
    }
    __device__ __forceinline__ int chunk() const { return (tid % CPR) ^ turn(tid / CPR); }  // k contiguous: of every piece (rows differ by 16s)

    __device__ __forceinline__ void init(const Operand& o, int row0, int nrows) {
        static_assert(KACROSS || RPP % 16 == 0, "");
        tid = threadIdx.x;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            if (!KACROSS) {
                const int row = row0 + j * RPP + tid / CPR;
                p[j] = o.p + (row < nrows ? row : nrows - 1) * o.ld + chunk() * 16;
            } else {
                const int c = row0 + ((tid % CPR) ^ swz(j * RPP + tid / CPR)) * PER;
                p[j] = o.p + (c < nrows ? c : 0) * (int)sizeof(T);
            }
        }
    }
    // piece j of the step at k0
    __device__ __forceinline__ void issue(const Operand& o, unsigned lds, int k0, int K, int j) const {
        const char* src;
        if (!KACROSS) {
            src = p[j] + (long long)k0 * (int)sizeof(T);
            if (k0 + STEP > K) src = k0 + chunk() * PER >= K ? (const char*)vc_lce_zero_page : src;
        } else {
            const int k = k0 + j * RPP + tid / CPR;
            src = p[j] + (unsigned long long)(unsigned)(k < K ? k : K - 1) * (unsigned)o.ld;
        }
        dma(lds + j * NTHR * 16, src);
    }
    // the fragment of rows [row, row + 16), k of fragment `sub`
    static __device__ __forceinline__ typename Mma<T>::frag frag(const char* lds, int row, int sub, int l15, int lg) {
        if (!KACROSS) return *(const typename Mma<T>::frag*)(lds + row * ROWB + l15 * ROWB + (((sub * 4 + lg) ^ turn(l15)) << 4));
        const int u = row / 16;
        typename Mma<T>::frag f;
        if constexpr (sizeof(T) == 2) {
            const int k = lg * 8 + (l15 >> 2);
            const char* q = lds + (sub * 32 + k) * (ROWS * 2) + ((u ^ (swz(k) >> 1)) << 5) + (l15 & 3) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ltr_t)q), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ltr_t)(q + 4 * ROWS * 2));
            f = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = *(const float*)(lds + (sub * 16 + lg * 4 + i) * (ROWS * 4) + ((u ^ lg) << 6) + l15 * 4);
        }
        return f;
    }
};

// how a product's tiles come in: fragments of k a step, buffers of the ring
// Large tiles: where rows of k are read, 128 bytes of them (half a line a row costs the forward 15 %) and two buffers, all that
// fits; with k across four buffers of one fragment.
template <int EPI, int B>
struct Feed {
    static constexpr bool ROWS_OF_K = EPI == EPI_STATS || EPI == EPI_KEEP || EPI == EPI_PROB;
    static constexpr int SUBS = ROWS_OF_K || B == 64 ? 2 : 1, RING = ROWS_OF_K && B > 64 ? 2 : 4;
};

// Two 16 x 16 blocks of results, side by side: lane (l15, lg) holds u = columns 4 lg .. of row l15 of the first, v of the second.
// As bf16 they change hands so that a lane has 8 columns of one block (16-byte stores, 64 bytes of a row beside each other, where
// four columns make 8-byte ones, 32 bytes: the products of 2048 x 1024 of 32768 that store bf16 take 156 and 121 us instead of 167
// and 127); `at` is the first block's row.
template <typename T>
__device__ __forceinline__ void store_pair(T* at, int lg, f32x4 u, f32x4 v) {
    if constexpr (sizeof(T) == 2) {
        const uint2 a = __builtin_bit_cast(uint2, (bf16x4){f2bf(u[0]), f2bf(u[1]), f2bf(u[2]), f2bf(u[3])});
        const uint2 b = __builtin_bit_cast(uint2, (bf16x4){f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])});
        const auto x = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false), y = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
        const uint4 q = make_uint4(x[0], y[0], x[1], y[1]);
        __builtin_memcpy(at + (lg & 1) * 16 + (lg >> 1) * 8, &q, 16);
    } else {
        __builtin_memcpy(at + lg * 4, &u, 16);
        __builtin_memcpy(at + 16 + lg * 4, &v, 16);
    }
}

template <typename T, int EPI, int BR, int BS, int WR, int WS>
__global__ __launch_bounds__(WR* WS * 64, 2) void lce_gemm(const Gemm g) {
    constexpr int NTHR = WR * WS * 64, SUBS = Feed<EPI, BR>::SUBS, RING = Feed<EPI, BR>::RING, STEP = Mma<T>::KF * SUBS;
    constexpr int NA = BR / WR / 16, NB = BS / WS / 16;
    constexpr bool RK = EPI == EPI_DX || EPI == EPI_DW, SK = EPI == EPI_DW;
    typedef Tile<T, BR, SUBS, NTHR, RK> TR;
    typedef Tile<T, BS, SUBS, NTHR, SK> TS;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BUF = TR::BYTES + TS::BYTES;
    if (g.when != nullptr && *g.when == 0) return;
    const int ns = __builtin_amdgcn_readfirstlane(g.ns_dev != nullptr ? *g.ns_dev : g.ns);
    const int K = __builtin_amdgcn_readfirstlane(g.k_dev != nullptr ? *g.k_dev : g.K);
    // tile order: XCD x (workgroups go round the 8 XCDs) takes the x-th share of an order in which 4 tiles of s by all tiles of r
    // follow each other, so that the 32 workgroups of an XCD share 4 + 8 operand panels in its L2.  The shares are of the tiles
    // that there are: ns may be far below what the launch had to allow for (shares of all tiles of the launch: the XCDs with the
    // last tiles of s idle, 1777 rows of which 1244 count 221 us instead of 155).
    // A product with splits of k has its splits one after the other in that order: the tiles of a split share their panels.
    const int stiles = (ns + BS - 1) / BS, z = EPI == EPI_DX ? g.splits.of(ns) : 1;
    int r0, s0, st, split;
    {
        const unsigned tiles = (unsigned)g.rtiles * stiles, total = tiles * z;
        const unsigned lin = blockIdx.x, x = lin & 7u, base = total >> 3, rem = total & 7u;
        if (lin >= total) return;
        unsigned t = x * base + (x < rem ? x : rem) + (lin >> 3);
        split = (int)(t / tiles), t -= split * tiles;
        const unsigned per = 4u * g.rtiles, grp = t / per, in = t - grp * per;
        const unsigned left = stiles - grp * 4u, w = left < 4u ? left : 4u;
        r0 = (int)(in / w) * BR, st = (int)(grp * 4u + in % w), s0 = st * BS;
    }
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = (wave % WR) * (BR / WR), wsx = (wave / WR) * (BS / WS);
    f32x4 acc[NA][NB];
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[a][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
    int kb = 0, ke = K;
    if constexpr (EPI == EPI_DX) {
        const int each = ((K + z - 1) / z + 127) / 128 * 128;
        kb = split * each, ke = K < kb + each ? K : kb + each;
    }
    if (kb < ke) {
        TR tr;
        TS ts;
        tr.init(g.R, r0, g.nr);
        ts.init(g.S, s0, SK ? (int)(g.S.ld / (int)sizeof(T)) : ns);  // (P has whole tiles)
        constexpr int PIECES = TR::PIECES + TS::PIECES, SL = SUBS * NA;
        static_assert((RING - 2) * PIECES == 8 || RING == 2, "the waits below");
        const int ks = SK ? (K + STEP - 1) / STEP * STEP : K;  // (P has zeros up to there)
        const unsigned dst = (unsigned)(uintptr_t)(lptr_t)smem + wave * 1024;
        const int steps = (ke - kb + STEP - 1) / STEP;
        auto issue = [&](int t, int j) {
            const unsigned to = dst + (t & (RING - 1)) * BUF;
            if (j < TR::PIECES) tr.issue(g.R, to, kb + t * STEP, K, j);
            else ts.issue(g.S, to + TR::BYTES, kb + t * STEP, ks, j - TR::PIECES);
        };
        // A step is SL slots: one fragment of R and NB matrix instructions each.  Fragments are read two slots ahead of their
        // use.  Two slots before its end a wave has read all of the step's tiles: there it waits for the next step's tiles
        // (those of later steps may be under way) and meets the others; the last two slots run while the first fragments of
        // the next step are read.  The tiles of the step RING - 1 from here go to the buffer that the step before read, a
        // few pieces a slot: asked for all at once, they keep the wave from issuing anything else.
        constexpr int D = 2;  // slots from a fragment's read to its use
        static_assert(SL % (2 * D) == 0 && NB % D == 0, "");
        typename Mma<T>::frag fr[2 * D], fs[2][NB];
        for (int t = 0; t < RING - 1 && t < steps; ++t)
#pragma unroll
            for (int j = 0; j < PIECES; ++j) issue(t, j);
        if (RING > 2 && steps > RING - 2) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int b = 0; b < NB; ++b) fs[0][b] = TS::frag(smem + TR::BYTES, wsx + b * 16, 0, l15, lg);
#pragma unroll
        for (int i = 0; i < D; ++i) fr[i] = TR::frag(smem, wr + i * 16, 0, l15, lg);
        // A wave whose rows or columns all lie behind the end (its part of a tile at the end of the list) fetches and meets the others,
        // and leaves the matrix cores to the wave beside it (2048 x 1024 of 32768, 1843 rows: EPI_KEEP 154 -> 149 us; 6 x 1024 of
        // 114608 fp32: 168 -> 150)
        const bool some = s0 + wsx < ns && r0 + wr < g.nr;
        auto idle = [&](int t) {
            const bool more = t + RING - 1 < steps;
#pragma unroll
            for (int j = 0; j < PIECES; ++j)
                if (more) issue(t + RING - 1, j);
            if (RING > 2 && more) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        auto step = [&](int t, auto parity) {
            constexpr int Q = decltype(parity)::value;
            const char* const lr = smem + (t & (RING - 1)) * BUF;
            const char* const nr = smem + ((t + 1) & (RING - 1)) * BUF;
            const bool more = t + RING - 1 < steps;
#pragma unroll
            for (int i = 0; i < SL; ++i) {
                constexpr int PER_SLOT = 4;
                if (i * PER_SLOT < PIECES && more)
#pragma unroll
                    for (int j = 0; j < PER_SLOT; ++j) issue(t + RING - 1, i * PER_SLOT + j);
                if (i == SL - D) {
                    if (RING > 2 && more) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
                    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
                // (behind the last step what is read here is not used)
                const int n = (i + D) % SL;
                fr[(i + D) % (2 * D)] = TR::frag(i + D < SL ? lr : nr, wr + n % NA * 16, n / NA, l15, lg);
                // S: the fragments of the step's second half, of the next step's first
                if (SUBS == 2 && i >= NA - D && i < NA)
#pragma unroll
                    for (int b = 0; b < NB / D; ++b) {
                        const int c = (i - (NA - D)) * (NB / D) + b;
                        fs[1][c] = TS::frag(lr + TR::BYTES, wsx + c * 16, 1, l15, lg);
                    }
                if (i >= SL - D)
#pragma unroll
                    for (int b = 0; b < NB / D; ++b) {
                        const int c = (i - (SL - D)) * (NB / D) + b;
                        fs[SUBS == 2 ? 0 : Q ^ 1][c] = TS::frag(nr + TR::BYTES, wsx + c * 16, 0, l15, lg);
                    }
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[i % NA][b] = Mma<T>::run(fr[i % (2 * D)], fs[SUBS == 2 ? i / NA : Q][b], acc[i % NA][b]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (!some) {
            for (int t = 0; t < steps; ++t) idle(t);
        } else if constexpr (SUBS == 2) {
            for (int t = 0; t < steps; ++t) step(t, std::integral_constant<int, 0>());
        } else
            for (int t = 0; t < steps; t += 2) {
                step(t, std::integral_constant<int, 0>());
                if (t + 1 < steps) step(t + 1, std::integral_constant<int, 1>());
            }
    }
    // acc[a][b][j] = out[s = s0 + wsx + 16 b + l15][r = r0 + wr + 16 a + 4 lg + j]
    if constexpr (EPI == EPI_STATS || EPI == EPI_KEEP || EPI == EPI_PROB) {
        const bool edge = r0 + BR > g.nr;
        if (g.bias != nullptr || edge)
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = r0 + wr + a * 16 + lg * 4 + j;
                    const float bias = g.bias != nullptr && r < g.nr ? (float)((const T*)g.bias)[g.v0 + r] : 0.f;
#pragma unroll
                    for (int b = 0; b < NB; ++b) acc[a][b][j] = r < g.nr ? acc[a][b][j] + bias : -INFINITY;
                }
    }
    constexpr float LOG2E = 1.44269504088896340736f;
    // exp(z - ref): with bf16 operands in one multiply-add and one exp2 (ref log2(e) rounds once for the row, 2^-24 |ref| of every
    // term alike: far below what P is rounded by); with fp32 the difference first, which is exact near the largest terms
    // (and with references whose multiple could overflow: words masked by the lowest value)
    auto ex = [&](float z, float ref, float ref2, bool direct) {
        return __builtin_amdgcn_exp2f(direct ? __builtin_fmaf(z, LOG2E, -ref2) : (z - ref) * LOG2E);
    };
    auto direct = [&](float ref) { return sizeof(T) == 2 && __all(!(fabsf(ref) > 1e30f)); };
    if constexpr (EPI == EPI_STATS || EPI == EPI_KEEP) {
        __syncthreads();  // (the tiles have been read)
        float2* const join = (float2*)smem;  // [WR][BS]
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int s = s0 + wsx + b * 16 + l15;
            const long long label = s < ns ? g.labels[g.rows[s]] - g.v0 - r0 - wr : -1;
            float m, e = 0.f;
            if (__any(label >= 0 && label < BR / WR))  // (a wave in V / 128 has a row's label)
#pragma unroll
                for (int a = 0; a < NA; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (label == a * 16 + lg * 4 + j) g.zlab[s] = acc[a][b][j];
            // EPI_KEEP: exponentials relative to the row's own label, stored; their sum is the tile's.  A row whose label is 44 nats
            // or more behind some word (or no word, or not finite) has the pass over its logits made as if nothing were kept.
            if constexpr (EPI == EPI_KEEP) {
                m = s < ns ? g.ref[s] : 0.f;
                bool ok = __all(fabsf(m) <= 1e30f);
                if (ok) {
                    const float ref2 = m * LOG2E;
                    T* const row = (T*)g.P + (long long)s * g.ldp + r0 + wr;
#pragma unroll
                    for (int a = 0; a < NA; a += 2) {
                        f32x4 u, v;
#pragma unroll
                        for (int j = 0; j < 4; ++j) u[j] = ex(acc[a][b][j], m, ref2, sizeof(T) == 2);
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] = ex(acc[a + 1][b][j], m, ref2, sizeof(T) == 2);
                        e += ((u[0] + u[1]) + (u[2] + u[3])) + ((v[0] + v[1]) + (v[2] + v[3]));
                        if (s < ns) store_pair(row + a * 16, lg, u, v);
                    }
                    e += __shfl_xor(e, 16, 64);
                    e += __shfl_xor(e, 32, 64);
                    ok = __all(s >= ns || e < 0x1p64f);
                }
                if (ok) {
                    if (lg == 0) join[(wave % WR) * BS + wsx + b * 16 + l15] = make_float2(m, e);
                    continue;
                }
                if (lane == 0) __hip_atomic_store(g.gave_up, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                e = 0.f;
            }
            m = acc[0][b][0];
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) m = fmaxf(m, acc[a][b][j]);
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float ref = m == -INFINITY ? 0.f : m, ref2 = ref * LOG2E;
            if (direct(ref))
#pragma unroll
                for (int a = 0; a < NA; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) e += ex(acc[a][b][j], ref, ref2, true);
            else
#pragma unroll
                for (int a = 0; a < NA; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) e += ex(acc[a][b][j], ref, ref2, false);
            e += __shfl_xor(e, 16, 64);
            e += __shfl_xor(e, 32, 64);
            if (lg == 0) join[(wave % WR) * BS + wsx + b * 16 + l15] = make_float2(m, e);
        }
        __syncthreads();
        if (tid < BS && s0 + tid < ns) {
            float m = -INFINITY, e = 0.f;
#pragma unroll
            for (int w = 0; w < WR; ++w) m = fmaxf(m, join[w * BS + tid].x);
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int w = 0; w < WR; ++w) e += join[w * BS + tid].y * __builtin_amdgcn_exp2f((join[w * BS + tid].x - ref) * LOG2E);
            g.part[(long long)(s0 + tid) * g.part_ld + g.part0 + r0 / BR] = make_float2(m, e);
        }
    }
    if constexpr (EPI == EPI_PROB) {
        f32x4 cs[NA];
#pragma unroll
        for (int a = 0; a < NA; ++a) cs[a] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int s = s0 + wsx + b * 16 + l15;
            const bool in = s < ns;
            const int n = in ? g.rows[s] : 0;
            const long long label = in ? g.labels[n] - g.v0 - r0 - wr : -1;
            const float lse = in ? g.lse[n] : 0.f, lse2 = lse * LOG2E;
            if (direct(lse))
#pragma unroll
                for (int a = 0; a < NA; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[a][b][j] = ex(acc[a][b][j], lse, lse2, true);
            else
#pragma unroll
                for (int a = 0; a < NA; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[a][b][j] = ex(acc[a][b][j], lse, lse2, false);
            if (__any(label >= 0 && label < BR / WR))
#pragma unroll
                for (int a = 0; a < NA; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[a][b][j] -= label == a * 16 + lg * 4 + j ? 1.f : 0.f;
            if (g.scale != nullptr) {
                const float sc = in ? g.scale[n] : 0.f;
#pragma unroll
                for (int a = 0; a < NA; ++a) acc[a][b] *= sc;
            }
            if (s0 + BS > ns || r0 + BR > g.nr)  // behind the last row and the last word: 0, whatever lse is
#pragma unroll
                for (int a = 0; a < NA; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[a][b][j] = in && r0 + wr + a * 16 + lg * 4 + j < g.nr ? acc[a][b][j] : 0.f;
            T* const row = (T*)g.P + (long long)s * g.ldp + r0 + wr;
#pragma unroll
            for (int a = 0; a < NA; a += 2) {
                cs[a] += acc[a][b], cs[a + 1] += acc[a + 1][b];
                store_pair(row + a * 16, lg, acc[a][b], acc[a + 1][b]);
            }
        }
        if (g.dbpart != nullptr) {
            __syncthreads();
            float* const colsum = (float*)smem;  // [WS][BR]
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v = cs[a][j];
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
                    if (l15 == 0) colsum[(wave / WR) * BR + wr + a * 16 + lg * 4 + j] = v;
                }
            __syncthreads();
            if (tid < BR) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < WS; ++w) v += colsum[w * BR + tid];
                g.dbpart[(long long)st * g.ldp + r0 + tid] = v;
            }
        }
    }
    if constexpr (EPI == EPI_DX || EPI == EPI_DW) {
        const float f = EPI == EPI_DW ? g.factor.get() : 1.f;
        const bool wide = r0 + BR <= g.nr;  // (rows begin anywhere: the stores take any address)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int s = s0 + wsx + b * 16 + l15;
            if (s >= ns) continue;
            if (EPI == EPI_DW && wide) {
                T* const q = (T*)g.out + (long long)s * g.nr + r0 + wr;
#pragma unroll
                for (int a = 0; a < NA; a += 2) store_pair(q + a * 16, lg, acc[a][b] * f, acc[a + 1][b] * f);
                continue;
            }
#pragma unroll
            for (int a = 0; a < NA; ++a) {
                const int r = r0 + wr + a * 16 + lg * 4;
                if constexpr (EPI == EPI_DX) {
                    float* const q = g.acc + split * g.acc_split + (long long)s * g.nr + r;
                    if (r + 4 <= g.nr) {
                        f32x4 v = {0.f, 0.f, 0.f, 0.f};
                        if (g.add) __builtin_memcpy(&v, q, 16);
                        v += acc[a][b];
                        __builtin_memcpy(q, &v, 16);
                    } else
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (r + j < g.nr) q[j] = acc[a][b][j] + (g.add ? q[j] : 0.f);
                } else {
                    T* const q = (T*)g.out + (long long)s * g.nr + r;
                    const f32x4 v = acc[a][b] * f;
                    if (r + 4 <= g.nr) {
                        if constexpr (sizeof(T) == 2) {
                            const bf16x4 o = {f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])};
                            __builtin_memcpy(q, &o, 8);
                        } else
                            __builtin_memcpy(q, &v, 16);
                    } else
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (r + j < g.nr) q[j] = (T)v[j];
                }
            }
        }
    }
}

// a row of D elements to one of ld, zeros behind D; VEC: both begin at 16-byte chunks and D is whole ones
template <typename T, bool VEC>
__device__ __forceinline__ void copy_row(const T* from, T* to, int D, int ld, int i, int n) {
    if (VEC) {
        const int c = D * (int)sizeof(T) / 16;
        for (int d = i; d < ld * (int)sizeof(T) / 16; d += n) ((uint4*)to)[d] = d < c ? ((const uint4*)from)[d] : make_uint4(0, 0, 0, 0);
    } else
        for (int d = i; d < ld; d += n) to[d] = d < D ? from[d] : (T)0.f;
}
// words of w (a wave each), for the reasons that Plan gives
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void lce_words_of_w_kernel(const T* w, long long ldw, int n, int D, int ld, T* out, const int* when) {
    if (when != nullptr && *when == 0) return;
    for (int v = blockIdx.x * 4 + (threadIdx.x >> 6); v < n; v += gridDim.x * 4)
        copy_row<T, VEC>(w + v * ldw, out + (long long)v * ld, D, ld, threadIdx.x & 63, 64);
}
// the rows of x that count, one after the other (13 us of the 7 ms of 8192 x 2048 x 65536; the products then read x in order,
// with k across too, and never a row that does not count).  LIST: the list itself is made here too: every workgroup counts the
// labels before its row (up to 1024 rows: one launch instead of two; 2048 rows 9.2 us against 4.7 + 6.3, no shorter a step, 4096
// rows 17.6 against 5.7 + 8.6).  With ref: ref[i] = the logit of the row's label, or inf where
// that is no word or none that exponentials can be relative to.
struct LabelLogit {
    float* ref;  // nullable
    const void* w;
    long long ldw;
    const void* bias;
    int V;
    bool chunks;  // w's rows are whole 16-byte chunks
};
template <typename T, bool VEC, bool LIST>
__global__ __launch_bounds__(256) void lce_rows_of_x_kernel(const T* x, long long ldx, int* rows, const long long* labels, long long ignore,
                                                            int N, int D, int ld, T* out, LabelLogit q) {
    int i = blockIdx.x, n;
    if (LIST) {
        __shared__ int before_sh[4], all_sh[4];
        n = i;
        int before = 0, all = 0;
        for (int k = threadIdx.x; k < N; k += 256) {
            const int keep = labels[k] != ignore ? 1 : 0;
            all += keep;
            before += k < n ? keep : 0;
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) before += __shfl_xor(before, o, 64), all += __shfl_xor(all, o, 64);
        if ((threadIdx.x & 63) == 0) before_sh[threadIdx.x >> 6] = before, all_sh[threadIdx.x >> 6] = all;
        __syncthreads();
        before = before_sh[0] + before_sh[1] + before_sh[2] + before_sh[3];
        const bool keep = labels[n] != ignore;
        i = before;
        if (threadIdx.x == 0) {
            rows[keep ? before : N - 1 - (n - before)] = n;
            if (n == 0) rows[N] = all_sh[0] + all_sh[1] + all_sh[2] + all_sh[3], rows[N + 1] = 0, rows[N + 2] = 0;
        }
        if (!keep) return;
    } else {
        if (i >= rows[N]) return;
        n = rows[i];
    }
    copy_row<T, VEC>(x + n * ldx, out + (long long)i * ld, D, ld, threadIdx.x, 256);
    if (q.ref == nullptr) return;
    __shared__ float sum_sh[4];
    const long long y = labels[n];
    const bool word = y >= 0 && y < q.V;
    const T *const xr = x + n * ldx, *const wr = (const T*)q.w + (word ? y : 0) * q.ldw;
    float s = 0.f;
    constexpr int PER = 16 / (int)sizeof(T);
    typedef T chunk_t __attribute__((ext_vector_type(PER)));
    if (VEC && q.chunks)
        for (int d = threadIdx.x * PER; d < D; d += 256 * PER) {
            const chunk_t u = *(const chunk_t*)(xr + d), v = *(const chunk_t*)(wr + d);
#pragma unroll
            for (int j = 0; j < PER; ++j) s = __builtin_fmaf((float)u[j], (float)v[j], s);
        }
    else
        for (int d = threadIdx.x; d < D; d += 256) s = __builtin_fmaf((float)xr[d], (float)wr[d], s);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) sum_sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = (sum_sh[0] + sum_sh[1]) + (sum_sh[2] + sum_sh[3]) + (q.bias != nullptr && word ? (float)((const T*)q.bias)[y] : 0.f);
        q.ref[i] = word && fabsf(s) <= 1e30f ? s : INFINITY;
    }
}

// ---------------------------------------------------------------- the small launches around it
// A wave joins the pairs of one row: lse, loss.  With `loss` the workgroup that is done last sums the rows up, in their order.
// (It reads what the others wrote: their stores are device-scope atomics, complete before the workgroup counts itself done.)
// 16 rows a workgroup: workgroups count themselves on one word, 15 ns each (4 rows: 34 us for 8192 rows, 16: 14 us)
__global__ __launch_bounds__(1024) void lce_rows_kernel(const float2* part, int tiles, const float* zlab, const long long* labels,
                                                       int* rows, int N, int V, float* lse, float* loss_rows, float* plab, int mean, float* loss) {
    __shared__ double sums[16];
    __shared__ int last;
    const int wave = threadIdx.x >> 6, i = blockIdx.x * 16 + wave, lane = threadIdx.x & 63, count = rows[N];
    if (i < N) {
        const int n = rows[i];
        float m = -INFINITY, e = 0.f, l = 0.f, loss_n = 0.f;
        if (i < count) {
            for (int t0 = lane; t0 < tiles; t0 += 256) {  // (four pairs under way)
                float2 p[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = t0 + j * 64 < tiles ? part[(size_t)i * tiles + t0 + j * 64] : make_float2(-INFINITY, 0.f);
                float k = m;
#pragma unroll
                for (int j = 0; j < 4; ++j) k = fmaxf(k, p[j].x);
                const float ref = k == -INFINITY ? 0.f : k;
                e *= __expf(m - ref);
#pragma unroll
                for (int j = 0; j < 4; ++j) e += p[j].y * __expf(p[j].x - ref);
                m = k;
            }
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) {
                const float m2 = __shfl_xor(m, o, 64), e2 = __shfl_xor(e, o, 64);
                const float k = fmaxf(m, m2), ref = k == -INFINITY ? 0.f : k;
                e = e * __expf(m - ref) + e2 * __expf(m2 - ref);
                m = k;
            }
            const long long y = labels[n];
            const bool ok = y >= 0 && y < V;
            l = ok ? m + logf(e) : NAN;  // (a label that is no word: NaN, as with vc_softmax_ce)
            loss_n = ok ? l - zlab[i] : NAN;
            if (plab != nullptr && lane == 0) plab[i] = expm1f(-loss_n);  // P at the label: p - 1
        }
        if (lane == 0) {
            lse[n] = l;
            __hip_atomic_store(loss_rows + n, loss_n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (loss == nullptr) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(rows + N + 1, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    double s = 0.0;
    for (int n0 = threadIdx.x; n0 < N; n0 += 8192) {  // (eight loads under way)
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            v[k] = n0 + k * 1024 < N ? __hip_atomic_load(loss_rows + n0 + k * 1024, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += (double)v[k];
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 16; ++w) s += sums[w];
        loss[0] = (float)(mean ? s / (double)(count > 0 ? count : 1) : s);
    }
}
// What EPI_KEEP stored becomes P, where it lies: E[s][v] exp(ref_s - lse_s), at the label its own value; and db's partial sums.
// A workgroup takes a row tile by 64 chunks of 16 bytes, a wave a quarter of the rows.  P is rounded a second time, which is what
// not computing the logits again costs, and db sums values that are rounded once.  (bf16, error of dx against 64 bits, which its own
// rounding makes most of: P in fp32 / rounded once / twice 1.66e-3 / 1.67e-3 / 1.67e-3 for 2048 x 1024 of 32768, 1.65e-3 / 1.79e-3 /
// 1.81e-3 for 30 x 1024 of 1000.)
template <typename T>
__global__ __launch_bounds__(256) void lce_kept_kernel(T* E, long long lde, const int* rows, const float* lse, const float* ref, const float* plab,
                                                       const long long* labels, int N, int V, int tile, float* dbpart) {
    constexpr int PER = 16 / (int)sizeof(T);
    typedef T chunk_t __attribute__((ext_vector_type(PER)));
    __shared__ float by[256], at[256];
    __shared__ int label[256];
    __shared__ float sums[4][64][PER + 1];
    const int cols = (V + 64 * PER - 1) / (64 * PER), st = blockIdx.x / cols;
    const int count = rows[N], s0 = st * tile, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    if (s0 >= count || rows[N + 2] != 0) return;
    if (tid < tile) {
        const int s = s0 + tid;
        const bool in = s < count;
        const int n = in ? rows[s] : 0;
        by[tid] = in ? __expf(ref[s] - lse[n]) : 0.f;
        at[tid] = in ? plab[s] : 0.f;
        label[tid] = in ? (int)labels[n] : -PER;  // (a label that is no word: EPI_KEEP gave up)
    }
    __syncthreads();
    const int col0 = (blockIdx.x - st * cols) * 64 * PER, col = col0 + lane * PER;
    float cs[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) cs[j] = 0.f;
    if (col < V) {
        T* const from = E + (long long)s0 * lde + col;
        const int each = tile / 4;
        for (int k0 = wave * each; k0 < (wave + 1) * each; k0 += 8) {
            chunk_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = s0 + k0 + k < count ? *(const chunk_t*)(from + (k0 + k) * lde) : (chunk_t)(T)0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float c = by[k0 + k];
                const int l = label[k0 + k] - col;
                float f[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) f[j] = (float)v[k][j] * c;
                if (l >= 0 && l < PER) {
                    const float p = at[k0 + k];
#pragma unroll
                    for (int j = 0; j < PER; ++j) f[j] = j == l ? p : f[j];
                }
                chunk_t o;
#pragma unroll
                for (int j = 0; j < PER; ++j) cs[j] += f[j], o[j] = (T)f[j];
                *(chunk_t*)(from + (k0 + k) * lde) = o;
            }
        }
    }
    if (dbpart == nullptr) return;
#pragma unroll
    for (int j = 0; j < PER; ++j) sums[wave][lane][j] = cs[j];
    __syncthreads();
    for (int c = tid; c < 64 * PER; c += 256) {
        const int l = c / PER, j = c % PER;
        if (col0 + c < V) dbpart[(long long)st * lde + col0 + c] = (sums[0][l][j] + sums[1][l][j]) + (sums[2][l][j] + sums[3][l][j]);
    }
}
// what is stored last: workgroup i < N the row i of the list of dx (its splits' sums; zeros for a row that does not count), the
// others 256 words of db each (the sums of its row tiles)
struct Last {
    const float* acc;
    Splits splits;
    long long split;  // from split to split
    const float* part;
    long long ld;
    int bs, words, nx;  // nx: workgroups for dx, N or 0
    void *dx, *db;
};
template <typename T>
__global__ __launch_bounds__(256) void lce_last_kernel(const Last q, const int* rows, Factor factor, int N, int D) {
    const float g = factor.get();
    const int count = rows[N];
    if ((int)blockIdx.x >= q.nx) {
        const int r = (blockIdx.x - q.nx) * 256 + threadIdx.x;
        if (r >= q.words) return;
        const int tiles = (count + q.bs - 1) / q.bs;
        float s = 0.f;
        for (int t = 0; t < tiles; ++t) s += q.part[t * q.ld + r];
        ((T*)q.db)[r] = (T)(s * g);
        return;
    }
    const int i = blockIdx.x, n = rows[i], splits = q.splits.of(count);
    const bool keep = i < count;
    const float* const from = q.acc + (long long)i * D;
    T* const to = (T*)q.dx + (long long)n * D;
    for (int d0 = threadIdx.x * 4; d0 < D; d0 += 1024) {
        const int d = d0 + 4 > D && D >= 4 ? D - 4 : d0, left = D - d;  // (the last four once more, in part: the same values)
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (keep && left >= 4)
            for (int k0 = 0; k0 < splits; k0 += 8) {  // (eight sums under way)
                f32x4 t[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) __builtin_memcpy(&t[k], from + (k0 + k < splits ? k0 + k : splits - 1) * q.split + d, 16);
#pragma unroll
                for (int k = 0; k < 8; ++k) v += k0 + k < splits ? t[k] : (f32x4){0.f, 0.f, 0.f, 0.f};
            }
        else if (keep)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                for (int k = 0; k < splits && j < left; ++k) v[j] += from[k * q.split + d + j];
        v *= g;
        if (!keep) v = (f32x4){0.f, 0.f, 0.f, 0.f};  // (g may be no number)
        if (left >= 4) {
            if constexpr (sizeof(T) == 2) {
                const bf16x4 o = {f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])};
                __builtin_memcpy(to + d, &o, 8);
            } else
                __builtin_memcpy(to + d, &v, 16);
        } else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < left) to[d + j] = (T)v[j];
    }
}

// ---------------------------------------------------------------- plan and workspace
// side of the tiles of an ns x nr product: the largest that makes work for most of the 256 CUs (96, 192 and 384 tiles as the
// border measured alike within 2 %; 256 against 128 wide tiles where both fill the chip: 0.88 x the time)
int pick_tile(long long ns, long long nr) {
    for (int b = 256; b > 64; b /= 2)
        if (ns > b / 2 && nr > b / 2 && ((ns + b - 1) / b) * ((nr + b - 1) / b) >= 192) return b;
    return 64;
}

struct Plan {
    size_t bytes = 0;
    int tile, tile_dx, tile_dw;  // sides of the tiles of N x V, N x D, piece x D
    int piece;                   // words of a piece, a multiple of 256
    int tiles;                   // tiles of the vocabulary
    Splits dx;
    int kd;                      // features, in whole 16-byte chunks
    int ld;                      // row length of copies of x, w: whole 128-byte lines
    size_t acc, P, dbpart, part, zlab, loss_rows, xp, wp;
    long long lde;               // row length of what EPI_KEEP stores
    size_t take(size_t n) {
        const size_t at = bytes;
        bytes += (n + 255) & ~(size_t)255;
        return at;
    }
    // row length of a copy: whole 128-byte lines; whether the copy of x is kept for the backward (up to 32 MB)
    static int row(int D, int elem) { return (D * elem + 127) / 128 * 128 / elem; }
    static bool saves_x(int N, int D, int elem) { return (long long)N * row(D, elem) * elem <= (32 << 20); }
    // what the forward leaves for the backward: lse [N], the list [N + 4], the copy of x
    static size_t list_at(int N) { return ((size_t)N * 4 + 255) & ~(size_t)255; }
    static size_t x_at(int N) { return list_at(N) + ((((size_t)N + 4) * 4 + 255) & ~(size_t)255); }
    static size_t ref_at(int N, int D, int elem) { return x_at(N) + (((saves_x(N, D, elem) ? (size_t)N * row(D, elem) * elem : 0) + 255) & ~(size_t)255); }
    // with `keep` also: ref [N], P at the label [N], the exponentials, which become P, and db's partial sums; with 2 the copy of w
    static size_t plab_at(int N, int D, int elem) { return ref_at(N, D, elem) + list_at(N); }
    static size_t exps_at(int N, int D, int elem) { return plab_at(N, D, elem) + list_at(N); }
    static size_t row_tiles(int N, int V) { return ((size_t)N + pick_tile(N, V) - 1) / pick_tile(N, V); }
    static size_t exps(int N, int V, int elem) { return row_tiles(N, V) * pick_tile(N, V) * (((size_t)V + 255) / 256 * 256) * elem; }
    static size_t dbpart_at(int N, int D, int V, int elem) { return exps_at(N, D, elem) + exps(N, V, elem); }
    static size_t w_at(int N, int D, int V, int elem) { return dbpart_at(N, D, V, elem) + row_tiles(N, V) * (((size_t)V + 255) / 256 * 256) * 4; }
    static size_t saved(int N, int D, int V, int elem, int keep) {
        return keep ? w_at(N, D, V, elem) + (keep == 2 ? (size_t)V * row(D, elem) * elem : 0) : ref_at(N, D, elem);
    }
    Plan(int N, int D, int V, int elem, int op, bool pack, int keep) {
        kd = (D * elem + 15) / 16 * 16 / elem;
        ld = row(D, elem);
        const long long np = ((long long)N + 255) / 256 * 256, all = ((long long)V + 255) / 256 * 256;
        long long fit = (512ll << 20) / elem / np / 256 * 256;
        if (op == 0 || keep) fit = pack && keep < 2 ? (512ll << 20) / elem / ld / 256 * 256 : all;  // (a piece of w's copy is all there is)
        if (op == 0 || keep) {  // a launch has fewer than 2^32 lanes (HIP's limit), 512 for a tile of 256 x 256
            const long long most = ((1ll << 23) - 1) / (np / 256) * 256;
            fit = fit < most ? fit : most;
        }
        fit = fit < 256 ? 256 : fit;
        lde = all;
        piece = (int)(fit < all ? fit : all);
        tile = pick_tile(N, piece < V && !keep ? piece : V);
        tiles = (int)(((long long)V + tile - 1) / tile);
        if (!saves_x(N, D, elem)) xp = take((size_t)N * ld * elem);
        if (pack && keep < 2) wp = take((size_t)(piece < V ? piece : V) * ld * elem);
        if (op == 0) {
            part = take((size_t)N * tiles * sizeof(float2));
            zlab = take((size_t)N * 4);
            loss_rows = take((size_t)N * 4);
            return;
        }
        // dx: smaller tiles need fewer splits of k, i.e. fewer sums to write and join (500 x 256 of 100000 words, 2 tiles of 256:
        // 338 us with 256, 275 with 128; 1600 x 1000 of 50257, 28 tiles: 794 against 845; 8192 x 2048 of 65536: 6.96 against 7.73 ms)
        tile_dx = N > 128 && D > 128 && (N + 255ll) / 256 * ((D + 255) / 256) >= 16 ? 256 : N > 64 && D > 64 ? 128 : 64;
        tile_dw = pick_tile(piece < V ? piece : V, D);
        // up to 64 splits (16: the product of 224 rows x 768 of 75745 words 57 us instead of 30), 256 MB of sums, 128 words a split
        // (512: the kernels of a step of 64 x 512 of 400 classes 57.7 us instead of 51.3)
        dx = {tile_dx == 256 ? 256 : 512, 64, (D + tile_dx - 1) / tile_dx, tile_dx};
        const long long room = (256ll << 20) / ((long long)N * D * 4), least = piece / 128;
        dx.most = (int)(dx.most > room ? room : dx.most);
        dx.most = (int)(dx.most > least ? least : dx.most);
        dx.most = dx.most < 1 ? 1 : dx.most;
        acc = take((size_t)dx.most * N * D * 4);
        if (keep) return;
        P = take((size_t)np * piece * elem);
        dbpart = take((size_t)(np / 64) * piece * 4);
    }
};

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        vc_set_error("%s launch failed: %s", what, hipGetErrorString(e));
        return -1;
    }
    return 0;
}

template <typename T, int EPI, int B>
void gemm_tile(const Gemm& g, int tiles, int splits, hipStream_t s) {
    constexpr int WR = 2, WS = B == 256 ? 4 : 2, LDS = Feed<EPI, B>::RING * Feed<EPI, B>::SUBS * 2 * B * 64;
    const auto kernel = lce_gemm<T, EPI, B, B, WR, WS>;
    static VcPerDeviceOnce once;
    once.run([&] { (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS); });
    hipLaunchKernelGGL((lce_gemm<T, EPI, B, B, WR, WS>), dim3(tiles * splits), dim3(WR * WS * 64), LDS, s, g);
}
template <typename T, int EPI>
void gemm(Gemm& g, int tile, int ns_most, int splits, hipStream_t s) {
    g.rtiles = (g.nr + tile - 1) / tile;
    const int tiles = g.rtiles * ((ns_most + tile - 1) / tile);
    if (tile == 256) gemm_tile<T, EPI, 256>(g, tiles, splits, s);
    else if (tile == 128) gemm_tile<T, EPI, 128>(g, tiles, splits, s);
    else gemm_tile<T, EPI, 64>(g, tiles, splits, s);
}

// x as the products read it, and w from word v0 on
template <typename T>
struct Source {
    const VcLceParams& p;
    const Plan& L;
    hipStream_t s;
    Operand x;
    static bool chunks(const void* q, long long ld, int D) { return (((uintptr_t)q | (uintptr_t)(ld * sizeof(T)) | (uintptr_t)(D * sizeof(T))) & 15) == 0; }
    float *lse, *ref, *plab;
    int* rows;
    T* exps;
    float* dbpart;
    T* kept_w;
    bool forward;
    Source(const VcLceParams& p, const Plan& L, hipStream_t s, bool forward) : p(p), L(L), s(s), forward(forward) {
        char* const saved = (char*)p.saved;
        const bool kept = Plan::saves_x(p.N, p.D, sizeof(T));
        lse = (float*)saved, rows = (int*)(saved + Plan::list_at(p.N));
        ref = p.keep ? (float*)(saved + Plan::ref_at(p.N, p.D, sizeof(T))) : nullptr;
        plab = p.keep ? (float*)(saved + Plan::plab_at(p.N, p.D, sizeof(T))) : nullptr;
        exps = p.keep ? (T*)(saved + Plan::exps_at(p.N, p.D, sizeof(T))) : nullptr;
        dbpart = p.keep && p.bias != nullptr ? (float*)(saved + Plan::dbpart_at(p.N, p.D, p.V, sizeof(T))) : nullptr;
        kept_w = p.keep == 2 ? (T*)(saved + Plan::w_at(p.N, p.D, p.V, sizeof(T))) : nullptr;
        T* const to = (T*)(kept ? saved + Plan::x_at(p.N) : (char*)p.ws + L.xp);
        x = {(const char*)to, L.ld * (long long)sizeof(T)};
        if (!forward && kept) return;
        const bool list = forward && p.N <= 1024, vec = chunks(p.x, p.ldx, p.D);
        if (forward && !list) hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(1024), 0, s, p.labels, p.ignore_index, p.N, rows);
        const auto kernel = list ? (vec ? lce_rows_of_x_kernel<T, true, true> : lce_rows_of_x_kernel<T, false, true>)
                                 : (vec ? lce_rows_of_x_kernel<T, true, false> : lce_rows_of_x_kernel<T, false, false>);
        const LabelLogit q = {forward ? ref : nullptr, p.w, p.ldw, p.bias, p.V, !p.pack};
        hipLaunchKernelGGL(kernel, dim3(p.N), dim3(256), 0, s, (const T*)p.x, p.ldx, rows, p.labels, p.ignore_index, p.N, p.D, L.ld, to, q);
    }
    Operand w(int v0, int nv, const int* when) const {
        const T* at = (const T*)p.w + v0 * p.ldw;
        if (!p.pack) return {(const char*)at, p.ldw * (long long)sizeof(T)};
        T* const to = kept_w != nullptr ? kept_w + (long long)v0 * L.ld : (T*)((char*)p.ws + L.wp);
        if (kept_w != nullptr && !forward) return {(const char*)to, L.ld * (long long)sizeof(T)};
        const auto kernel = chunks(at, p.ldw, p.D) ? lce_words_of_w_kernel<T, true> : lce_words_of_w_kernel<T, false>;
        hipLaunchKernelGGL(kernel, dim3(nv < 16384 ? (nv + 3) / 4 : 4096), dim3(256), 0, s, at, p.ldw, nv, p.D, L.ld, to, when);
        return {(const char*)to, L.ld * (long long)sizeof(T)};
    }
};

template <typename T>
int fwd(const VcLceParams& p, hipStream_t s) {
    const Plan L(p.N, p.D, p.V, sizeof(T), 0, p.pack, p.keep);
    char* ws = (char*)p.ws;
    float2* part = (float2*)(ws + L.part);
    float* zlab = (float*)(ws + L.zlab);
    float* loss_rows = p.loss_rows != nullptr ? p.loss_rows : (float*)(ws + L.loss_rows);
    (void)hipGetLastError();
    const Source<T> src(p, L, s, true);
    int* const gave_up = src.rows + p.N + 2;
    Gemm g = {};
    g.ns_dev = src.rows + p.N, g.K = L.kd, g.S = src.x, g.bias = p.bias, g.labels = p.labels, g.rows = src.rows;
    g.part = part, g.part_ld = L.tiles, g.zlab = zlab, g.ref = src.ref, g.gave_up = gave_up, g.ldp = L.lde;
    for (int v0 = 0; v0 < p.V; v0 += L.piece) {
        g.nr = p.V - v0 < L.piece ? p.V - v0 : L.piece, g.R = src.w(v0, g.nr, nullptr);
        g.v0 = v0, g.part0 = v0 / L.tile;
        if (p.keep) g.P = src.exps + v0, gemm<T, EPI_KEEP>(g, L.tile, p.N, 1, s);
        else gemm<T, EPI_STATS>(g, L.tile, p.N, 1, s);
    }
    hipLaunchKernelGGL(lce_rows_kernel, dim3((p.N + 15) / 16), dim3(1024), 0, s, part, L.tiles, zlab, p.labels, src.rows, p.N, p.V, src.lse,
                       loss_rows, src.plab, p.reduction == 1, p.reduction != 0 ? p.loss : nullptr);
    if (p.keep) {
        hipLaunchKernelGGL((lce_kept_kernel<T>), dim3((p.V + 1024 / (int)sizeof(T) - 1) / (1024 / (int)sizeof(T)) * ((p.N + L.tile - 1) / L.tile)),
                           dim3(256), 0, s, src.exps, L.lde, src.rows, src.lse, src.ref, src.plab, p.labels, p.N, p.V, L.tile, src.dbpart);
        // where EPI_KEEP gave up (4.7 us of workgroups that leave at once where it did not)
        g.when = gave_up, g.lse = src.lse;
        for (int v0 = 0; v0 < p.V; v0 += L.piece) {
            g.nr = p.V - v0 < L.piece ? p.V - v0 : L.piece;
            if (L.piece < p.V) g.R = src.w(v0, g.nr, gave_up);
            g.v0 = v0, g.P = src.exps + v0, g.dbpart = src.dbpart != nullptr ? src.dbpart + v0 : nullptr;
            gemm<T, EPI_PROB>(g, L.tile, p.N, 1, s);
        }
    }
    return launched("linear_ce_fwd");
}

template <typename T>
int bwd(const VcLceParams& p, hipStream_t s) {
    const Plan L(p.N, p.D, p.V, sizeof(T), 1, p.pack, p.keep);
    char* ws = (char*)p.ws;
    float *acc = (float*)(ws + L.acc), *dbpart = p.keep ? nullptr : (float*)(ws + L.dbpart);
    const long long ld = p.keep ? L.lde : L.piece;
    (void)hipGetLastError();
    const Source<T> src(p, L, s, false);
    const int* count = src.rows + p.N;
    const Factor factor = {p.dloss, count, p.reduction};
    for (int v0 = 0; v0 < p.V; v0 += L.piece) {
        const int nv = p.V - v0 < L.piece ? p.V - v0 : L.piece;
        const bool wants_w = !p.keep || p.dx != nullptr;
        const Operand w = wants_w ? src.w(v0, nv, nullptr) : Operand{};
        T* const P = p.keep ? src.exps + v0 : (T*)(ws + L.P);
        if (p.keep) dbpart = src.dbpart != nullptr ? src.dbpart + v0 : nullptr;
        else {
            Gemm g = {};
            g.R = w, g.S = src.x;
            g.nr = nv, g.ns_dev = count, g.K = L.kd;
            g.bias = p.bias, g.labels = p.labels, g.rows = src.rows, g.v0 = v0;
            g.lse = src.lse, g.scale = p.reduction == 0 ? p.dloss : nullptr, g.P = P, g.ldp = ld, g.dbpart = p.db != nullptr ? dbpart : nullptr;
            gemm<T, EPI_PROB>(g, L.tile, p.N, 1, s);
        }
        if (p.dx != nullptr) {
            Gemm x = {};
            x.R = w, x.S = {(const char*)P, ld * (long long)sizeof(T)};
            x.nr = p.D, x.ns_dev = count, x.K = nv, x.acc = acc, x.add = v0 > 0, x.acc_split = (long long)p.N * p.D;
            x.splits = L.dx;
            gemm<T, EPI_DX>(x, L.tile_dx, p.N, L.dx.most, s);
        }
        if (p.dw != nullptr) {
            Gemm d = {};
            d.R = src.x, d.S = {(const char*)P, ld * (long long)sizeof(T)};
            d.nr = p.D, d.ns = nv, d.k_dev = count, d.out = (T*)p.dw + (long long)v0 * p.D, d.factor = factor;
            gemm<T, EPI_DW>(d, L.tile_dw, nv, 1, s);
        }
        const bool end = v0 + nv == p.V && p.dx != nullptr;
        if (p.db == nullptr && !end) continue;
        const Last q = {acc, L.dx, (long long)p.N * p.D, dbpart, ld, L.tile, nv, end ? p.N : 0, p.dx, p.db != nullptr ? (T*)p.db + v0 : nullptr};
        hipLaunchKernelGGL((lce_last_kernel<T>), dim3(q.nx + (p.db != nullptr ? (nv + 255) / 256 : 0)), dim3(256), 0, s, q, src.rows, factor, p.N, p.D);
    }
    return launched("linear_ce_bwd");
}

}  // namespace

// Whether the products read a copy of w: where its rows are no whole 16-byte chunks or begin at none (or lie 4 GB apart).
// (Rows that begin inside 128-byte lines are read as they are: copies cost more than they give, also where the forward's is kept for
// the backward.  Kernels of a step, as they are / copied: 1777 x 1000 of 50257 519 / 534 us, 1600 x 1000 of 50257 656 / 657, 4000 x
// 360 of 32000 515 / 520; without anything kept 636 / 677, 757 / 803, 538 / 550.)  w_align: the address of w, modulo 16.
bool vc_lce_pack(int D, long long ldw, int w_align, bool is_bf16) {
    const int elem = is_bf16 ? 2 : 4;
    return (D * elem) % 16 != 0 || (ldw * elem) % 16 != 0 || w_align != 0 || ldw * elem >= (1ll << 32);
}
// Whether the forward keeps the logits' gradient for the backward, which then need not compute the logits again: that saves a
// product and costs storing, reading and storing N x V, and two launches.  By itself up to 2 GB (under 1 % of the memory) and
// where there is enough to save: a long sum, a large product, or a large w that few rows would read again.  Kernels of a step,
// again / kept in us, bf16: 2048 x 1024 of 32768 555 / 477, 8192 x 2048 of 65536 7170 / 5900, 4000 x 384 of 32000 553 / 535, 8192 x
// 256 of 60000 1660 / 1470, 512 x 512 of 8192 80 / 74, 30 x 1024 of 1000 45.3 / 43.8, 1 x 2048 of 32000 125 / 110; but 8192 x 128
// of 60000 1200 / 1332, 200 x 512 of 8000 59.6 / 61.7.  fp32: 1000 x 1024 of 32000 2030 / 1590, 1000 x 64 of 20000 214 / 190, 64 x
// 512 of 400 61 / 52; but 300 x 128 of 10000 121.5 / 122.4.  Few rows: bf16 16 x 256 of 130000 108 / 92, 100 x 128 of 130000
// 115 / 108, fp32 6 x 415 of 85803 362 / 316; but 16 x 512 of 8000 46.3 / 46.2.
// 2: and the copy of w, where the products read one and there is room.
int vc_lce_keep(int N, int D, int V, bool is_bf16, bool pack, int reduction, long long keep_bytes) {
    if (reduction == 0) return 0;  // (its rows' factors come with the backward)
    const int elem = is_bf16 ? 2 : 4;
    const size_t bytes = Plan::exps(N, V, elem), limit = keep_bytes >= 0 ? (size_t)keep_bytes : (size_t)2 << 30;
    const double work = (double)N * V * D;
    const bool pays = (N <= D && (double)D * V >= 0x1p23) || (is_bf16 ? D >= 1024 || (D >= 256 && work >= 0x1p31) : D >= 512 || work >= 0x1p29);
    if (bytes > limit || (keep_bytes < 0 && !pays)) return 0;
    return pack && bytes + (size_t)V * Plan::row(D, elem) * elem <= limit ? 2 : 1;
}
size_t vc_lce_saved(int N, int D, int V, bool is_bf16, int keep) { return Plan::saved(N, D, V, is_bf16 ? 2 : 4, keep); }
size_t vc_lce_workspace(int N, int D, int V, bool is_bf16, bool pack, int keep, int op) { return Plan(N, D, V, is_bf16 ? 2 : 4, op, pack, keep).bytes; }
int vc_lce_launch_fwd(const VcLceParams& p, bool is_bf16, hipStream_t s) { return is_bf16 ? fwd<bf16>(p, s) : fwd<float>(p, s); }
int vc_lce_launch_bwd(const VcLceParams& p, bool is_bf16, hipStream_t s) { return is_bf16 ? bwd<bf16>(p, s) : bwd<float>(p, s); }
