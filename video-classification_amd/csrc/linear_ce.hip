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
// round by the same amount in all of them, an error that adds up (measured: 3.5e-3 of dw instead of 2.3e-3 with bf16).  N x V is never held: the forward keeps N floats, the backward one N x piece block.
//
// Rows whose label is ignore_index take no part: the rows that count are listed first (rows_kernel) and all products run
// over that list, so that an ignored row costs nothing and whatever it holds (NaN included) reaches nothing.
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
    if (tid == 0) rows[N] = base;
}

// ---------------------------------------------------------------- matrix product, any sizes and strides
// out[s][r] = sum_k S(s, k) R(r, k), 128 x 128 per workgroup of four waves (64 x 64 each).  An operand is addressed by row
// and k strides (one of them is 1) and optional gather lists of its rows or its k.
struct Operand {
    const void* p;
    long long row, k;  // strides in elements
    const int* rows;   // nullable: row i is at rows[i]
    const int* ks;     // nullable: k is at ks[k]
};

enum { EPI_STATS, EPI_PROB, EPI_DX, EPI_DW };

struct Gemm {
    Operand R, S;
    int nr, ns, K;
    const int* ns_dev;  // nullable: ns is *ns_dev
    const int* k_dev;   // nullable: K is *k_dev
    // EPI_STATS / EPI_PROB: r = word v0 + r, s = listed row
    const void* bias;
    const long long* labels;
    const int* rows;
    int v0;
    float2* part;  // [s][tiles]
    int tiles;
    float* zlab;   // [s]: logit of the row's label
    const float* lse;
    const float* scale;  // nullable: [N], each row's own factor
    void* P;
    long long ldp;
    float* dbpart;  // [s tiles][nr]
    float* acc;     // EPI_DX: [s][nr]
    int add;
    void* out;       // EPI_DW: [s][nr]
    const float* g;  // EPI_DW: the factor common to all rows
};

template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    static constexpr int KSTEP = 32, PER = 8;  // k of an instruction, of a lane
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<float> {
    static constexpr int KSTEP = 16, PER = 4;  // four instructions of k = 4; k is dealt to the lanes in fours, alike for both operands
    typedef f32x4 frag;
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

template <typename T>
__device__ __forceinline__ T fetch(const Operand& o, int row, int nrows, int k, int K) {
    if (row >= nrows || k >= K) return (T)0.f;
    const long long i = o.rows != nullptr ? o.rows[row] : row, j = o.ks != nullptr ? o.ks[k] : k;
    return ((const T*)o.p)[i * o.row + j * o.k];
}

template <typename T, int EPI>
__global__ __launch_bounds__(256) void lce_gemm_any(const Gemm g) {
    constexpr int BK = Mma<T>::KSTEP, PITCH = BK + Mma<T>::PER;
    __shared__ __attribute__((aligned(16))) T sR[128][PITCH], sS[128][PITCH];
    const int ns = g.ns_dev != nullptr ? *g.ns_dev : g.ns, K = g.k_dev != nullptr ? *g.k_dev : g.K;
    const int r0 = blockIdx.x * 128, s0 = blockIdx.y * 128;
    if (s0 >= ns) return;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l15 = lane & 15, lg = lane >> 4;
    const int wr = (wave & 1) * 64, wsx = (wave >> 1) * 64;
    f32x4 acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < K; k0 += BK) {
        // neighbouring threads take neighbouring addresses: along k where k is contiguous, along the rows otherwise
        for (int i = tid; i < 128 * BK; i += 256) {
            const int rr = g.R.k == 1 ? i / BK : i % 128, rk = g.R.k == 1 ? i % BK : i / 128;
            sR[rr][rk] = fetch<T>(g.R, r0 + rr, g.nr, k0 + rk, K);
            const int sr = g.S.k == 1 ? i / BK : i % 128, sk = g.S.k == 1 ? i % BK : i / 128;
            sS[sr][sk] = fetch<T>(g.S, s0 + sr, ns, k0 + sk, K);
        }
        __syncthreads();
        typename Mma<T>::frag fs[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) fs[b] = *(const typename Mma<T>::frag*)&sS[wsx + b * 16 + l15][lg * Mma<T>::PER];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const typename Mma<T>::frag fr = *(const typename Mma<T>::frag*)&sR[wr + a * 16 + l15][lg * Mma<T>::PER];
#pragma unroll
            for (int b = 0; b < 4; ++b) acc[a][b] = Mma<T>::run(fr, fs[b], acc[a][b]);
        }
        __syncthreads();
    }
    // acc[a][b][j] = out[s = s0 + wsx + 16 b + l15][r = r0 + wr + 16 a + 4 lg + j]
    if (EPI == EPI_STATS || EPI == EPI_PROB) {
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = r0 + wr + a * 16 + lg * 4 + j;
                const float bias = g.bias != nullptr && r < g.nr ? (float)((const T*)g.bias)[g.v0 + r] : 0.f;
#pragma unroll
                for (int b = 0; b < 4; ++b) acc[a][b][j] = r < g.nr ? acc[a][b][j] + bias : -INFINITY;
            }
    }
    if (EPI == EPI_STATS) {
        __shared__ float2 join[2][128];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int s = s0 + wsx + b * 16 + l15;
            const long long label = s < ns ? g.labels[g.rows[s]] - g.v0 : -1;
            float m = -INFINITY, e = 0.f;
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m = fmaxf(m, acc[a][b][j]);
                    if (r0 + wr + a * 16 + lg * 4 + j == label && label < g.nr) g.zlab[s] = acc[a][b][j];
                }
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) e += __expf(acc[a][b][j] - ref);
            e += __shfl_xor(e, 16, 64);
            e += __shfl_xor(e, 32, 64);
            if (lg == 0) join[wave & 1][wsx + b * 16 + l15] = make_float2(m, e);
        }
        __syncthreads();
        if (tid < 128 && s0 + tid < ns) {
            const float2 p = join[0][tid], q = join[1][tid];
            const float m = fmaxf(p.x, q.x), ref = m == -INFINITY ? 0.f : m;
            g.part[(size_t)(s0 + tid) * g.tiles + blockIdx.x] = make_float2(m, p.y * __expf(p.x - ref) + q.y * __expf(q.x - ref));
        }
        return;
    }
    if (EPI == EPI_PROB) {
        __shared__ float colsum[2][128];
        f32x4 cs[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) cs[a] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int s = s0 + wsx + b * 16 + l15;
            if (s < ns) {
                const int n = g.rows[s];
                const long long label = g.labels[n] - g.v0;
                const float lse = g.lse[n], sc = g.scale != nullptr ? g.scale[n] : 1.f;
#pragma unroll
                for (int a = 0; a < 4; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = r0 + wr + a * 16 + lg * 4 + j;
                        const float v = (__expf(acc[a][b][j] - lse) - (r == label ? 1.f : 0.f)) * sc;
                        if (r < g.nr) {
                            cs[a][j] += v;
                            ((T*)g.P)[(size_t)s * g.ldp + r] = (T)v;
                        }
                    }
            }
        }
        if (g.dbpart != nullptr) {
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v = cs[a][j];
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
                    if (l15 == 0) colsum[wave >> 1][wr + a * 16 + lg * 4 + j] = v;
                }
            __syncthreads();
            if (tid < 128 && r0 + tid < g.nr) g.dbpart[(size_t)blockIdx.y * g.nr + r0 + tid] = colsum[0][tid] + colsum[1][tid];
        }
        return;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int s = s0 + wsx + b * 16 + l15;
        if (s >= ns) continue;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = r0 + wr + a * 16 + lg * 4 + j;
                if (r >= g.nr) continue;
                if (EPI == EPI_DX) {
                    float* q = g.acc + (size_t)s * g.nr + r;
                    *q = acc[a][b][j] + (g.add ? *q : 0.f);
                } else
                    ((T*)g.out)[(size_t)s * g.nr + r] = (T)(acc[a][b][j] * *g.g);
            }
    }
}

// ---------------------------------------------------------------- the small launches around it
// a wave joins the pairs of one row: lse, loss
__global__ __launch_bounds__(256) void lce_rows_kernel(const float2* part, int tiles, const float* zlab, const long long* labels,
                                                       const int* rows, int N, int V, float* lse, float* loss_rows) {
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (i >= N) return;
    const int n = rows[i];
    if (i >= rows[N]) {  // does not count
        if (lane == 0) lse[n] = 0.f, loss_rows[n] = 0.f;
        return;
    }
    float m = -INFINITY, e = 0.f;
    for (int t = lane; t < tiles; t += 64) {
        const float2 p = part[(size_t)i * tiles + t];
        const float k = fmaxf(m, p.x), ref = k == -INFINITY ? 0.f : k;
        e = e * __expf(m - ref) + p.y * __expf(p.x - ref);
        m = k;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float m2 = __shfl_xor(m, o, 64), e2 = __shfl_xor(e, o, 64);
        const float k = fmaxf(m, m2), ref = k == -INFINITY ? 0.f : k;
        e = e * __expf(m - ref) + e2 * __expf(m2 - ref);
        m = k;
    }
    if (lane == 0) {
        const long long y = labels[n];
        const bool ok = y >= 0 && y < V;
        const float l = ok ? m + logf(e) : NAN;  // (a label that is no word: NaN, as with vc_softmax_ce)
        lse[n] = l;
        loss_rows[n] = ok ? l - zlab[i] : NAN;
    }
}
__global__ __launch_bounds__(1024) void lce_mean_kernel(const float* loss_rows, const int* rows, int N, int mean, float* loss) {
    __shared__ double part[16];
    double s = 0.0;
    for (int n = threadIdx.x; n < N; n += 1024) s += (double)loss_rows[n];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 16; ++w) s += part[w];
        const int count = rows[N];
        loss[0] = (float)(mean ? s / (double)(count > 0 ? count : 1) : s);
    }
}
// the factor common to all rows
__global__ void lce_factor_kernel(const float* dloss, const int* rows, int N, int reduction, float* g) {
    const int count = rows[N];
    g[0] = reduction == 0 ? 1.f : reduction == 1 ? dloss[0] / (float)(count > 0 ? count : 1) : dloss[0];
}
// dx of the rows that count from their sums, zeros for the others
template <typename T>
__global__ __launch_bounds__(256) void lce_dx_kernel(const float* acc, const int* rows, const float* g, int N, int D, T* dx) {
    const int i = blockIdx.x, n = rows[i];
    const bool keep = i < rows[N];
    for (int d = threadIdx.x; d < D; d += 256) dx[(size_t)n * D + d] = keep ? (T)(acc[(size_t)i * D + d] * *g) : (T)0.f;
}
template <typename T>
__global__ __launch_bounds__(256) void lce_db_kernel(const float* part, const int* count, const float* g, int nr, T* db) {
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (r >= nr) return;
    const int tiles = (*count + 127) / 128;
    float s = 0.f;
    for (int t = 0; t < tiles; ++t) s += part[(size_t)t * nr + r];
    db[r] = (T)(s * *g);
}

// ---------------------------------------------------------------- workspace
struct Layout {
    size_t bytes = 0;
    size_t take(size_t n) {
        const size_t at = bytes;
        bytes += (n + 255) & ~(size_t)255;
        return at;
    }
};
struct FwdLayout : Layout {
    size_t part, zlab, loss_rows;
    int tiles;
    FwdLayout(int N, int V) {
        tiles = (V + 127) / 128;
        part = take((size_t)N * tiles * sizeof(float2));
        zlab = take((size_t)N * 4);
        loss_rows = take((size_t)N * 4);
    }
};
struct BwdLayout : Layout {
    size_t g, acc, P, dbpart;
    int piece;
    BwdLayout(int N, int D, int V, int elem) {
        // a piece's P takes up to 256 MB (what stays near the chip between its writer and its two readers), in whole tiles
        const long long fit = (256ll << 20) / elem / N / 128 * 128;
        const long long all = (V + 127ll) / 128 * 128;
        piece = (int)(fit < 128 ? 128 : fit < all ? fit : all);
        g = take(4);
        acc = take((size_t)N * D * 4);
        P = take((size_t)N * piece * elem);
        dbpart = take((size_t)((N + 127) / 128) * piece * 4);
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

template <typename T>
int fwd(const VcLceParams& p, hipStream_t s) {
    const FwdLayout L(p.N, p.V);
    char* ws = (char*)p.ws;
    float2* part = (float2*)(ws + L.part);
    float* zlab = (float*)(ws + L.zlab);
    float* loss_rows = p.loss_rows != nullptr ? p.loss_rows : (float*)(ws + L.loss_rows);
    (void)hipGetLastError();
    hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(1024), 0, s, p.labels, p.ignore_index, p.N, p.rows);
    Gemm g = {};
    g.R = {p.w, p.ldw, 1, nullptr, nullptr};
    g.S = {p.x, p.ldx, 1, p.rows, nullptr};
    g.nr = p.V, g.ns_dev = p.rows + p.N, g.K = p.D;
    g.bias = p.bias, g.labels = p.labels, g.rows = p.rows, g.part = part, g.tiles = L.tiles, g.zlab = zlab;
    hipLaunchKernelGGL((lce_gemm_any<T, EPI_STATS>), dim3(L.tiles, (p.N + 127) / 128), dim3(256), 0, s, g);
    hipLaunchKernelGGL(lce_rows_kernel, dim3((p.N + 3) / 4), dim3(256), 0, s, part, L.tiles, zlab, p.labels, p.rows, p.N, p.V, p.lse,
                       loss_rows);
    if (p.reduction != 0)
        hipLaunchKernelGGL(lce_mean_kernel, dim3(1), dim3(1024), 0, s, loss_rows, p.rows, p.N, p.reduction == 1, p.loss);
    return launched("linear_ce_fwd");
}

template <typename T>
int bwd(const VcLceParams& p, hipStream_t s) {
    const BwdLayout L(p.N, p.D, p.V, sizeof(T));
    char* ws = (char*)p.ws;
    float *factor = (float*)(ws + L.g), *acc = (float*)(ws + L.acc), *dbpart = (float*)(ws + L.dbpart);
    const int* count = p.rows + p.N;
    const int st = (p.N + 127) / 128, dt = (p.D + 127) / 128;
    (void)hipGetLastError();
    hipLaunchKernelGGL(lce_factor_kernel, dim3(1), dim3(1), 0, s, p.dloss, p.rows, p.N, p.reduction, factor);
    for (int v0 = 0; v0 < p.V; v0 += L.piece) {
        const int nv = p.V - v0 < L.piece ? p.V - v0 : L.piece, vt = (nv + 127) / 128;
        const T* w = (const T*)p.w + (long long)v0 * p.ldw;
        Gemm g = {};
        g.R = {w, p.ldw, 1, nullptr, nullptr};
        g.S = {p.x, p.ldx, 1, p.rows, nullptr};
        g.nr = nv, g.ns_dev = count, g.K = p.D;
        g.bias = p.bias, g.labels = p.labels, g.rows = p.rows, g.v0 = v0;
        g.lse = p.lse, g.scale = p.reduction == 0 ? p.dloss : nullptr, g.P = ws + L.P, g.ldp = L.piece, g.dbpart = p.db != nullptr ? dbpart : nullptr;
        hipLaunchKernelGGL((lce_gemm_any<T, EPI_PROB>), dim3(vt, st), dim3(256), 0, s, g);
        if (p.db != nullptr)
            hipLaunchKernelGGL((lce_db_kernel<T>), dim3((nv + 255) / 256), dim3(256), 0, s, dbpart, count, factor, nv, (T*)p.db + v0);
        if (p.dx != nullptr) {
            Gemm x = {};
            x.R = {w, 1, p.ldw, nullptr, nullptr};
            x.S = {ws + L.P, L.piece, 1, nullptr, nullptr};
            x.nr = p.D, x.ns_dev = count, x.K = nv, x.acc = acc, x.add = v0 > 0;
            hipLaunchKernelGGL((lce_gemm_any<T, EPI_DX>), dim3(dt, st), dim3(256), 0, s, x);
        }
        if (p.dw != nullptr) {
            Gemm d = {};
            d.R = {p.x, 1, p.ldx, nullptr, p.rows};
            d.S = {ws + L.P, 1, L.piece, nullptr, nullptr};
            d.nr = p.D, d.ns = nv, d.k_dev = count, d.out = (T*)p.dw + (size_t)v0 * p.D, d.g = factor;
            hipLaunchKernelGGL((lce_gemm_any<T, EPI_DW>), dim3(dt, vt), dim3(256), 0, s, d);
        }
    }
    if (p.dx != nullptr) hipLaunchKernelGGL((lce_dx_kernel<T>), dim3(p.N), dim3(256), 0, s, acc, p.rows, factor, p.N, p.D, (T*)p.dx);
    return launched("linear_ce_bwd");
}

}  // namespace

size_t vc_lce_workspace(int N, int D, int V, bool is_bf16, int op) {
    return op == 0 ? FwdLayout(N, V).bytes : BwdLayout(N, D, V, is_bf16 ? 2 : 4).bytes;
}
int vc_lce_launch_fwd(const VcLceParams& p, bool is_bf16, hipStream_t s) { return is_bf16 ? fwd<bf16>(p, s) : fwd<float>(p, s); }
int vc_lce_launch_bwd(const VcLceParams& p, bool is_bf16, hipStream_t s) { return is_bf16 ? bwd<bf16>(p, s) : bwd<float>(p, s); }
