// Host-side check of the operators of long sequences and large vocabularies (include/vc3d.h: vc_gated_scan_*, vc_linear_ce_*,
// vc_adamw_step, vc_bias_columns) under AddressSanitizer + UndefinedBehaviorSanitizer, no GPU needed.  The HIP calls that a launch makes are defined
// here: they write the launch down and succeed, so the planners, workspace layouts and loops over pieces run to their end, for
// small, odd and the largest sizes, with addresses that are never read.  What is checked of every launch: fewer than 2^32 lanes in a
// dimension, no empty grid; of sequences that take several launches, where each part begins.
// Built and run by tests/test_sequence_host_cpu.py (make -C csrc sequencecheck).
#include <cstdio>
#include <cstring>
#include <vector>

#include "kernels.h"
#include "vc3d.h"

struct Launch {
    dim3 grid, block;
    VcScanParams scan;  // (of launches of 1024 threads in a scan: its argument)
};
static std::vector<Launch> launches;
static bool in_scan = false;

static Launch next;
extern "C" hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t, hipStream_t) { return next.grid = grid, next.block = block, hipSuccess; }
extern "C" hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* s) {
    return *grid = next.grid, *block = next.block, *lds = 0, *s = nullptr, hipSuccess;
}
extern "C" hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void** args, size_t, hipStream_t) {
    Launch l = {grid, block, {}};
    if (in_scan && block.x == 1024) memcpy(&l.scan, args[0], sizeof(l.scan));
    launches.push_back(l);
    return hipSuccess;
}
extern "C" hipError_t hipGetLastError(void) { return hipSuccess; }
extern "C" hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
extern "C" hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }

static int failures = 0, calls = 0;
#define CHECK(c, ...)                        \
    do {                                     \
        if (!(c)) {                          \
            ++failures;                      \
            printf("line %d: ", __LINE__);   \
            printf(__VA_ARGS__);             \
            printf(" [%s]\n", vc_last_error()); \
        }                                    \
    } while (0)

static char* const P = (char*)(uintptr_t)(1ull << 44);  // never read
template <typename F>
static void run(const char* what, long long a, long long b, long long c, F f) {
    launches.clear();
    ++calls;
    const int rc = f();
    CHECK(rc == 0, "%s %lld x %lld x %lld: %d", what, a, b, c, rc);
    CHECK(rc != 0 || !launches.empty(), "%s %lld x %lld x %lld: nothing launched", what, a, b, c);
    for (const Launch& l : launches) {
        const unsigned long long x = (unsigned long long)l.grid.x * l.block.x, y = (unsigned long long)l.grid.y * l.block.y;
        CHECK(x > 0 && x < (1ull << 32) && y > 0 && y < (1ull << 32) && l.grid.z == 1 && l.block.x <= 1024, "%s %lld x %lld x %lld: a launch of %u x %u",
              what, a, b, c, l.grid.x, l.block.x);
    }
}

static void scan(int B, int T, int H, bool bf16) {
    const long long elem = bf16 ? 2 : 4;
    vc_scan_desc d = {B, T, H, bf16, 0, 0, 2ll * H * T, 2ll * H};
    const size_t w[2] = {vc_gated_scan_workspace_bytes(&d, 0), vc_gated_scan_workspace_bytes(&d, 1)};
    float* const F = (float*)(P + (1ll << 40));
    in_scan = true;
    for (int op = 0; op < 2; ++op) {
        run(op ? "scan backward" : "scan", B, T, H, [&] {
            return op == 0 ? vc_gated_scan_fwd(&d, P, F, (const int32_t*)F, P, F, F, w[0] ? P : nullptr, w[0], nullptr)
                           : vc_gated_scan_bwd(&d, P, (const int32_t*)F, F, P, F, P, F, w[1] ? P : nullptr, w[1], nullptr);
        });
        int b = 0;
        for (const Launch& l : launches) {
            if (l.block.x != 1024) continue;
            const VcScanParams& q = l.scan;
            const long long row = (long long)b * H, steps = row * T, chunks = (T + 63) / 64;
            CHECK(q.B > 0 && q.T == T && q.H == H && q.gates == P + 2 * steps * elem && q.lengths == (const int*)F + b && q.states == F + row * chunks,
                  "scan %d x %d x %d: the part from %d on", B, T, H, b);
            if (op == 0) CHECK(q.h0 == F + row && q.last == F + row && q.h == P + steps * elem, "scan %d x %d x %d: the part from %d on", B, T, H, b);
            else CHECK(q.dlast == F + row && q.dh0 == F + row && q.dy == P + steps * elem && q.dgates == P + 2 * steps * elem, "scan %d x %d x %d: the part from %d on", B, T, H, b);
            b += q.B;
        }
        CHECK(b == B, "scan %d x %d x %d: %d sequences are launched", B, T, H, b);
    }
    in_scan = false;
    run("step", B, 1, H, [&] { return vc_gated_scan_step(P, 2ll * H, bf16, F, P, B, H, nullptr); });
}

static void loss(int N, int D, int V, bool bf16, int reduction, int64_t keep, bool bias, int odd) {
    const int align = odd ? (bf16 ? 2 : 4) : 0;
    vc_linear_ce_desc d = {N, D, V, bf16, reduction, align, D, D + (odd > 1), -100, keep};
    const size_t w0 = vc_linear_ce_workspace_bytes(&d, 0), w1 = vc_linear_ce_workspace_bytes(&d, 1), s = vc_linear_ce_saved_bytes(&d);
    CHECK(w0 > 0 && w1 > 0 && s >= (size_t)N * 8, "loss %d x %d x %d: sizes %zu %zu %zu", N, D, V, w0, w1, s);
    const char* const w = P + align;
    const void* const b = bias ? P : nullptr;
    float* const F = (float*)P;
    run("loss", N, D, V, [&] { return vc_linear_ce_fwd(&d, P, w, b, (const int64_t*)P, F, P, P, w0, nullptr); });
    for (int want = 1; want < 8; ++want) {
        if ((want & 4) && !bias) continue;
        run("loss backward", N, D, V, [&] {
            return vc_linear_ce_bwd(&d, P, w, b, (const int64_t*)P, P, F, want & 1 ? P : nullptr, want & 2 ? P : nullptr, want & 4 ? P : nullptr, P, w1, nullptr);
        });
    }
}

static void adamw(const std::vector<int64_t>& sizes, bool bf16, int bits) {
    std::vector<vc_adamw_tensor> t;
    for (int64_t n : sizes) t.push_back({P, P, P, P, (float*)P, (float*)P, n});
    const vc_adamw_hyper h = {1e-3, 0.9, 0.999, 1e-8, 0.01, 1.0, 5};
    run("adamw", (long long)sizes.size(), sizes[0], bits, [&] { return vc_adamw_step(t.data(), (int32_t)t.size(), bf16, bits, &h, nullptr, nullptr); });
}

int main() {
    for (bool bf16 : {false, true}) {
        for (int64_t rows : {(int64_t)1, (int64_t)5, (int64_t)262143, (int64_t)1 << 40})
            for (int D : {4, 64, 1 << 24}) run("bias columns", rows, D, 0, [&] { return vc_bias_columns((float*)P, D == 64 ? (float*)P : nullptr, P, bf16, rows, D, nullptr); });
        for (int B : {1, 3, 64, 65535})
            for (int T : {1, 2, 63, 64, 65, 129, 1531, 8192})
                for (int H : {1, 2, 15, 16, 17, 33, 127, 128, 129, 1000, 4096}) scan(B, T, H, bf16);
        scan(1, 1 << 30, 1, bf16), scan(1, 1 << 28, 128, bf16), scan(1, 1, 1 << 24, bf16), scan(3, 129, (1 << 24) - 1, bf16);
        // more workgroups than a launch has room for
        scan(65535, 1, 8193, bf16), scan(65535, 1, 1 << 20, bf16), scan(40000, 129, 16000, bf16), scan(2, 257, 1 << 24, bf16);
        vc_scan_desc d = {1, 1 << 30, 1 << 24, bf16, 0, 0, 1, 1};  // one sequence that has more
        CHECK(vc_gated_scan_workspace_bytes(&d, 0) == 0 && vc_gated_scan_fwd(&d, P, nullptr, nullptr, P, (float*)P, nullptr, P, 1, nullptr) == -2, "accepted");
        for (int reduction = 0; reduction < 3; ++reduction)
            for (int64_t keep : {(int64_t)0, (int64_t)-1, (int64_t)1 << 50})
                for (int odd = 0; odd < 3; ++odd)
                    for (int N : {1, 63, 129, 1777})
                        for (int D : {1, 7, 64, 1000})
                            for (int V : {1, 400, 50257}) loss(N, D, V, bf16, reduction, keep, (N + D + V) % 2, odd);
        for (int64_t keep : {(int64_t)0, (int64_t)-1})
            for (int odd = 0; odd < 3; ++odd) {
                // the largest: more tiles of logits than a launch has room for
                loss(1 << 23, 64, 1 << 23, bf16, 1, keep, true, odd), loss(1 << 20, 1024, 1 << 19, bf16, 1, keep, false, odd);
                loss((1 << 23) - 1, 1, (1 << 23) - 1, bf16, 0, keep, true, odd), loss(1, 1 << 14, 1 << 23, bf16, 2, keep, true, odd);
                loss(1 << 23, 1 << 14, 1, bf16, 1, keep, true, odd), loss(1 << 17, 1 << 20, 1000, bf16, 1, keep, true, odd);
            }
        vc_linear_ce_desc e = {1 << 23, 1 << 20, 10, bf16, 1, 0, 1 << 20, 1 << 20, -100, 0};
        CHECK(vc_linear_ce_workspace_bytes(&e, 0) == 0, "accepted");
        for (int bits : {8, 32}) {
            adamw({1}, bf16, bits), adamw({255, 256, 257, 4096, 4097}, bf16, bits), adamw(std::vector<int64_t>(200, 1000), bf16, bits);
            adamw({(1ll << 36) - 4096}, bf16, bits), adamw({1ll << 35, 1ll << 35, 1ll << 35, 7}, bf16, bits);
            vc_adamw_tensor t = {P, P, P, P, (float*)P, (float*)P, 1ll << 36};
            const vc_adamw_hyper h = {1e-3, 0.9, 0.999, 1e-8, 0.01, 1.0, 5};
            CHECK(vc_adamw_step(&t, 1, bf16, bits, &h, nullptr, nullptr) == -2, "accepted");
        }
    }
    printf("calls %d, failures %d\n", calls, failures);
    return failures != 0;
}
