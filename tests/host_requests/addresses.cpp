// Calls the entry points of the gated recurrence and of the adapters, built for the host, over
// random sizes and strides with buffers of exactly the extents that they describe.
//   addresses FAMILY COUNT SEED
#include <hip/hip_runtime.h>

#include <random>
#include <vector>

#include "mamba_int.h"

dim3 blockIdx, threadIdx, blockDim, gridDim;
int8_t *host_dynamic_lds;
int host_vote, host_cus = 256, host_dry, host_error;
const char *host_kernel = "";

void host_die(const char *what, long long a, long long b) {
    printf("%s: %lld of %lld in %s\n", what, a, b, host_kernel);
    fflush(stdout);
    abort();
}

namespace {

std::mt19937 rng;
int uni(int a, int b) { return a + (int)(rng() % (unsigned)(b - a + 1)); }
int logu(int lo, int hi) {
    const int v = (int)lround(exp(log(lo) + (log(hi) - log(lo)) * (rng() / 4294967296.0)));
    return v < lo ? lo : v > hi ? hi : v;
}
struct Pool {
    std::vector<void *> v;
    ~Pool() { for (void *p : v) free(p); }
    void *get(size_t bytes, size_t skip = 0) {   // `bytes` bytes that begin `skip` bytes past an aligned address
        char *p = (char *)malloc(bytes + skip ? bytes + skip : 1);
        v.push_back(p);
        for (size_t i = 0; i < bytes + skip; i += 1 + rng() % 7) p[i] = (char)(rng() >> 3);
        return p + skip;
    }
    template <class T> T *arr(size_t n) { return (T *)get(n * sizeof(T)); }
};
struct View {
    void *p;
    int64_t ld, bs;
};
// rows [batch, len, dim] that end with the buffer, at any element's address
View rows(Pool &p, int64_t batch, int64_t len, int64_t dim, int size, bool out = false) {
    int64_t ld = dim + (uni(0, 1) ? 0 : uni(0, 9)), bs = len * ld + (uni(0, 1) ? 0 : uni(0, 20));
    if (!out && uni(0, 7) == 0) bs = 0;          // one sequence for all
    if (!out && uni(0, 7) == 0) ld = 0;          // one row for all
    const int64_t n = batch && len ? (batch - 1) * bs + (len - 1) * ld + dim : 0;
    return {p.get(n * size, (size_t)uni(0, 8) * size), ld, bs};
}
int calls, refused;
void call(mi_status st) {
    ++calls;
    if (st != MI_OK) {
        ++refused;
        printf("refused: %s\n", mi_last_error_string());
    }
}

void gated() {
    Pool p;
    const int t = uni(0, 2), e = t ? 2 : 4, B = logu(1, 4), L = uni(0, 3) ? logu(1, 2600) : uni(0, 20), D = logu(1, L > 400 ? 140 : 400);
    host_cus = uni(0, 1) ? 256 : 1;
    const View x = rows(p, B, L, D, e), r = rows(p, B, L, D, e), i = rows(p, B, L, D, e), z = rows(p, B, L, D, e), y = rows(p, B, L, D, e, true),
               dy = rows(p, B, L, D, e);
    size_t forward = 0, backward = 0, saved = 0;
    call(mi_gated_scan_sizes(B, L, D, &forward, &backward, &saved));
    float *h = p.arr<float>((size_t)B * D), *ho = uni(0, 1) ? h : p.arr<float>((size_t)B * D), *sv = (float *)p.get(saved);
    const bool gate = uni(0, 1);
    int32_t *lens = uni(0, 1) ? p.arr<int32_t>(B) : nullptr;
    if (lens && uni(0, 2))
        for (int b = 0; b < B; ++b) lens[b] = uni(0, L);
    float *decay = p.arr<float>(D);
    call(mi_gated_scan(x.p, x.ld, x.bs, r.p, r.ld, r.bs, i.p, i.ld, i.bs, decay, 8.0f, gate ? z.p : nullptr, z.ld, z.bs, uni(0, 1) ? h : nullptr,
                       uni(0, 1) ? ho : nullptr, lens, y.p, y.ld, y.bs, uni(0, 1) ? sv : nullptr, t, B, L, D, p.get(forward), forward, nullptr));
    const size_t n = (size_t)B * L * D * e;
    call(mi_gated_scan_backward(dy.p, dy.ld, dy.bs, x.p, x.ld, x.bs, r.p, r.ld, r.bs, i.p, i.ld, i.bs, decay, 8.0f, gate ? z.p : nullptr, z.ld,
                                z.bs, lens, sv, uni(0, 2) ? p.get(n) : nullptr, uni(0, 2) ? p.get(n) : nullptr, uni(0, 2) ? p.get(n) : nullptr,
                                gate ? p.get(n) : nullptr, uni(0, 2) ? p.arr<float>(D) : nullptr, uni(0, 1) ? p.arr<float>((size_t)B * D) : nullptr,
                                t, B, L, D, p.get(backward), backward, nullptr));
}

void adapter() {
    Pool p;
    const int t = uni(0, 2), w = uni(0, 2), ew = w ? 2 : 4, xt = uni(0, 2) ? t : 4, ex = xt == 4 ? 1 : xt ? 2 : 4, e = t ? 2 : 4;
    const int B = logu(1, 6), L = uni(0, 1) ? 1 : logu(1, 90), K = uni(0, 15) ? logu(1, 700) : 0, N = logu(1, 600), R = uni(0, 4) ? logu(1, 40) : uni(0, 2) ? uni(0, 128) : 0,
              bank = logu(1, 5);
    const View x = rows(p, B, L, K, ex), y = rows(p, B, L, N, e, true), o = rows(p, B, L, N, e, true);
    size_t bytes = 0;
    call(mi_adapter_workspace_size(B, L, R, &bytes));
    int32_t *ids = p.arr<int32_t>(B), *lens = uni(0, 1) ? p.arr<int32_t>(B) : nullptr;
    for (int b = 0; b < B; ++b) ids[b] = uni(0, 9) ? uni(-1, bank - 1) : (int)rng();
    if (lens && uni(0, 2))
        for (int b = 0; b < B; ++b) lens[b] = uni(0, L);
    const View &to = uni(0, 1) ? y : o;
    call(mi_adapter_add(x.p, xt, x.ld, x.bs, xt == 4 ? p.arr<float>((size_t)B * L) : nullptr, p.get((size_t)bank * R * K * ew),
                        p.get((size_t)bank * N * R * ew), w, uni(0, 1) ? p.arr<float>(bank) : nullptr, ids, lens, y.p, y.ld, y.bs, to.p, to.ld, to.bs,
                        t, B, L, K, N, R, bank, p.get(bytes), bytes, nullptr));
}

// the largest sizes that the checks let pass are launches within the runtime's limits
void limits() {
    static char byte[64];
    void *a = (void *)(((uintptr_t)byte + 15) / 16 * 16);
    float *f = (float *)a;
    int32_t *n = (int32_t *)a;
    host_dry = 1;
    for (int t : {0, 1}) {
        const struct { int B, L, D; } sizes[] = {{65535, 1, 64}, {65535, 1, 64 * 127}, {65535, 2, 64 * 127}, {65535, 16, 64 * 127},
                                                 {65535, 17, 64 * 127}, {65535, 64, 64 * 127}, {1, (1 << 29) - 64, 1}, {1, 1, 1 << 24}, {8, 1 << 19, 6400}};
        for (const auto &s : sizes) {
            size_t w[3];
            call(mi_gated_scan_sizes(s.B, s.L, s.D, w, w + 1, w + 2));
            call(mi_gated_scan(a, 0, 0, a, 0, 0, a, 0, 0, f, 8.0f, a, 0, 0, f, f, n, a, 1 << 24, 0, f, t, s.B, s.L, s.D, a, w[0], nullptr));
            call(mi_gated_scan_backward(a, 0, 0, a, 0, 0, a, 0, 0, a, 0, 0, f, 8.0f, a, 0, 0, n, f, a, a, a, a, f, f, t, s.B, s.L, s.D, a, w[1], nullptr));
        }
        const struct { int B, L, K, N, R; } adapters[] = {{(1 << 22) - 1, 1, 1 << 23, 1 << 23, 128}, {1, (1 << 22) - 1, 1 << 23, 1 << 23, 128},
                                                          {(1 << 22) - 1, 1, 64, 1, 1}, {2047, 2048, 8192, 8192, 16}, {1 << 20, 3, 64, 64, 0}};
        for (const auto &s : adapters) {
            size_t w = 0;
            call(mi_adapter_workspace_size(s.B, s.L, s.R, &w));
            call(mi_adapter_add(a, t, 0, 0, nullptr, a, a, 1, f, n, n, a, 0, 0, (char *)a + 4, 1 << 23, 0, t, s.B, s.L, s.K, s.N, s.R, 4, a, w, nullptr));
        }
    }
}

}  // namespace

int main(int argc, char **argv) {
    const std::string family = argv[1];
    const int count = atoi(argv[2]), seed = atoi(argv[3]);
    for (int i = 0; i < (family == "limits" ? 1 : count); ++i) {
        rng.seed(seed * 100003 + i);
        host_vote = i & 1;
        if (family == "gated") gated();
        if (family == "adapter") adapter();
        if (family == "limits") limits();
    }
    printf("%d calls, %d refused\n", calls, refused);
    return refused != 0;
}
