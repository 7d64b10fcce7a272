// Calls the float operators' entry points, built for the host, over random sizes and
// strides with buffers of exactly the extents that they describe.
//   addresses FAMILY COUNT SEED
#include <hip/hip_runtime.h>

#include <random>
#include <vector>

#include "mamba_int.h"

dim3 blockIdx, threadIdx, blockDim, gridDim;
int8_t *host_dynamic_lds;
int host_vote, host_cus, host_dry, host_error;
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

void norm() {
    Pool p;
    const int T = logu(1, 40), d = uni(0, 3) ? logu(1, 2100) : logu(2000, 16384), xt = uni(0, 2), rt = uni(0, 1) ? xt : 0;
    const int e = xt ? 2 : 4, er = rt ? 2 : 4, ldq = d + uni(0, 70), mode = uni(1, 3);
    const View x = rows(p, 1, T, d, e), r = rows(p, 1, T, d, er), y = rows(p, 1, T, d, e, true), ro = rows(p, 1, T, d, er, true);
    const bool in_place = uni(0, 3) == 0;
    call(mi_add_rms_norm(x.p, xt, x.ld, uni(0, 3) ? (in_place ? ro.p : r.p) : nullptr, rt, in_place ? ro.ld : r.ld,
                         p.arr<float>(d), 1e-5f, mode & 1 ? y.p : nullptr, y.ld, mode & 2 ? p.arr<int8_t>((size_t)(T - 1) * ldq + ldq) : nullptr,
                         ldq, p.arr<float>(T), uni(0, 3) ? ro.p : nullptr, ro.ld, T, d, nullptr));
}

void conv() {
    Pool p;
    const int B = logu(1, 5), L = uni(0, 4) ? logu(1, 200) : uni(0, 3), D = logu(1, 600), W = uni(1, 8), t = uni(0, 2), e = t ? 2 : 4;
    const View x = rows(p, B, L, D, e), y = rows(p, B, L, D, e, true);
    void *st = p.get((size_t)B * (W - 1) * D * e), *so = uni(0, 1) ? st : p.get((size_t)B * (W - 1) * D * e);
    call(mi_causal_conv(x.p, x.ld, x.bs, t, p.arr<float>((size_t)D * W), uni(0, 1) ? p.arr<float>(D) : nullptr, W, uni(0, 1),
                        uni(0, 2) ? st : nullptr, uni(0, 2) ? so : nullptr, uni(0, 1) ? p.arr<int32_t>(B) : nullptr, y.p, y.ld, y.bs,
                        B, L, D, nullptr));
}

void scan() {
    Pool p;
    const int G = uni(0, 2) ? 1 : uni(2, 4), t = uni(0, 2), e = t ? 2 : 4;
    const int N = uni(0, 2) ? logu(1, 64) : logu(60, 256), B = logu(1, 3);
    const int D = G * logu(1, 150), L = uni(0, 3) ? logu(1, N > 64 ? 60 : 400) : uni(0, 6);
    host_cus = uni(0, 1) ? 256 : 4;
    const View u = rows(p, B, L, D, e), dt = rows(p, B, L, D, e), b = rows(p, B, L, (int64_t)G * N, e), c = rows(p, B, L, (int64_t)G * N, e),
               z = rows(p, B, L, D, e), y = rows(p, B, L, D, e, true);
    float *h = p.arr<float>((size_t)B * D * N), *ho = uni(0, 1) ? h : p.arr<float>((size_t)B * D * N);
    size_t bytes = 0;
    call(mi_selective_scan_workspace_size(B, L, D, N, G, &bytes));
    call(mi_selective_scan(u.p, u.ld, u.bs, dt.p, dt.ld, dt.bs, p.arr<float>((size_t)D * N), b.p, b.ld, b.bs, c.p, c.ld, c.bs,
                           uni(0, 1) ? p.arr<float>(D) : nullptr, uni(0, 1) ? z.p : nullptr, z.ld, z.bs,
                           uni(0, 1) ? p.arr<float>(D) : nullptr, uni(0, 1), uni(0, 1) ? h : nullptr, uni(0, 1) ? ho : nullptr,
                           uni(0, 1) ? p.arr<int32_t>(B) : nullptr, y.p, y.ld, y.bs, t, B, L, D, N, G, bytes ? p.get(bytes) : nullptr,
                           bytes, nullptr));
}

void w4() {
    Pool p;
    const int M = logu(1, 80), N = logu(1, 700), K = uni(0, 1) ? 128 * uni(1, 6) : logu(1, 900), t = uni(0, 2), e = t ? 2 : 4;
    const int group = std::vector<int>{32, 64, 128, 256, 640}[uni(0, 4)], st = uni(0, 1) ? 0 : 2, es = st ? 2 : 4;
    host_cus = uni(0, 1) ? 256 : uni(1, 12);
    const int64_t nb = (N + 15) / 16, kb = (K + 127) / 128, have = (K + group - 1) / group, ng = group < 128 ? kb * 128 / group : have;
    uint8_t *packed = (uint8_t *)p.get(nb * kb * 1024);
    void *s = p.get(nb * ng * 16 * es);
    const bool zeros = uni(0, 1);
    uint8_t *z = zeros ? (uint8_t *)p.get(nb * ng * 16) : nullptr;
    call(mi_pack_w4((uint8_t *)p.get((size_t)N * K), p.get(N * have * es), st, zeros ? (uint8_t *)p.get(N * have) : nullptr, packed, s, z, N,
                    K, group, nullptr));
    const View x = rows(p, 1, M, K, e), y = rows(p, 1, M, N, e, true);
    call(mi_w4_matvec(x.p, x.ld, t, packed, s, st, z, uni(0, 1) ? p.arr<float>(N) : nullptr, y.p, y.ld, M, N, K, group, nullptr));
}

// the largest sizes that the checks let pass are launches within the runtime's limits
void limits() {
    static char byte[64];
    void *a = (void *)(((uintptr_t)byte + 15) / 16 * 16);
    float *f = (float *)a;
    host_dry = 1;
    for (int cus : {256, 4}) {
        host_cus = cus;
        for (int t : {0, 1}) {
            for (int d : {1, 7, 8, 768, 4096, 16384})
                call(mi_add_rms_norm(a, t, d, a, 0, d, f, 0.0f, a, d, nullptr, 0, nullptr, a, d, (1 << 22) - 1, d, nullptr));
            for (int L : {1, 4, 4096}) call(mi_causal_conv(a, 64, 0, t, f, f, 4, 1, a, a, nullptr, a, 64, 0, 1 << 20, L, 64, nullptr));
            for (int N : {1, 16, 64, 256})
                for (int L : {1, 5, 100000}) {
                    size_t bytes = 0;
                    call(mi_selective_scan_workspace_size(1 << 15, L, 1024, N, 1, &bytes));
                    call(mi_selective_scan(a, 0, 0, a, 0, 0, f, a, 0, 0, a, 0, 0, f, a, 0, 0, f, 1, f, f, nullptr, a, 1024, 0, t, 1 << 15, L,
                                           1024, N, 1, bytes ? a : nullptr, bytes, nullptr));
                }
            call(mi_w4_matvec(a, 0, t, (uint8_t *)a, a, 2, nullptr, nullptr, a, 1000, 32 * 65535, 1000, 128, 128, nullptr));
            call(mi_w4_matvec(a, 0, t, (uint8_t *)a, a, 2, nullptr, nullptr, a, 1 << 28, 7, 1 << 28, 128, 128, nullptr));
        }
    }
}

}  // namespace

int main(int argc, char **argv) {
    const std::string family = argv[1];
    const int count = atoi(argv[2]);
    rng.seed((unsigned)atoi(argv[3]));
    host_cus = 256;
    if (family == "limits") limits();
    for (int i = 0; i < count; ++i) {
        if (family == "norm") norm();
        if (family == "conv") conv();
        if (family == "scan") scan();
        if (family == "w4") w4();
    }
    printf("%d calls, %d refused\n", calls, refused);
    return refused ? 1 : 0;
}
