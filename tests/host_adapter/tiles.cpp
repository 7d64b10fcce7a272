// Calls the adapters' entry point, built for the host, over sizes whose first product takes 64
// tokens a block and whose second takes several turns of tokens, with buffers of exactly the
// extents that it describes.
//   tiles CUS COUNT SEED
#include <hip/hip_runtime.h>

#include <random>
#include <vector>

#include "mamba_int.h"

dim3 blockIdx, threadIdx, blockDim, gridDim;
int8_t *host_dynamic_lds;
int host_vote, host_cus, host_dry, host_error, host_nan;
const char *host_kernel = "";

void host_die(const char *what, long long a, long long b) {
    printf("%s: %lld of %lld in %s\n", what, a, b, host_kernel);
    fflush(stdout);
    abort();
}

namespace {

std::mt19937 rng;
int uni(int a, int b) { return a + (int)(rng() % (unsigned)(b - a + 1)); }
struct Pool {
    std::vector<void *> v;
    ~Pool() { for (void *p : v) free(p); }
    void *get(size_t bytes, size_t skip = 0) {
        char *p = (char *)calloc(bytes + skip ? bytes + skip : 1, 1);
        v.push_back(p);
        return p + skip;
    }
};

}  // namespace

int main(int, char **argv) {
    host_cus = atoi(argv[1]);
    int refused = 0;
    for (int i = 0; i < atoi(argv[2]); ++i) {
        rng.seed(atoi(argv[3]) * 100003 + i);
        Pool p;
        // every fourth with columns for 1024 blocks of 64 tokens
        const bool wide = i % 4 == 3;
        const int t = uni(0, 2), w = uni(0, 2), ew = w ? 2 : 4, xt = uni(0, 2) ? t : 4, ex = xt == 4 ? 1 : xt ? 2 : 4, e = t ? 2 : 4;
        const int B = wide ? 4 : uni(1, 3), L = uni(8, 400), K = uni(0, 9) ? uni(1, 300) : uni(1, 2000), bank = uni(1, 3),
                  N = wide ? 1024 * 256 / (B * ((L + 63) / 64)) + uni(0, 300) : uni(1, 500), R = uni(0, 4) ? uni(1, 40) : uni(41, 128);
        const int64_t ldx = K + uni(0, 5), bsx = L * ldx + uni(0, 9), ldy = N + uni(0, 5), bsy = L * ldy + uni(0, 9);
        const size_t ys = (size_t)((B - 1) * bsy + (L - 1) * ldy + N) * e;
        host_nan = uni(0, 1) ? 0 : wide ? 5000 : 50;
        void *x = p.get((size_t)((B - 1) * bsx + (L - 1) * ldx + K) * ex, (size_t)uni(0, 8) * ex), *y = p.get(ys, (size_t)uni(0, 8) * e);
        int32_t *ids = (int32_t *)p.get(B * 4), *lens = uni(0, 1) ? (int32_t *)p.get(B * 4) : nullptr;
        for (int b = 0; b < B; ++b) {
            ids[b] = uni(-1, bank - 1);
            if (lens) lens[b] = uni(0, L);
        }
        size_t bytes = 0;
        mi_adapter_workspace_size(B, L, R, &bytes);
        if (mi_adapter_add(x, xt, ldx, bsx, xt == 4 ? (float *)p.get((size_t)B * L * 4) : nullptr, p.get((size_t)bank * R * K * ew),
                           p.get((size_t)bank * N * R * ew), w, uni(0, 1) ? (float *)p.get(bank * 4) : nullptr, ids, lens, y, ldy, bsy,
                           uni(0, 1) ? y : p.get(ys), ldy, bsy, t, B, L, K, N, R, bank, p.get(bytes), bytes, nullptr) != MI_OK) {
            ++refused;
            printf("refused: %s\n", mi_last_error_string());
        }
    }
    return refused != 0;
}
