// Draws the tokens of the cases in a file with the sampling kernels built for the host:
//   draw CASES RESULTS
// A case: int32 type, rows, vocab, all (the first row's parameters as the call's numbers);
// double scale; float u, temperature, top_p, min_p [rows]; int32 top_k [rows]; the logits.
// A result: int64 ids [rows], float logprob [rows].  Buffers are of exactly these extents.
#include <hip/hip_runtime.h>

#include <string.h>

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

int main(int, char **argv) {
    FILE *in = fopen(argv[1], "rb"), *out = fopen(argv[2], "wb");
    int32_t head[4];
    while (fread(head, 4, 4, in) == 4) {
        const int t = head[0], B = head[1], V = head[2], all = head[3];
        double scale;
        if (fread(&scale, 8, 1, in) != 1) return 3;
        const auto read = [&](size_t bytes) {
            void *p = malloc(bytes);
            if (fread(p, 1, bytes, in) != bytes) exit(3);
            return p;
        };
        float *u = (float *)read(B * 4), *temperature = (float *)read(B * 4), *p = (float *)read(B * 4), *least = (float *)read(B * 4);
        int32_t *k = (int32_t *)read(B * 4);
        void *logits = read((size_t)B * V * (t == MI_F32 || t == MI_I32 ? 4 : 2));
        int64_t *ids = (int64_t *)malloc(B * 8);
        float *lp = (float *)malloc(B * 4);
        memset(ids, 0x5a, B * 8);
        memset(lp, 0x5a, B * 4);
        size_t bytes = 0;
        mi_sample_workspace_size(B, V, &bytes);
        char *ws = bytes ? (char *)aligned_alloc(16, bytes) : nullptr;
        memset(ws, 0xa5, bytes);
        const mi_status st = mi_sample_tokens(logits, t, V, scale, u, all ? nullptr : temperature, temperature[0], all ? nullptr : k, k[0],
                                              all ? nullptr : p, p[0], all ? nullptr : least, least[0], ids, lp, B, V, ws, bytes, nullptr);
        if (st != MI_OK) {
            printf("refused: %s\n", mi_last_error_string());
            return 4;
        }
        fwrite(ids, 8, B, out);
        fwrite(lp, 4, B, out);
        for (void *q : {(void *)u, (void *)temperature, (void *)p, (void *)least, (void *)k, logits, (void *)ids, (void *)lp, (void *)ws}) free(q);
        printf("%d x %d of type %d\n", B, V, t);
        fflush(stdout);
    }
    fclose(out);
    return 0;
}
