/* The fixed-rate operators' entry points (dc_host_lowbit.c) under AddressSanitizer and UBSan, with recorded launches
 * (lowbit_host_stubs.c): arguments at and past the edges of every field, in random combinations.  Each call is taken or
 * refused; what is taken has a plan whose workspace the second call accepts. */
#include <limits.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include "../../include/dc_gpu.h"

int stub_launches(void);
unsigned stub_splits(void);

static unsigned long long state = 88172645463325252ull;
static unsigned long long next(void) {
    state ^= state << 13;
    state ^= state >> 7;
    return state ^= state << 17;
}
static const long long EDGES[] = {0, 1, 2, 3, 8, 15, 16, 17, 32, 48, 64, 128, 255, 256, 257, 1000, 4096, 65535, 1 << 20, (1 << 30) - 1, 1 << 30,
                                  INT_MAX, 1ll << 32, 1ll << 35, 1ll << 40, 1ll << 62, LLONG_MAX, -1, -16, INT_MIN, LLONG_MIN};
static long long any(void) { return EDGES[next() % (sizeof EDGES / sizeof *EDGES)]; }
static int any_int(void) { return (int)any(); }
/* mostly a value that is taken */
static long long good(const long long* v, int n) { return next() % 8 ? v[next() % n] : any(); }
#define GOOD(...) good((const long long[]){__VA_ARGS__}, (int)(sizeof((const long long[]){__VA_ARGS__}) / sizeof(long long)))
static void* place(void) { return (void*)(uintptr_t)(next() % 16 ? 0x100000 + GOOD(0, 16, 32, 2, 4, 8) % 4096 : 0); }

int main(void) {
    int taken = 0, refused = 0;
    for (int i = 0; i < 400000; i++) {
        const dc_kv_cache c = {place(), GOOD(1, 4, 1000, 1 << 20), (int)GOOD(16, 48, 64, 1 << 30), (int)GOOD(1, 2, 8), (int)GOOD(32, 64, 96, 128, 256), (int)GOOD(4, 8)};
        const int width = (int)GOOD(1, 3, 1000);
        const dc_kv_batch at = {(int)GOOD(1, 2, 4, 64), (int)GOOD(1, 2, 17, 500), place(), next() % 2 ? place() : NULL, next() % 4 ? place() : NULL, width,
                                next() % 8 ? width : any(), any_int()};
        const long long s[3] = {GOOD(4096, 1 << 20, 64), GOOD(512, 64), GOOD(64, 128)}, t[3] = {GOOD(4096, 1 << 20, 64), GOOD(512, 64), GOOD(64, 128)};
        const int dtype = (int)GOOD(0, 1, 2), heads = (int)GOOD(2, 8, 16, 32);
        const long long context = GOOD(16, 640, 641, 4096, 1 << 20);
        int rc;
        switch (next() % 5) {
            case 0: rc = dc_kv_write_device(&c, &at, dtype, place(), s, place(), t, place()); break;
            case 1: rc = dc_kv_read_device(next() % 16 ? &c : NULL, &at, dtype, place(), s, place(), t, place()); break;
            case 2: {
                const size_t need = dc_kv_attention_workspace(&c, at.batch, at.tokens, heads, context);
                rc = dc_kv_attention_device(&c, next() % 16 ? &at : NULL, dtype, heads, place(), s, 0.125f, 1, context, place(), t, place(),
                                            need ? (void*)0x1000000 : NULL, need, place());
                if (rc == 0 && at.batch && at.tokens && (stub_splits() > 1) != (need > 0)) {
                    printf("a workspace of %zu for %u pieces\n", need, stub_splits());
                    return 1;
                }
                break;
            }
            case 3: rc = dc_act_forward_device((int)GOOD(0, 1, 2), dtype, GOOD(1, 3, 1000), GOOD(1, 8, 37, 4096), place(), GOOD(8, 4096, 8192), next() % 2 ? place() : NULL,
                                               GOOD(8, 4096), place(), GOOD(8, 4096), place(), place(), place()); break;
            default: rc = dc_act_backward_device((int)GOOD(0, 1, 2), dtype, GOOD(1, 3, 1000), GOOD(1, 8, 37, 4096), place(), GOOD(8, 4096, 8192), place(),
                                                 next() % 2 ? place() : NULL, place(), GOOD(8, 4096), next() % 2 ? place() : NULL, GOOD(8, 4096), next() % 2 ? place() : NULL,
                                                 GOOD(8, 4096), place());
        }
        if (rc != 0 && rc != DC_ERR_ARG) {
            printf("call %d: %d\n", i, rc);
            return 1;
        }
        if (rc) refused++;
        else taken++;
    }
    printf("fine: %d taken, %d refused, %d launches\n", taken, refused, stub_launches());
    return 0;
}
