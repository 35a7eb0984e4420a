/* Calls that may fail on several threads at once (lpta.serving's threads share a
 * device's handle: its own calls, sizes asked for, calls that queue), on the HIP
 * runtime of host_paths_check.c: each error's message is whole, whoever reads it
 * when. */
#define main host_paths_main
#include "host_paths_check.c"
#undef main
#include <pthread.h>

enum { ROUNDS = 100000, THREADS = 4 };
static tl_handle* H;
static const char* const messages[2] = {"group must be 32, 64 or 128 and k a multiple of it, at most 1024 groups",
                                        "empty weights"};

static int known(const char* s) { return !strcmp(s, messages[0]) || !strcmp(s, messages[1]); }

static void* fails(void* arg) {
    const long me = (long)arg;
    long bad = 0;
    int64_t bytes;
    for (int i = 0; i < ROUNDS; i++) {
        const int want = me & 1 ? TL_ERR_BAD_DESCRIPTOR : TL_ERR_UNSUPPORTED;
        const int got = tl_w4_packed_bytes(H, me & 1 ? 0 : 32, 256, me & 1 ? 64 : 16, TL_F32, &bytes);
        bad += got != want || !known(tl_last_error(H));
    }
    return (void*)bad;
}

int main(void) {
    H = make(1024, 4);
    int64_t bytes;
    long wrong = tl_w4_packed_bytes(H, 0, 256, 64, TL_F32, &bytes) != TL_ERR_BAD_DESCRIPTOR;
    pthread_t t[THREADS];
    for (long i = 0; i < THREADS; i++) pthread_create(&t[i], NULL, fails, (void*)i);
    for (int i = 0; i < THREADS; i++) {
        void* bad;
        pthread_join(t[i], &bad);
        wrong += (long)bad;
    }
    tl_destroy(H);
    printf("%ld wrong\n", wrong);
    return wrong != 0;
}
