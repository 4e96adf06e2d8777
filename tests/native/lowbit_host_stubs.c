/* Stands in for the GPU side of dc_host_lowbit.c: the launches are recorded instead of made, HIP says what the test sets.
 * Linked with that file into a library for tests/test_lowbit_host.py. */
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
#include <string.h>

#include "../../data-compression_amd/csrc/dc_shared.h"
#include "../../include/dc_gpu.h"

static KvArgs last_kv;
static ActArgs last_act;
static int launches;
static unsigned word[16];
static char message[256];
static unsigned takes_bits;
static int device_of_streams, capture_beside;

int dc_init(int device) { (void)device; return DC_OK; }
int dc_get_device(void) { return 0; }
static hipError_t left;                     /* what HIP's last error is */
hipError_t hipGetLastError(void) {
    const hipError_t e = left;
    left = hipSuccess;
    return e;
}
hipError_t hipStreamGetDevice(hipStream_t st, hipDevice_t* d) {
    (void)st;
    *d = device_of_streams;
    return device_of_streams < 0 ? hipErrorInvalidHandle : hipSuccess;
}
hipError_t hipGetDevice(int* d) { return hipStreamGetDevice(NULL, d); }
unsigned* dc_kv_status_word(void) { return word; }
int dc_set_error(int code, const char* msg) {
    strncpy(message, msg, sizeof message - 1);
    return code;
}
int dc_kv_wide_cols(int dim) { return dim <= 160 ? 32 : 16; }
int dc_launch_kv_rows(const KvArgs* a, int write, dc_hip_stream st) {
    (void)write; (void)st;
    last_kv = *a;
    launches++;
    return 0;
}
int dc_launch_kv_attention(const KvArgs* a, dc_hip_stream st) { return dc_launch_kv_rows(a, 0, st); }
int dc_launch_act(const ActArgs* a, int back, dc_hip_stream st) {
    (void)back; (void)st;
    last_act = *a;
    launches++;
    return 0;
}
int dc_launch_kv_take(unsigned* w, dc_hip_stream st) {
    (void)st;
    w[1] = w[0];
    w[0] = takes_bits;                  /* (of a call on another stream) */
    return 0;
}
hipError_t hipStreamIsCapturing(hipStream_t st, hipStreamCaptureStatus* s) {
    (void)st;
    *s = hipStreamCaptureStatusNone;
    return left = capture_beside ? hipErrorStreamCaptureImplicit : hipSuccess;
}
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind k, hipStream_t st) {
    (void)k; (void)st;
    memcpy(d, s, n);
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t st) { (void)st; return hipSuccess; }

/* for the test */
int stub_launches(void) { return launches; }
const char* stub_message(void) { return message; }
void stub_word(unsigned now, unsigned then) { word[0] = now; takes_bits = then; }
void stub_device(int d) { device_of_streams = d; }
void stub_capture_beside(int on) { capture_beside = on; }
int stub_left(void) { return left; }
int stub_vec(void) { return last_kv.vec; }
int stub_vec_out(void) { return last_kv.vec_out; }
unsigned stub_splits(void) { return last_kv.splits; }
long long stub_rows(void) { return last_kv.rows; }
int stub_act_mode(void) { return last_act.mode; }
