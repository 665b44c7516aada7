// A workspace of attention weights that is sized for the largest context (csrc/tsr_evict4.hip) does for every smaller one, and the cut's
// parts lie in it.
#include <hip/hip_runtime.h>

hipError_t hipSetDevice(int);
#include "tsr_evict4.hip"

#include <cstdio>

static size_t used;
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus * s) { *s = hipStreamCaptureStatusNone; return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipMalloc(void ** p, size_t) { *p = (void *)(uintptr_t)0x10000; return hipSuccess; }
hipError_t hipFree(void *) { return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *, unsigned) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
int tsr::hip_err(hipError_t e, const char *) { return e == hipSuccess ? 0 : TSR_HIP_E_HIP; }
int tsr_launch_attn4_weights(const tsr::Attn4Args &, const tsr::Weights4Plan & p, const float *, float, hipStream_t) {
    used = p.ws_bytes;
    return 0;
}
int tsr_launch_kv_pick(const float *, uint32_t, uint32_t, uint32_t, uint32_t, int64_t *, float *, hipStream_t) { return 0; }
int tsr_launch_kv_gather(const tsr::KvGatherArgs &, uint32_t, uint32_t, hipStream_t) { return 0; }
int tsr_launch_kv_rows_copy(uint8_t *, size_t, const uint8_t *, size_t, size_t, uint32_t, hipStream_t) { return 0; }

int main() {
    static tsr_hip_ctx ctx;
    ctx.n_cu = 256;
    tsr_hip_kv k;
    k.type = TSR_HIP_KV_Q4_0;
    uint32_t n = 0;
    for (uint32_t D : { 64u, 128u, 256u, 512u })
        for (uint32_t hkv : { 1u, 2u, 3u, 8u })
            for (uint32_t G : { 1u, 4u, 7u, 8u, 20u, 32u, 64u }) {
                if ((uint64_t)hkv * G * D > 32768u) continue;
                k.E = hkv * D;
                for (uint32_t T : { 1u, 2u, 3u, 9u, 64u, 512u, 20000u, 65535u }) {
                    size_t before = 0u;
                    for (uint64_t cells = 1; cells <= 0x7FFFFFFFu; cells = cells < 4096u ? cells + 1u + cells / 40u * 7u : cells + cells / 50u) {
                        const size_t ws = tsr_hip_attn_weights_kv4_ws(&ctx, T, D, hkv * G, hkv, (uint32_t)cells);
                        k.kv_size = (uint32_t)cells;
                        const int rc = tsr_hip_attn_weights_kv4(&ctx, (const float *)0x1000, T, hkv * G * D, &k, D, hkv * G, hkv, 0.1f, (uint32_t)cells,
                                                                nullptr, nullptr, 0.0f, (float *)0x2000, (void *)0x8000, ws, nullptr);
                        if (ws < before || rc != 0 || used > ws) {
                            printf("T %u D %u heads %u G %u: %zu bytes for %llu cells (rc %d, %zu used), %zu for fewer\n", T, D, hkv, G, ws,
                                   (unsigned long long)cells, rc, used, before);
                            return 1;
                        }
                        before = ws;
                        ++n;
                    }
                }
            }
    printf("%u workspaces\n", n);
    return 0;
}
