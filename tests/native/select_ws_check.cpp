// A workspace of the block selection that is sized for the largest context and the most tokens (csrc/tsr_sparse4.hip) does for every smaller
// one, and a launch's keys lie in it.
#include <hip/hip_runtime.h>

hipError_t hipSetDevice(int);
#include "tsr_sparse4.hip"

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
int tsr_launch_kv4_bounds(const tsr::Kv4BoundsArgs &, hipStream_t) { return 0; }
int tsr_launch_kv4_select(const tsr::Kv4SelectArgs & a, hipStream_t) {
    used = std::max(used, (size_t)8u * a.T * a.n_head_kv * a.n_blocks);
    return 0;
}
int tsr_launch_attn4_blocks(const tsr::Attn4BlocksArgs &, uint32_t, hipStream_t) { return 0; }

int main() {
    static tsr_hip_ctx ctx;
    ctx.n_cu = 256;
    uint32_t n = 0;
    for (uint32_t block : { 32u, 64u, 96u, 1024u })
        for (uint32_t hkv : { 1u, 3u, 8u, 512u })
            for (uint64_t cells = 0; cells <= 0x7FFFFFFFu; cells = cells < 4096u ? cells + 31u : cells + cells / 25u) {
                size_t before = 0u;
                for (uint32_t T : { 1u, 2u, 3u, 33u, 300u, 512u, 513u, 2000u, 32768u, 65535u }) {
                    const size_t ws = tsr_hip_kv4_select_ws(&ctx, T, hkv, block, (uint32_t)cells);
                    const size_t more = tsr_hip_kv4_select_ws(&ctx, T, hkv, block, (uint32_t)std::min<uint64_t>(0x7FFFFFFFu, cells + block));
                    used = 0u;
                    const int rc = tsr_hip_kv4_select(&ctx, (const float *)0x1000, T, hkv * 64u, (const uint32_t *)0x2000, 0xFFFFFFFFu, 64u, hkv, hkv, block,
                                                      (uint32_t)cells, nullptr, 8u, 1u, 1u, (int32_t *)0x3000, (void *)0x8000, ws, nullptr);
                    if (ws < before || more < ws || rc != 0 || used > ws) {
                        printf("T %u KV heads %u block %u cells %llu: %zu bytes (rc %d, %zu used), %zu for fewer tokens, %zu for more cells\n", T, hkv, block,
                               (unsigned long long)cells, ws, rc, used, before, more);
                        return 1;
                    }
                    before = ws;
                    ++n;
                }
            }
    printf("%u workspaces\n", n);
    return 0;
}
