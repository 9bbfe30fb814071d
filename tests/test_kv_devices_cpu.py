"""Which device the key/value calls work on: the C-ABI layer with a CUDA runtime of two devices that only keeps account."""
import os
import shutil
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "kv_api.cpp"
#include <cstdarg>
#include <cstdio>
#include <cstring>
#define CHECK(c) do { if (!(c)) { printf("line %d: %s (%s)\n", __LINE__, #c, error); return 1; } } while (0)

static char error[512];
static int current = 0, allocated_on = -1, configured_on = -1, cleared_on = -1, launched_on = -1, allocations = 0, launches = 0;
int nnb::fail(int code, const char*, int, const char* fmt, ...) {
    va_list a;
    va_start(a, fmt);
    vsnprintf(error, sizeof error, fmt, a);
    va_end(a);
    return code;
}
extern "C" {
cudaError_t cudaSetDevice(int d) { return d < 2 ? (current = d, cudaSuccess) : cudaErrorInvalidDevice; }
cudaError_t cudaGetDevice(int* d) { return *d = current, cudaSuccess; }
cudaError_t cudaMalloc(void** p, size_t) { return *p = (void*)0x1000, allocated_on = current, ++allocations, cudaSuccess; }
cudaError_t cudaFree(void*) { return cudaSuccess; }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cleared_on = current, cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "an error"; }
cudaError_t cudaEventCreate(cudaEvent_t*) { return cudaErrorUnknown; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
}
namespace nnb {
cudaError_t attention_configure() { return configured_on = current, cudaSuccess; }
bool encode_attention_maps(const KvView&, AttnMaps*) { return true; }
bool attention_countable(const AttnArgs&, int) { return true; }
static cudaError_t launched() { return launched_on = current, ++launches, cudaSuccess; }
cudaError_t launch_kv_write(const KvWriteArgs&, cudaStream_t, bool) { return launched(); }
cudaError_t launch_kv_read(const KvReadArgs&, cudaStream_t, bool) { return launched(); }
cudaError_t launch_attention(const AttnArgs& a, const AttnMaps&, int, int, cudaStream_t, bool, int* n) { return *n = 1, a.counters ? launched() : cudaErrorUnknown; }
}

static nn_buf at(size_t i) { return (nn_buf)(i << 20); }
static nn_kv_batch batch = {1, 2, 2, 64, 4, at(3), at(4), at(5)};
static int attention(nn_context* c, nn_kv_cache* h) { return nn_attention(c, h, &batch, 4, at(64), 0, at(65), 0, 0.125f, 0, 0); }
static int write(nn_context* c, nn_kv_cache* h) { return nn_kv_write(c, h, &batch, at(64), 0, at(65), 0); }
static int read(nn_context* c, nn_kv_cache* h) { return nn_kv_read(c, h, &batch, at(64), 0, at(65), 0); }

int main() {
    nn_context zero, one, other;   // two contexts of device 1
    zero.sm_count = one.sm_count = other.sm_count = 148;
    one.device = other.device = 1;
    nn_kv_cache *h0 = nullptr, *h1 = nullptr;
    CHECK(nn_kv_cache_create(&one, NN_KV_FP16, 4, 16, 2, 64, at(1), at(2), nullptr, nullptr, &h1) == NN_OK && allocated_on == 1 && configured_on == 1 && cleared_on == 1);
    CHECK(nn_kv_cache_create(&zero, NN_KV_FP16, 4, 16, 2, 64, at(1), at(2), nullptr, nullptr, &h0) == NN_OK && allocated_on == 0);

    // a cache of another device: refused, and nothing is made for it
    current = 0;
    allocations = 0;
    for (auto call : {attention, write, read}) CHECK(call(&other, h0) == NN_ERR_ARG && strstr(error, "device"));
    CHECK(allocations == 0 && !other.attn_work && launches == 0);

    // rows go in and out without the attention's workspace, while a recording is going on too, on the context's device
    other.capturing = true;
    for (auto call : {write, read}) {
        current = 0;
        CHECK(call(&other, h1) == NN_OK && launched_on == 1);
    }
    CHECK(allocations == 0 && !other.attn_work);
    // the attention needs it: refused inside a recording, under its own name
    current = 0;
    CHECK(attention(&other, h1) == NN_ERR_UNSUPPORTED && !strncmp(error, "nn_attention", 12) && allocations == 0 && !other.attn_work);
    other.capturing = false;

    // a first call from a thread with another current device: all that it makes is on the context's
    current = 0;
    allocated_on = configured_on = cleared_on = launched_on = -1;
    CHECK(attention(&other, h1) == NN_OK && other.attn_work);
    CHECK(allocated_on == 1 && configured_on == 1 && cleared_on == 1 && launched_on == 1 && allocations == 1);
    current = 0;
    CHECK(attention(&other, h1) == NN_OK && launched_on == 1 && allocations == 1);   // once
    nn_kv_cache_free(h0);
    nn_kv_cache_free(h1);
    return 0;
}
"""


def test_calls_work_on_the_contexts_device(tmp_path):
    src, exe = tmp_path / "devices.cpp", tmp_path / "devices"
    cuda = os.path.join(os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc")), "include")
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(REPO, "adreno-llms_b200", "csrc"), "-isystem", cuda, str(src),
                           "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
