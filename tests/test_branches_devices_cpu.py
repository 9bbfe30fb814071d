"""Which device the calls on trees, moves and beams work on, and what they launch: the C-ABI layer with a CUDA runtime of two devices that only keeps account."""
import os
import shutil
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "kv_api.cpp"
#include "branch_api.cpp"
#include <cstdarg>
#include <cstdio>
#include <cstring>
#define CHECK(c) do { if (!(c)) { printf("line %d: %s (%s)\n", __LINE__, #c, error); return 1; } } while (0)

static char error[512];
static int current = 0, launched_on = -1, launches = 0, layers = 0, tables = 0, heads = 0, pages = 0;
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
cudaError_t cudaMalloc(void** p, size_t) { return *p = (void*)0x1000, cudaSuccess; }
cudaError_t cudaFree(void*) { return cudaSuccess; }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "an error"; }
cudaError_t cudaEventCreate(cudaEvent_t*) { return cudaErrorUnknown; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
}
namespace nnb {
static bool refuse = false;
static cudaError_t launched() { return launched_on = current, ++launches, refuse ? cudaErrorUnknown : cudaSuccess; }
cudaError_t attention_configure() { return cudaSuccess; }
bool encode_attention_maps(const KvView&, AttnMaps*) { return true; }
bool attention_countable(const AttnArgs&, int) { return true; }
cudaError_t launch_kv_write(const KvWriteArgs& a, cudaStream_t, bool) { return a.position ? launched() : cudaErrorUnknown; }
cudaError_t launch_kv_read(const KvReadArgs&, cudaStream_t, bool) { return launched(); }
cudaError_t launch_attention(const AttnArgs& a, const AttnMaps&, int, int, cudaStream_t, bool, int* n) { return *n = 1, a.tree && a.tree_words == 2 && !a.window ? launched() : cudaErrorUnknown; }
cudaError_t launch_tree_layout(const TreeLayoutArgs&, cudaStream_t, bool) { return launched(); }
static void count(const CellRowsOfLayers& c, int most_heads) { layers += c.n; heads = most_heads; }
cudaError_t launch_kv_move(const KvMoveArgs& a, cudaStream_t, bool) { return count(a.caches, a.most_heads), pages = a.num_pages, launched(); }
cudaError_t launch_kv_reorder(const KvReorderArgs& a, cudaStream_t, bool) { return count(a.caches, a.most_heads), tables += a.with_table, pages = a.num_pages, launched(); }
cudaError_t launch_beam_select(const BeamSelectArgs& a, int sms, cudaStream_t, bool) { return a.counters && a.rows && a.parts && sms == 148 ? launched() : cudaErrorUnknown; }
void beam_segments(int, int, int, int* segs, int* per) { *segs = 3, *per = 1024; }
}

static nn_buf at(size_t i) { return (nn_buf)(i << 20); }
static nn_kv_batch batch = {2, 4, 2, 64, 4, at(3), at(4), at(5)};
static int layout(nn_context* c, nn_kv_cache*) { return nn_tree_layout(c, &batch, at(20), 2, at(21), at(22)); }
static int tree(nn_context* c, nn_kv_cache* h) { return nn_attention_tree(c, h, &batch, 4, at(64), 0, at(65), 0, 0.125f, 2, at(21)); }
static int rope(nn_context* c, nn_kv_cache* h) { return nn_rope_kv_write_at(c, h, &batch, at(22), at(30), at(31), 64, 64, 4, at(64), 0, at(64), 0, at(66), 0, at(67), 0); }
static int move(nn_context* c, nn_kv_cache* h) { return nn_kv_move(c, &h, 1, &batch, at(23)); }
static int reorder(nn_context* c, nn_kv_cache* h) { return nn_kv_reorder(c, &h, 1, &batch, 2, at(23)); }
static int select(nn_context* c, nn_kv_cache*) { return nn_beam_select(c, 2, 2, 100, at(40), 0, at(41), nullptr, -1, 4, at(42), at(43), at(44), nullptr); }

int main() {
    nn_context zero, one;
    zero.sm_count = one.sm_count = 148;
    one.device = 1;
    zero.beam_work = one.beam_work = (void*)0x10000;
    nn_kv_cache *h0 = nullptr, *h1 = nullptr;
    CHECK(nn_kv_cache_create(&one, NN_KV_FP16, 4, 16, 2, 64, at(1), at(2), nullptr, nullptr, &h1) == NN_OK);
    CHECK(nn_kv_cache_create(&zero, NN_KV_FP16, 4, 16, 2, 64, at(1), at(2), nullptr, nullptr, &h0) == NN_OK);
    // a cache of another device is refused
    for (auto call : {tree, rope, move, reorder}) CHECK(call(&one, h0) == NN_ERR_ARG && strstr(error, "device") && launches == 0);
    // each call is one launch on its context's device, whatever is current, and needs nothing that a recording could not make
    one.capturing = true;
    for (auto call : {layout, tree, rope, move, reorder, select}) {
        current = 0;
        const long long before = one.launches;
        const int n = launches;
        CHECK(call(&one, h1) == NN_OK && launched_on == 1 && launches == n + 1 && one.launches == before + 1);
    }
    one.capturing = false;
    // what CUDA refuses is reported
    refuse = true;
    for (auto call : {layout, tree, rope, move, reorder, select}) CHECK(call(&one, h1) == NN_ERR_CUDA && strstr(error, "launch failed"));
    refuse = false;
    // what they write is known to be on its way
    one.in_flight.ordered();
    CHECK(select(&one, nullptr) == NN_OK && one.in_flight.may_write(at(43), 4) && one.in_flight.may_write((char*)at(42) + 28, 4) && !one.in_flight.may_write(at(41), 4));
    CHECK(reorder(&one, h1) == NN_OK && one.in_flight.may_write(at(5), 4) && one.in_flight.may_write(at(2), 4) && !one.in_flight.may_write(at(4), 4));
    CHECK(layout(&one, nullptr) == NN_OK && one.in_flight.may_write(at(21), 32) && one.in_flight.may_write(at(22), 16) && !one.in_flight.may_write(at(20), 16));
    // many layers: all of them, 64 to a launch, the table once; heads and pages that differ
    nn_kv_cache* many[130];
    for (int i = 0; i < 130; ++i) CHECK(nn_kv_cache_create(&zero, NN_KV_FP16, 4 + i % 3, 16, 1 + i % 5, 64, at(1000 + 2 * i), at(1001 + 2 * i), nullptr, nullptr, &many[i]) == NN_OK);
    launches = layers = tables = 0;
    CHECK(nn_kv_move(&zero, many, 130, &batch, at(23)) == NN_OK && launches == 3 && layers == 130 && heads == 5);   // (of the last two: 4 and 5)
    launches = layers = 0;
    CHECK(nn_kv_reorder(&zero, many, 130, &batch, 2, at(23)) == NN_OK && launches == 3 && layers == 130 && tables == 1 && pages == 4);   // (6 and 4)
    CHECK(nn_kv_reorder(&zero, many, 64, &batch, 2, at(23)) == NN_OK && launches == 4 && pages == 4 && heads == 5);
    // a page is in all layers or in none, whichever launch they are in (the last of these alone has 6)
    pages = 0;
    CHECK(nn_kv_move(&zero, many + 1, 65, &batch, at(23)) == NN_OK && pages == 4);
    pages = 0;
    CHECK(nn_kv_reorder(&zero, many + 1, 65, &batch, 2, at(23)) == NN_OK && pages == 4);
    // the segments have room
    CHECK(nn_beam_select(&zero, 2731, 1, 100, at(40), 0, at(41), nullptr, -1, 4, at(42), at(43), at(44), nullptr) == NN_ERR_UNSUPPORTED && strstr(error, "segments"));
    CHECK(nn_beam_select(&zero, 2730, 1, 100, at(40), 0, at(41), nullptr, -1, 4, at(42), at(43), at(44), nullptr) == NN_OK);
    CHECK(nn_beam_select(&zero, 1, 1, (1 << 26) + 1, at(400), 0, at(41), nullptr, -1, 4, at(42), at(43), at(44), nullptr) == NN_ERR_UNSUPPORTED);
    for (nn_kv_cache* c : many) nn_kv_cache_free(c);
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
