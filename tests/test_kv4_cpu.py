"""Refusals of the 4-bit key/value cache's entry points and the sizes they report; nothing is launched."""
import ctypes
import random

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from qwen_engine_b200 import build
    build.build()
    from qwen_engine_b200 import _lib
    return _lib.load()


P = 4096          # an address that is never followed: argument checks come first


def views(**changes):
    from qwen_engine_b200._lib import KV4BatchView, KV4CacheView
    c = dict(pages=P, key_weight=P, num_pages=8, num_kv_heads=2, page_size=16)
    b = dict(block_table=P, seq_lens=P, query_start=P, num_seqs=3, max_pages_per_seq=4, num_tokens=5)
    for k, v in changes.items():
        (c if k in c else b)[k] = v
    return ctypes.byref(KV4CacheView(*c.values())), ctypes.byref(KV4BatchView(*b.values()))


def calls(lib, **changes):
    """Every entry point with good arguments but for `changes`; their statuses."""
    c, b = views(**{k: v for k, v in changes.items() if k in (
        "pages", "key_weight", "num_pages", "num_kv_heads", "page_size", "block_table", "seq_lens", "query_start", "num_seqs", "max_pages_per_seq", "num_tokens")})
    a = dict(q=P, k=P, v=P, q_bias=None, k_bias=None, v_bias=None, positions=None, inv=None, q_out=P, heads=12, q_stride=0, kv_stride=0, out=P, lse=P, ws=P,
             ws_bytes=1 << 40, f32=0, scale=0.088, dst=2 * P, new_lens=2 * P, kept=P, dst_pages=2, budget=32, sink=4, recent=8)
    a.update({k: v for k, v in changes.items() if k in a})
    return {
        "append": lib.w4a16_kv4_append(c, b, a["q"], a["k"], a["v"], a["q_bias"], a["k_bias"], a["v_bias"], a["positions"], a["inv"], a["q_out"], a["heads"],
                                       a["q_stride"], a["kv_stride"], None),
        "read": lib.w4a16_kv4_read(c, b, a["k"], a["v"], None),
        "attention": lib.w4a16_attention_kv4(c, b, a["q"], a["out"], a["lse"], a["ws"], a["heads"], a["ws_bytes"], a["f32"], a["scale"], a["q_stride"], None),
        "weights": lib.w4a16_kv4_add_key_weights(c, b, a["q"], a["lse"], a["heads"], a["scale"], a["q_stride"], None),
        "evict": lib.w4a16_kv4_evict(c, b, a["dst"], a["new_lens"], a["kept"], a["dst_pages"], a["budget"], a["sink"], a["recent"], None),
    }


ALL = {"append", "read", "attention", "weights", "evict"}
REFUSED = [
    (dict(pages=None), -1, ALL), (dict(block_table=None), -1, ALL), (dict(seq_lens=None), -1, ALL), (dict(num_pages=0), -1, ALL),
    (dict(num_kv_heads=0), -1, ALL), (dict(num_seqs=0), -1, ALL), (dict(max_pages_per_seq=0), -1, ALL), (dict(num_tokens=0), -1, ALL),
    (dict(query_start=None), -1, ALL), (dict(page_size=8), -2, ALL), (dict(page_size=48), -2, ALL), (dict(page_size=8192), -2, ALL),
    (dict(pages=P + 8), -3, ALL), (dict(seq_lens=P + 2), -3, ALL), (dict(key_weight=P + 4), -3, ALL), (dict(num_seqs=70000), -5, ALL), (dict(num_tokens=1 << 25), -5, ALL),
    (dict(k=None), -1, {"append"}), (dict(v=None), -1, {"append"}), (dict(q_out=None), -1, {"append"}), (dict(q=None), -1, {"append", "attention", "weights"}),
    (dict(q=None, q_out=None, q_bias=P), -1, {"append", "attention", "weights"}), (dict(k=None, v=None), -1, {"append", "read"}),
    (dict(heads=0), -1, {"append", "attention", "weights"}), (dict(heads=11), -2, {"append", "attention", "weights"}),
    (dict(q_stride=-8), -1, {"append", "attention", "weights"}), (dict(q_stride=1528), -2, {"append", "attention", "weights"}),
    (dict(q_stride=1540), -3, {"append", "attention", "weights"}), (dict(kv_stride=248), -2, {"append"}), (dict(q=P + 8), -3, {"append", "attention", "weights"}),
    (dict(k=P + 2), -3, {"append", "read"}), (dict(heads=1 << 12, num_tokens=1 << 20), -5, {"append", "attention", "weights"}),
    (dict(out=None), -1, {"attention"}), (dict(scale=0.0), -1, {"attention", "weights"}), (dict(scale=float("nan")), -1, {"attention", "weights"}),
    (dict(scale=float("inf")), -1, {"attention", "weights"}), (dict(ws=None), -1, {"attention"}), (dict(ws_bytes=16), -1, {"attention"}),
    (dict(ws=P + 8), -3, {"attention"}), (dict(lse=None), -1, {"weights"}), (dict(key_weight=None), -1, {"weights", "evict"}),
    (dict(dst=None), -1, {"evict"}), (dict(dst=P), -1, {"evict"}), (dict(new_lens=P), -1, {"evict"}), (dict(max_pages_per_seq=1 << 27), -5, ALL), (dict(kept=None), -1, {"evict"}), (dict(new_lens=None), -1, {"evict"}),
    (dict(budget=0), -1, {"evict"}), (dict(sink=-1), -1, {"evict"}), (dict(sink=30), -2, {"evict"}), (dict(budget=33), -2, {"evict"}),
    (dict(sink=2147483647, recent=2147483647), -2, {"evict"}),
]


@pytest.mark.parametrize("changes,status,where", REFUSED, ids=[str(sorted(r[0].items())) for r in REFUSED])
def test_refusals(lib, changes, status, where):
    got = calls(lib, **changes)
    assert {n for n in where if got[n] == status} == where, got
    if not torch.cuda.is_available():      # what is not refused gets as far as asking for a device
        assert all(s > 0 or s == -4 for n, s in got.items() if n not in where), got


@pytest.mark.parametrize("heads", [0, 11, 12])
@pytest.mark.parametrize("kv", [5, 8])
def test_an_append_without_queries_asks_nothing_of_query_heads(lib, heads, kv):
    """Keys and values alone: 5 or 8 heads of them are no divisors of the default number of query heads, 12."""
    if torch.cuda.is_available():
        pytest.skip("the addresses would be followed")
    status = calls(lib, q=None, q_out=None, num_kv_heads=kv, heads=heads, q_stride=4)["append"]
    assert status > 0 or status == -4          # as far as asking for a device


def test_null_views_are_refused(lib):
    c, b = views()
    assert lib.w4a16_kv4_read(None, b, P, P, None) == -1 and lib.w4a16_kv4_read(c, None, P, P, None) == -1


def test_workspace_sizes(lib):
    f = lib.w4a16_attention_kv4_workspace_bytes
    assert f(0, 1, 12, 2) == -1 and f(1, 1, 12, 5) == -2 and f(1 << 25, 1, 12, 2) == -5 and f(1 << 20, 1, 1 << 12, 2) == -5
    rng = random.Random(1)
    for _ in range(500):
        kv = rng.randint(1, 16)
        heads, seqs = kv * rng.randint(1, 16), rng.randint(1, 300)
        n = f(rng.randint(1, 5000), seqs, heads, kv)
        assert 0 <= n < 1 << 31 and n % 8 == 0
    assert lib.w4a16_kv4_page_bytes(16, 2) == 16 * 2 * 136 and lib.w4a16_kv4_page_bytes(24, 2) == -2 and lib.w4a16_kv4_page_bytes(16, 0) == -1


def test_the_batch_takes_its_sizes_from_the_tensors():
    from qwen_engine_b200 import KV4Batch
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    b = KV4Batch.of(i32(3, 5), i32(3))
    assert (b.num_seqs, b.max_pages_per_seq, b.num_tokens, b.query_start) == (3, 5, 3, None)
    assert KV4Batch.of(i32(3, 5), i32(3), i32(4), num_tokens=17).num_tokens == 17
    for bad in (lambda: KV4Batch.of(i32(3, 5), i32(2)), lambda: KV4Batch.of(i32(3, 5), i32(3), i32(3), 9), lambda: KV4Batch.of(i32(3, 5), i32(3), i32(4)),
                lambda: KV4Batch.of(i32(3, 5).long(), i32(3)), lambda: KV4Batch.of(i32(5, 3).t(), i32(3))):
        with pytest.raises(ValueError):
            bad()


def test_arguments_of_the_python_functions(lib):
    from types import SimpleNamespace

    from qwen_engine_b200 import _lib, ops

    class Device:
        is_cuda = True

        def data_ptr(self):
            return P

    d = Device()
    cache = SimpleNamespace(pages=d, key_weight=d, num_pages=8, num_kv_heads=2, page_size=24)
    batch = SimpleNamespace(block_table=d, seq_lens=d, query_start=None, num_seqs=3, max_pages_per_seq=4, num_tokens=3)
    with pytest.raises(_lib.W4A16Error) as e:
        ops.attention_kv4(cache, batch, d, d, None, None, 12, 0, True, 0.1, stream=0)
    assert e.value.status == -2 and "w4a16_attention_kv4" in str(e.value)
    with pytest.raises(TypeError):
        ops.attention_kv4(cache, batch, d, d, None, None, 12, 0, True, "0.1", stream=0)
    with pytest.raises(AttributeError):
        ops.kv4_read(SimpleNamespace(pages=d), batch, d, d, stream=0)
    with pytest.raises(ValueError):
        ops.kv4_read(SimpleNamespace(pages=torch.zeros(1), key_weight=None, num_pages=8, num_kv_heads=2, page_size=16), batch, d, d, stream=0)
    with pytest.raises(OverflowError):
        ops.attention_kv4(cache, batch, d, d, None, None, 12, 1 << 70, True, 0.1, stream=0)


def sweep_create(lib, desc_changes=(), **changes):
    from qwen_engine_b200._lib import KV4BatchView, KV4CacheView, LayerWeights, QwenBinBiases, SweepDesc, SweepKV4
    layers = (LayerWeights * 2)(*[LayerWeights(*[P] * 14)] * 2)
    c = dict(pages=P, key_weight=P, num_pages=8, num_kv_heads=2, page_size=16)
    b = dict(block_table=P, seq_lens=P, query_start=None, num_seqs=1, max_pages_per_seq=4, num_tokens=1)
    kv = dict(position=P, rope_inv_freq=P, workspace=P, softmax_scale=0.088, add_key_weights=1)
    d = dict(num_layers=2, hidden=512, inter=512, q_heads=4, kv_heads=2, head_dim=128, layers=layers, workspace=P, flags=37)
    bias = changes.pop("bias", P)
    for k, v in changes.items():
        next(x for x in (c, b, kv) if k in x)[k] = v
    d.update(desc_changes)
    good = KV4CacheView(P, P, 8, 2, 16)
    caches = (KV4CacheView * 2)(good, KV4CacheView(*c.values()))       # the last layer's is the bad one
    biases = (QwenBinBiases * 2)(QwenBinBiases(None, None, None), QwenBinBiases(P, bias, P))
    pod = SweepKV4(caches, KV4BatchView(*b.values()), biases, *kv.values())
    out = ctypes.c_void_p()
    status = lib.w4a16_sweep_create_kv4(ctypes.byref(SweepDesc(*d.values())), ctypes.byref(pod), None, ctypes.byref(out))
    assert not out.value
    return status


@pytest.mark.parametrize("desc,changes,status", [
    ({}, dict(pages=None), -1), ({}, dict(num_kv_heads=4), -1), ({}, dict(key_weight=None), -1), ({}, dict(page_size=24), -2),
    ({}, dict(num_seqs=2, num_tokens=2), -1), ({}, dict(num_tokens=2), -1), ({}, dict(query_start=P), -1), ({}, dict(seq_lens=None), -1),
    ({}, dict(workspace=None), -1), ({}, dict(workspace=P + 16), -3), ({}, dict(softmax_scale=0.0), -1), ({}, dict(softmax_scale=float("nan")), -1),
    ({}, dict(position=P + 2), -3), ({}, dict(rope_inv_freq=P + 2), -3), ({}, dict(bias=P + 8), -3), (dict(head_dim=64), {}, -2),
    (dict(flags=8), {}, -2), (dict(q_heads=5), {}, -2), (dict(num_layers=0), {}, -1), (dict(q_heads=0), {}, -1), (dict(q_heads=1 << 20), {}, -5)],
    ids=str)
def test_a_sweep_with_caches_refuses(lib, desc, changes, status):
    assert sweep_create(lib, desc, **changes) == status


def test_workspace_of_a_sweep_with_caches(lib):
    f = lib.w4a16_sweep_kv4_workspace_bytes
    assert f(12, 2) >= lib.w4a16_attention_kv4_workspace_bytes(1, 1, 12, 2) + 12 * 129 * 4 and f(12, 2) % 256 == 0
    assert f(0, 1) == -1 and f(3, 2) == -2


def test_a_sweep_cache_asks_for_one_cache_a_layer():
    from qwen_engine_b200 import KV4Batch, KV4Cache, SweepCache
    cache = KV4Cache.allocate(4, device="cpu")
    batch = KV4Batch.of(torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    for bad in (SweepCache([cache], batch, 0.1), SweepCache([cache] * 2, batch, 0.1, biases=[None])):
        with pytest.raises(ValueError, match="a layer"):
            bad.pod(2, 4, 2)
    for bad in (dict(position=torch.zeros(1)), dict(position=torch.zeros(2, dtype=torch.int32)), dict(rope_inv_freq=torch.zeros(128)[::2])):
        with pytest.raises(ValueError, match="contiguous values"):
            SweepCache([cache] * 2, batch, 0.1, **bad).pod(2, 4, 2)


@pytest.mark.parametrize("version", [1, 2])
def test_the_bias_table_is_the_file_s(lib, version):
    import pathlib
    from qwen_engine_b200.qwenbin import QwenBin
    qb = QwenBin(pathlib.Path(__file__).parent / "golden" / f"tiny_w4a16_v{version}.qwenbin")
    table, (_, _, want) = qb.bias_table(qb.host_base()), qb.tensors(qb.host_base())
    assert [{n: getattr(b, n) for n, _ in b._fields_} for b in table] == want
    heads = qb.dims()["num_q_heads"] * 128
    assert all(b["q_bias"] is None or qb.host_base() <= b["q_bias"] <= qb.host_base() + qb.bytes.size - 2 * heads for b in want)


SEARCH = r"""
// The eviction's search on host arrays: per line of input a count `need` and keys; prints the key of rank `need` from the top as the
// ranges of kv4_select.hpp lead to it, how many of that key are still to be taken, and how many keys lie above it.
#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>
#include "kv4_select.hpp"
int main() {
    for (std::string line; std::getline(std::cin, line);) {
        std::istringstream in(line);
        uint32_t need, k;
        in >> need;
        std::vector<uint32_t> keys;
        while (in >> k) keys.push_back(k);
        w4::KeyRange r;
        int rounds = 0;
        while (r.first != r.last && ++rounds < 8) {
            std::vector<uint32_t> hist(w4::kEvictBins);
            for (uint32_t key : keys) {
                if (r.clamp) key = key < r.first ? r.first : key > r.last ? r.last : key;
                if (key >= r.first && key <= r.last) ++hist.at((key - r.first) >> r.shift);
            }
            int bin = w4::kEvictBins - 1;
            for (; bin > 0 && hist[bin] < need; --bin) need -= hist[bin];
            r = w4::narrowed(r, bin);
        }
        uint32_t above = 0;
        for (uint32_t key : keys) above += key > r.last;
        std::printf("%u %u %u %d\n", r.last, need, above, rounds);
    }
}
"""


def test_the_evictions_search_finds_the_key_of_a_rank(lib, tmp_path):
    """Weights around both ends of the first range (2^-32, 2^32), zeros, infinities and NaNs among them, and all over fp32: the key found is
    the one of that rank, and what is still to be taken of it makes the count whole."""
    import pathlib
    import shutil
    import subprocess

    import numpy as np
    if shutil.which("g++") is None:
        pytest.skip("g++ not on PATH")
    csrc = pathlib.Path(__file__).parents[1] / "qwen_engine_b200" / "csrc"
    (tmp_path / "search.cpp").write_text(SEARCH)
    subprocess.run(["g++", "-std=c++20", "-O1", f"-I{csrc}", "-o", str(tmp_path / "search"), str(tmp_path / "search.cpp")], check=True)
    rng = np.random.default_rng(2)

    def keys_of(w):
        u = (w.astype(np.float32) + np.float32(0)).view(np.uint32)
        k = np.where(u >> np.uint32(31), ~u, u | np.uint32(1 << 31))
        return np.where(np.isnan(w), 0, k).astype(np.uint32)

    sets = []
    for i in range(300):
        n = int(rng.integers(1, 400))
        mid = 2.0 ** [-32, 32, 0][i % 3]
        w = mid * [2.0 ** rng.uniform(-1, 1, n), rng.uniform(1.0, 1.3, n), np.exp(6 * rng.standard_normal(n))][i // 3 % 3]
        w *= rng.choice([1, 1, 1, 0, -1], n)
        if i % 5 == 0:
            w[rng.random(n) < 0.2] = rng.choice([np.inf, np.nan, -np.inf, 1e38, 1e-40])
        sets.append((keys_of(w), int(rng.integers(1, n + 1))))
    sets.append((keys_of(np.array([1.01] * 300 + [1.1] * 200 + [5.0] * 100) * 2.0 ** -32), 400))
    lines = "\n".join(" ".join(map(str, [need, *k.tolist()])) for k, need in sets)
    out = subprocess.run([str(tmp_path / "search")], input=lines + "\n", capture_output=True, text=True, check=True, timeout=60).stdout.split("\n")
    for (k, need), line in zip(sets, out):
        key, left, above, rounds = map(int, line.split())
        assert key == np.sort(k)[::-1][need - 1] and above == (k > key).sum() and above + left == need and rounds <= 4


FAKES = r"""
// The entry points (c_abi.cu) over launchers and a device that are none: what they return where one kernel cannot run.
#include <cstdio>
#include <cstring>
#include "kv4_attention.hpp"
#include "w4a16_internal.hpp"
namespace w4 {
int quantize_set_attributes() { return 0; }
int gemv_set_attributes() { return 0; }
int gemm_set_attributes() { return 0; }
int kv4_set_attributes() { return 0; }
int kv4_chunk_set_attributes() { return 200; }
int kv4_read(const Kv4View&, __half*, __half*, cudaStream_t) { return 0; }
int kv4_attention(Kv4AttentionArgs, int, bool, void*, cudaStream_t) { return 0; }
int kv4_chunk_attention(Kv4ChunkArgs, int, void*, cudaStream_t) { return 0; }
Kv4AttentionPlan kv4_attention_plan(int, int, int, int) { return {1, 1, 1, 16, 32}; }
Kv4ChunkPlan kv4_chunk_plan(int, int, int, int) { return {1, 1, 16, 32}; }
}
int main() {
    alignas(16) static char m[64];
    const w4a16_kv4_cache c{m, nullptr, 8, 1, 16};
    const w4a16_kv4_batch b{reinterpret_cast<int32_t*>(m), reinterpret_cast<int32_t*>(m), reinterpret_cast<int32_t*>(m), 1, 8, 100};
    for (int turn = 0; turn < 2; ++turn)
        std::printf("%d %d %d ", w4a16_kv4_read(&c, &b, m, m, nullptr), w4a16_attention_kv4(&c, &b, m, m, nullptr, m, 1, 64, 1, 0.1f, 0, nullptr),
                    w4a16_attention_kv4(&c, &b, m, m, nullptr, m, 1, 64, 0, 0.1f, 0, nullptr));
}
"""

RUNTIME = r"""
extern "C" {
int cudaGetDevice(int* d) { *d = 0; return 0; }
int cudaDeviceGetAttribute(int* v, int a, int) { *v = a == 75 ? 10 : 148; return 0; }      // 75: compute capability, major
int cudaGetLastError() { return 0; }
void** __cudaRegisterFatBinary(void*) { static void* p; return &p; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
}
"""


def test_a_kernel_that_cannot_run_takes_no_other_call_with_it(tmp_path):
    """The chunk form's kernel wants a register count of its compiler.  Where it does not have it, calls that take it fail, no others."""
    import pathlib
    import shutil
    import subprocess

    from qwen_engine_b200 import build
    if shutil.which("nvcc") is None:
        pytest.skip("nvcc not on PATH")
    csrc = pathlib.Path(__file__).parents[1] / "qwen_engine_b200" / "csrc"
    (tmp_path / "fakes.cu").write_text(FAKES)
    (tmp_path / "runtime.cpp").write_text(RUNTIME)
    subprocess.run([build.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++20", "-O1", "--expt-relaxed-constexpr", f"-I{csrc}", "-cudart", "none",
                    "-Xcompiler", "-fno-pie", "-Xlinker", "-no-pie,-z,lazy,--unresolved-symbols=ignore-all", "-o", str(tmp_path / "calls"),
                    str(csrc / "c_abi.cu"), str(tmp_path / "fakes.cu"), str(tmp_path / "runtime.cpp")], check=True)
    out = subprocess.run([str(tmp_path / "calls")], capture_output=True, text=True, check=True, timeout=60).stdout
    assert out.split() == ["0", "0", "200"] * 2
