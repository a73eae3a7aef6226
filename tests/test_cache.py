"""CPU-side checks of the bounded paged KV cache: the C ABI refuses bad
descriptors and arguments before it touches a GPU."""
import ctypes as C

import pytest

GOOD = dict(k_pages=4096, v_pages=8192, num_pages=10, page_tables=64, table_stride=2, weights=128, positions=256,
            slot_stride=128, rows=4, max_len=128, kv_heads=2, head_dim=128, page_size=64, state=32)


def create(**change):
    from inference_b200 import lib
    from inference_b200._lib import CacheDesc

    d = CacheDesc(**{**GOOD, **change})
    h = C.c_void_p()
    return lib().q3_cache_create(C.byref(d), 0, C.byref(h)), h


@pytest.fixture
def cache():
    from inference_b200 import lib

    status, h = create()
    assert status == 0
    yield h
    lib().q3_cache_destroy(h)


@pytest.mark.parametrize("change,status", [
    (dict(k_pages=None), 1), (dict(v_pages=None), 1), (dict(page_tables=None), 1), (dict(state=None), 1),
    (dict(k_pages=4104), 1), (dict(page_tables=66), 1), (dict(weights=130), 1), (dict(state=34), 1),
    (dict(weights=None), 1), (dict(positions=None), 1), (dict(head_dim=64), 3), (dict(page_size=16), 3),
    (dict(kv_heads=0), 1), (dict(rows=0), 1), (dict(rows=4097), 1), (dict(max_len=0), 1),
    (dict(max_len=(1 << 20) + 1), 1), (dict(max_len=129), 1), (dict(slot_stride=127), 1), (dict(num_pages=0), 1),
    (dict(num_pages=1 << 25), 1), (dict(kv_heads=1 << 20), 1),
    (dict(rows=4096, kv_heads=1024, max_len=1 << 20, table_stride=1 << 14, slot_stride=1 << 20), 1),
    (dict(rows=4096, kv_heads=17, max_len=1 << 20, table_stride=1 << 14, slot_stride=1 << 20), 1)])
def test_create_refuses(change, status):
    got, h = create(**change)
    assert got == status and not h.value


def test_the_largest_cache():
    from inference_b200 import lib

    status, h = create(rows=4096, kv_heads=16, max_len=1 << 20, table_stride=1 << 14, slot_stride=1 << 20)
    assert status == 0
    assert lib().q3_cache_attention_workspace_bytes(h, 256, 1) > 2 ** 30 * 64 * 16 * 4  # the scores alone
    assert lib().q3_cache_destroy(h) == 0


def test_create_without_weights():
    from inference_b200 import lib

    status, h = create(weights=None, positions=None, slot_stride=0)
    assert status == 0
    L, x = lib(), 1024
    assert L.q3_cache_attention(h, x, 512, x, x, 512, 4, 1, x, 1 << 40, None) == 1
    assert b"no weights" in L.q3_last_error()
    assert L.q3_cache_evict(h, x, x, 64, 0, None, None, x, x, 1 << 40, None) == 1
    L.q3_cache_destroy(h)


def append_args(h, **change):
    a = dict(c=h, q=1024, q_stride=512, k=1024, k_stride=256, v=1024, v_stride=256, q_norm=1024, k_norm=1024, cos=1024,
             sin=1024, max_pos=100, token_pos=1024, slots=1024, row_seq=None, n=4, q_heads=4, q_out=2048,
             q_out_stride=512, lens_out=None, eps=1e-6, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [
    dict(c=None), dict(q=None), dict(k=None), dict(v=None), dict(q_norm=None), dict(k_norm=None), dict(cos=None),
    dict(sin=None), dict(token_pos=None), dict(slots=None), dict(q_out=None), dict(n=5), dict(n=1 << 32),
    dict(q_heads=0), dict(q_heads=5), dict(max_pos=0), dict(q_stride=516), dict(q_stride=504), dict(k_stride=128),
    dict(v_stride=0), dict(q_out_stride=8), dict(k_norm=1028), dict(sin=1032), dict(q=1026), dict(v=1032), dict(q_out=2050)])
def test_append_refuses(cache, change):
    from inference_b200 import lib

    assert lib().q3_cache_append(*append_args(cache, **change)) == 1
    assert b"q3_cache_append" in lib().q3_last_error()


def test_append_of_nothing_is_nothing(cache):
    from inference_b200 import lib

    assert lib().q3_cache_append(*append_args(cache, n=0)) == 0
    assert lib().q3_cache_append(*append_args(cache, n=0, q=None, slots=None)) == 0


@pytest.mark.parametrize("change,status", [
    (dict(c=None), 1), (dict(q=None), 1), (dict(lens=None), 1), (dict(out=None), 1), (dict(ws=None), 1),
    (dict(ws_bytes=16), 1), (dict(ws=1032), 1), (dict(q_heads=0), 1), (dict(q_heads=3), 1), (dict(q_heads=34), 3),
    (dict(q_stride=384), 1), (dict(out_stride=516), 1), (dict(q=1026), 1), (dict(out=1032), 1)])
def test_attention_refuses(cache, change, status):
    from inference_b200 import lib

    a = dict(c=cache, q=1024, q_stride=512, lens=1024, out=1024, out_stride=512, q_heads=4, accumulate=1, ws=1024,
             ws_bytes=1 << 40, stream=None)
    a.update(change)
    assert lib().q3_cache_attention(*a.values()) == status
    assert b"q3_cache_attention" in lib().q3_last_error()


@pytest.mark.parametrize("change", [
    dict(c=None), dict(lens=None), dict(next_pos=None), dict(lens_out=None), dict(keep=0), dict(recent=1 << 31),
    dict(weights_out=4096), dict(positions_out=4096), dict(weights_out=4098, positions_out=4096), dict(ws=None),
    dict(ws_bytes=0), dict(ws=1025), dict(weights_out=128, positions_out=4096)])
def test_evict_refuses(cache, change):
    from inference_b200 import lib

    a = dict(c=cache, lens=1024, next_pos=1024, keep=64, recent=8, weights_out=None, positions_out=None, lens_out=1024,
             ws=1024, ws_bytes=1 << 40, stream=None)
    a.update(change)
    assert lib().q3_cache_evict(*a.values()) == 1
    assert b"q3_cache_evict" in lib().q3_last_error()


def test_workspace_sizes(cache):
    from inference_b200 import lib

    L = lib()
    sizes = [L.q3_cache_attention_workspace_bytes(cache, qh, 1) for qh in (2, 4, 16, 32)]
    assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
    assert all(0 < L.q3_cache_attention_workspace_bytes(cache, qh, 0) <= n for qh, n in zip((2, 4, 16, 32), sizes))
    assert L.q3_cache_attention_workspace_bytes(cache, 3, 1) == 0
    assert L.q3_cache_attention_workspace_bytes(cache, 34, 1) == 0
    assert L.q3_cache_attention_workspace_bytes(None, 4, 1) == 0
    assert L.q3_cache_evict_workspace_bytes(cache, 64) > 0 and L.q3_cache_evict_workspace_bytes(cache, 1 << 40) > 0
    assert L.q3_cache_evict_workspace_bytes(cache, 0) == 0 and L.q3_cache_evict_workspace_bytes(None, 5) == 0


def test_sync_and_destroy_of_nothing():
    from inference_b200 import lib

    assert lib().q3_cache_sync(None, None) == 1
    assert lib().q3_cache_destroy(None) == 0


def test_python_handle_refuses_cpu_tensors():
    import torch

    from inference_b200 import PagedCache

    k = torch.zeros(2, 1, 64, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        PagedCache(k, k.clone(), torch.zeros(1, 1, dtype=torch.int32))


def test_work_shares(tmp_path):
    """The shares of the attention's work, from lengths in any state, against a walk over every tile."""
    import os
    import subprocess

    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cache_plan_check.cpp")
    exe = str(tmp_path / "cache_plan_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-o", exe, src], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_lengths_are_read_through_the_callers_reader(tmp_path):
    """The look-up of a tile with a reader of lengths: the same places as from the array, no other reads."""
    import os
    import subprocess

    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cache_lens_check.cpp")
    exe = str(tmp_path / "cache_lens_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-o", exe, src], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_a_cache_learns_of_every_stream_that_uses_it():
    """The state words belong to the library: a call on a stream that the allocator does not know yet tells it, once a stream."""
    import torch

    from inference_b200 import B200Backend

    class Cache:
        device, h, _streams, told = torch.device("cuda", 0), 1, {5}, []

        def _used_on(self, stream):
            self.told.append(stream)
            self._streams.add(stream)

    be, cache = B200Backend(0), Cache()
    for stream in (5, 7, 7, 5, 9):
        be._raw_stream = lambda index: stream
        assert be._cache_call(cache)[1:] == (0, stream)
    assert cache.told == [7, 9]
