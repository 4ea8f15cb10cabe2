"""Who owns and prepares the memory of the key/value caches and of attention (no GPU needed)."""
import pytest

from mlxl3_b200 import decoder, kv


@pytest.mark.parametrize("bits,buffers", [(16, 2), (8, 4), (4, 4)])
def test_a_new_cache_is_zeroed_when_its_constructor_returns(monkeypatch, bits, buffers):
    """Streams of the library do not wait for the default stream, on which the pool is zeroed: the constructor has to."""
    log = []

    class Buffer:
        def __init__(self, nbytes):
            self.nbytes, self.ptr = nbytes, 4096 * (len(log) + 1)
            log.append("new")

        def fill(self, byte):
            log.append("fill")

    class Stream:
        handle = None

        def sync(self):
            log.append("sync")
    monkeypatch.setattr(kv, "DeviceBuffer", Buffer)
    monkeypatch.setattr(kv, "DEFAULT_STREAM", Stream())
    cache = kv.KvCache(3, 16, 2, 64, bits=bits)
    assert log.count("new") == log.count("fill") == buffers and "sync" in log[len(log) - 1 - log[::-1].index("fill"):]
    assert [b.nbytes for b in cache._owned] == [3 * 2 * 16 * 64 * bits // 8] * 2 + [3 * 2 * 16 * 4] * (buffers - 2)
    del log[:]
    kv.KvCache(3, 16, 2, 64, d_k=4096, d_v=8192)
    assert not log


def test_a_new_attention_workspace_is_zeroed_when_the_function_returns(monkeypatch):
    log = []

    class Buffer:
        def __init__(self, nbytes):
            log.append("new")

        def fill(self, byte):
            log.append("fill")

    class Stream:
        handle = None

        def sync(self):
            log.append("sync")
    monkeypatch.setattr(decoder, "DeviceBuffer", Buffer)
    monkeypatch.setattr(decoder, "DEFAULT_STREAM", Stream())
    decoder.new_attention_workspace(32, 8)
    assert log == ["new", "fill", "sync"]
