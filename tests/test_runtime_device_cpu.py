"""A handle knows its device from the library: making one asks nothing of torch, which may be absent or unable to use
the GPU."""
import torch

from lpta import _native


class Library:
    """Stands in for libtl_int8.so: a handle on device 3."""

    def tl_create(self, cfg, max_seqs, out):
        out._obj.value = 4096
        return _native.TL_OK

    def tl_get_device(self, h, out):
        assert h.value == 4096
        out._obj.value = 3
        return _native.TL_OK

    def tl_sync(self, h):
        return _native.TL_OK

    def tl_destroy(self, h):
        pass


def test_runtime_without_torchs_gpu(monkeypatch):
    def refuse(*_):
        raise AssertionError("Torch not compiled with CUDA enabled")
    monkeypatch.setattr(_native, "load_library", Library)
    for name in ("current_device", "is_available", "init", "_lazy_init", "device_count"):
        monkeypatch.setattr(torch.cuda, name, refuse)
    rt = _native.Runtime(dict(hidden=64, intermediate=64, n_layers=1, n_heads=1, n_kv_heads=1, head_dim=64, vocab=64,
                              max_pos=64, rms_eps=1e-5, rope_theta=10000.0))
    assert rt.device == 3
    rt.call("tl_sync")
    rt.close()
