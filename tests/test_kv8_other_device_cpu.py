"""The paged cache's calls for tensors of a device that is not the current one are made there, with the arguments that they were
given. (Devices and the library are stood in for: no GPU takes part.)"""
import contextlib
import inspect

import pytest
import torch

from larder_b200 import kv8, ops

SHAPE = (4, 2, 2, 16, 64)


@pytest.fixture
def devices(monkeypatch):
    """The current device is 0, all tensors are on 1; `seen` lists the devices that calls were made on."""
    at, seen = [0], []

    @contextlib.contextmanager
    def device(d):
        was, at[0] = at[0], d
        yield
        at[0] = was

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "_device", lambda: at[0])
    monkeypatch.setattr(ops, "_kv8_pool", lambda pages, scales, table, what: (SHAPE, (1, 3), 1))
    return at, seen


class There(torch.Tensor):
    """A tensor that says it is on device 1."""

    @staticmethod
    def of(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype).as_subclass(There)

    def get_device(self):
        return 1


def i32(*shape):
    return There.of(*shape, dtype=torch.int32)


def test_each_call_is_made_on_its_tensors_device(devices, monkeypatch):
    at, seen = devices

    class Library:
        def __getattr__(self, name):
            if name.endswith("_size"):
                return lambda *a: 0
            return lambda *a: seen.append((name, at[0])) or 0

    monkeypatch.setattr(ops, "lib", Library)
    monkeypatch.setattr(ops, "_stream_of", lambda dev: 0)
    monkeypatch.setattr(ops, "_scratch", lambda n, stream: 0)
    monkeypatch.setattr(ops, "_scratch_done", lambda ptr: None)
    pages, scales = There.of(*SHAPE, dtype=torch.uint8).view(torch.float8_e4m3fn), There.of(*SHAPE[:3])
    x = There.of(1, 2, 3, 64)
    ops.kv8_append(pages, scales, x, x, i32(1, 3), i32(1))
    out = There.of(1, 2, 3, 64)
    assert ops.kv8_attend(x, pages, scales, i32(1, 3), i32(1), 0.1, True, out) is out
    assert ops.kv8_attend_packed(x, pages, scales, i32(1, 3), i32(1), i32(2), 0.1, True, out) is out
    ops.kv8_copy(pages, scales, i32(1), i32(1))
    ops.kv8_compact(pages, scales, i32(1, 3), i32(2), i32(2), i32(1, 1), i32(1))
    assert seen == [("lb2_" + n, 1) for n in ("kv8_append", "kv8_attend", "kv8_attend_packed", "kv8_copy", "kv8_compact")]
    assert at[0] == 0


@pytest.mark.parametrize("name", ["kv8_append", "kv8_attend", "kv8_attend_packed", "kv8_compact"])
def test_the_arguments_go_along(devices, monkeypatch, name):
    def elsewhere(dev, call, *args):
        return dev, call, args

    monkeypatch.setattr(ops, "_elsewhere", elsewhere)
    call = getattr(ops, name)
    given = [object() for _ in inspect.signature(call).parameters]
    assert call(*given) == (1, call, tuple(given))


def test_a_cache_on_another_device_appends_and_attends_there(devices, monkeypatch):
    at, seen = devices
    cache = kv8.Cache(4, 16, 2, 64, device="cpu")
    a = cache.add()
    step = cache.step([a], [3])
    monkeypatch.setattr(ops, "_elsewhere", lambda dev, call, *args: seen.append((dev, call.__name__)))
    cache.append(step, torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, 3, 64))
    cache.attend(step, torch.zeros(1, 4, 3, 64), 0.1)
    cache.attend(step, torch.zeros(1, 4, 3, 64), 0.1, packed=True)
    assert seen == [(1, "kv8_append"), (1, "kv8_attend"), (1, "kv8_attend_packed")]
