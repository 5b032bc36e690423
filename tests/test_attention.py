"""What the attention calls refuse before any launch, the rotation's table, and what they pass on (no GPU)."""
import ctypes
import math

import pytest
import torch

from ishizuki_amd import _bind, _lib, attention

P = ctypes.c_void_p(4096)
POOL = dict(k=P, v=P, ks=P, vs=P, format=0, blocks=4, heads=2, dim=128)


def rope(dtype=1, rows=1, dim=128, rot=128, q=P, q_row=512, q_head=128, q_heads=4, positions=P, turns=P, out=P):
    return _lib.lib().ishz_norm_rope(q, q_row, q_head, q_heads, P, 512, 128, 2, dtype, rows, dim, positions, turns, rot, 0,
                                     1.0, None, None, 1e-6, out, P, None)


def append(pool=POOL, dtype=1, rows=1, k=P, k_row=512, table=P, width=4, lengths=P, sequences=1, max_rows=1, q=P, q_heads=0,
           rot=0, q_out=P, **changed):
    return _lib.lib().ishz_kv_append(k, k_row, 128, P, 512, 128, dtype, rows, *{**pool, **changed}.values(), table, width,
                                     lengths, P, sequences, max_rows, q, 512, 128, q_heads, P, P, rot, 0, 1.0, None, None,
                                     1e-6, q_out, None)


def read(pool=POOL, dtype=1, width=4, lengths=P, sequences=1, tail=1, k_out=P, **changed):
    return _lib.lib().ishz_kv_read(*{**pool, **changed}.values(), P, width, lengths, sequences, tail, dtype, k_out, P, None)


def attend(pool=POOL, dtype=1, rows=1, q=P, q_row=512, q_heads=4, width=4, lengths=P, sequences=1, max_rows=1,
           max_length=256, causal=1, window=0, out=P, ws=None, ws_bytes=0, **changed):
    return _lib.lib().ishz_kv_attend(q, q_row, 128, q_heads, dtype, rows, *{**pool, **changed}.values(), P, width, lengths, P,
                                     sequences, max_rows, max_length, 1.0, causal, window, out, ws, ws_bytes, None)


@pytest.mark.parametrize("call", [append, read, attend])
@pytest.mark.parametrize("changed,status", [
    (dict(dtype=3), _lib.DECLINED), (dict(dtype=-1), _lib.DECLINED), (dict(format=2), _lib.DECLINED),
    (dict(dim=96), _lib.DECLINED), (dict(dim=0), _lib.DECLINED), (dict(width=1 << 26), _lib.DECLINED),
    (dict(blocks=0), _lib.EINVAL), (dict(heads=0), _lib.EINVAL), (dict(k=None), _lib.EINVAL), (dict(vs=None), _lib.EINVAL),
    (dict(ks=ctypes.c_void_p(4098)), _lib.EINVAL), (dict(lengths=None), _lib.EINVAL), (dict(sequences=-1), _lib.EINVAL),
    (dict(width=-1), _lib.EINVAL)])
def test_pool_and_sequences(call, changed, status):
    if "k" in changed and call is append:
        changed = {"pool": {**POOL, "k": None}}
    assert call(**changed) == status, _lib.last_error()


def test_cache_codes_must_be_aligned():
    assert read(v=ctypes.c_void_p(4100)) == _lib.EINVAL
    assert attend(v=ctypes.c_void_p(4104)) == _lib.EINVAL


@pytest.mark.parametrize("changed,status", [
    (dict(dtype=4), _lib.DECLINED), (dict(dim=192), _lib.DECLINED), (dict(rot=24), _lib.DECLINED), (dict(rot=144), _lib.DECLINED),
    (dict(rot=-16), _lib.DECLINED), (dict(q_row=516), _lib.DECLINED), (dict(q_head=2), _lib.DECLINED),
    (dict(q=ctypes.c_void_p(4104)), _lib.DECLINED), (dict(q=None), _lib.EINVAL), (dict(out=None), _lib.EINVAL),
    (dict(positions=None), _lib.EINVAL), (dict(turns=None), _lib.EINVAL), (dict(rows=-1), _lib.EINVAL),
    (dict(q_heads=-1), _lib.EINVAL)])
def test_norm_rope(changed, status):
    assert rope(**changed) == status, _lib.last_error()


@pytest.mark.parametrize("changed,status", [
    (dict(rot=8), _lib.DECLINED), (dict(k_row=511), _lib.DECLINED), (dict(max_rows=1 << 30, rows=1 << 30), _lib.DECLINED),
    (dict(k=None), _lib.EINVAL), (dict(q=None, q_heads=4), _lib.EINVAL), (dict(q_out=None, q_heads=4), _lib.EINVAL),
    (dict(max_rows=-1), _lib.EINVAL), (dict(table=None), _lib.EINVAL)])
def test_append(changed, status):
    assert append(**changed) == status, _lib.last_error()


@pytest.mark.parametrize("changed,status", [
    (dict(tail=(1 << 31) - 1), _lib.DECLINED), (dict(tail=-1), _lib.EINVAL), (dict(k_out=None), _lib.EINVAL),
    (dict(k_out=ctypes.c_void_p(8)), _lib.EINVAL)])
def test_read(changed, status):
    assert read(**changed) == status, _lib.last_error()


@pytest.mark.parametrize("changed,status", [
    (dict(dtype=0), _lib.DECLINED), (dict(q_row=510), _lib.DECLINED), (dict(rows=1 << 30, max_rows=1 << 30), _lib.DECLINED),
    (dict(q_heads=3), _lib.EINVAL), (dict(q_heads=0), _lib.EINVAL), (dict(window=-1), _lib.EINVAL),
    (dict(window=5, causal=0), _lib.EINVAL), (dict(max_length=-1), _lib.EINVAL), (dict(q=None), _lib.EINVAL),
    (dict(out=None), _lib.EINVAL), (dict(max_length=1 << 20), _lib.EINVAL), (dict(max_length=1 << 20, ws=P, ws_bytes=64), _lib.EINVAL),
    (dict(max_length=1 << 20, ws=ctypes.c_void_p(4100), ws_bytes=1 << 30), _lib.EINVAL)])
def test_attend(changed, status):
    assert attend(**changed) == status, _lib.last_error()


def test_nothing_to_do():
    assert rope(rows=0) == rope(q_heads=0, rows=0) == append(rows=0) == read(sequences=0) == read(tail=0) == _lib.OK
    assert attend(rows=0) == attend(sequences=0) == attend(max_rows=0) == _lib.OK


def test_workspace():
    size = _lib.lib().ishz_kv_attend_workspace_size
    assert size(1, 32, 8, 128, 1, 1, 64) == 0  # one block is not split
    assert size(0, 32, 8, 128, 1, 1, 64) == size(1, 0, 8, 128, 1, 1, 64) == size(1, 32, 8, 128, 0, 1, 64) == 0
    one = size(1, 32, 8, 128, 1, 1, 1 << 16)
    assert one > 0 and one % (32 * (128 + 2) * 4) == 0  # fp32 sums, a maximum and a total for each split and head


def test_turns():
    """The table's fractions give each position's angle to 2^-40 turns at positions where fp32 has lost it."""
    t = attention.turns(64, base=1e6, device="cpu")
    for position in (1, 131071, 1000003, 2 ** 31 - 1, -5):
        for i, bits in enumerate(t.tolist()):
            exact = math.fmod(position * 1e6 ** (-2.0 * i / 64) / (2 * math.pi), 1.0)
            got = (position * bits % (1 << 64)) / 2.0 ** 64
            off = abs(got - exact) % 1.0
            assert min(off, 1 - off) < (2.0 ** -20 if position == 2 ** 31 - 1 else 2.0 ** -30)
    assert torch.equal(attention.turns(inv_freq=[1.0, 0.5], device="cpu"), attention.turns(inv_freq=torch.tensor([1.0, 0.5]), device="cpu"))


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_size"):
                return 256
            self.calls.append((name, args))
            return _lib.OK
        return call


@pytest.fixture
def library(monkeypatch):
    lib = Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(attention, "require_cuda", lambda *ts: None)
    monkeypatch.setattr(attention, "stream", lambda: None)
    return lib


def batch(rows=3):
    i32 = dict(dtype=torch.int32)
    return attention.Batch(torch.zeros(1, 2, **i32), torch.tensor([rows], **i32), torch.tensor([0, rows], **i32), rows, rows)


def test_shapes_that_do_not_fit_are_refused(library):
    cache = attention.new_cache(2, 2, 128, device="cpu")
    x = torch.zeros(3, 2, 128, dtype=torch.float16)
    bad = [lambda: attention.attend(torch.zeros(3, 2, 64, dtype=torch.float16), cache, batch()),
           lambda: attention.append(x, x[:2], cache, batch()),
           lambda: attention.append(x, x.float(), cache, batch()),
           lambda: attention.append(x[:, :1], x[:, :1], cache, batch()),
           lambda: attention.append(x, x, cache, batch(), q=x[:2]),
           lambda: attention.append(x, x, cache, batch(), turns=attention.turns(128, device="cpu")),
           lambda: attention.append(x, x, cache, batch(), turns=torch.zeros(32), positions=torch.zeros(3, dtype=torch.int32)),
           lambda: attention.append(x, x, cache, batch(), k_weight=torch.ones(128, dtype=torch.float16)),
           lambda: attention.append(x, x, cache, batch(), k_weight=torch.ones(32)),
           lambda: attention.append(x, x, cache._replace(v=cache.k), batch()),
           lambda: attention.append(x, x, cache._replace(k_scale=cache.k_scale.half()), batch()),
           lambda: attention.read(cache._replace(v_scale=cache.v_scale[:1]), batch()),
           lambda: attention.read(cache, batch(), tail=-1),
           lambda: attention.attend(x, cache, batch()._replace(starts=torch.zeros(3, dtype=torch.int32))),
           lambda: attention.attend(x, cache, batch()._replace(lengths=torch.zeros(1))),
           lambda: attention.attend(x, cache, batch()._replace(table=torch.zeros(2, 2, dtype=torch.int32))),
           lambda: attention.attend(x[0], cache, batch()),
           lambda: attention.norm_rope(x, x[:2]),
           lambda: attention.new_cache(2, 2, 64, dtype=torch.float16, device="cpu")]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert library.calls == []


def test_strides_are_passed_and_odd_ones_copied(library):
    cache = attention.new_cache(2, 2, 64, device="cpu")
    qkv = torch.zeros(3, 8, 64, dtype=torch.float16)
    attention.append(qkv[:, 4:6], qkv[:, 6:], cache, batch(), q=qkv[:, :4])
    args = library.calls[-1][1]
    assert args[0] == qkv.data_ptr() + 2 * 4 * 64 and args[1:3] == (512, 64) and args[4:6] == (512, 64)
    assert args[22] == qkv.data_ptr() and args[23:26] == (512, 64, 4)
    odd = torch.zeros(3, 2, 65, dtype=torch.float16)[..., 1:]
    attention.attend(odd, cache, batch())
    args = library.calls[-1][1]
    assert args[0] % 16 == 0 and args[1:3] == (128, 64)


def test_binding_leaves_what_does_not_fit():
    """Without a GPU nothing fits: the compiled calls hand every call over, and raise nothing."""
    x = torch.zeros(3, 2, 64, dtype=torch.float16)
    cache = attention.new_cache(2, 2, 64, device="cpu")
    for out in (_bind.norm_rope(x, x, None, None, None, None, 1e-6, False, 1.0), _bind.norm_rope(x), _bind.norm_rope(*[None] * 9),
                _bind.attend(x, cache, batch(), None, True, 0), _bind.attend("q", (), 3, None, True, 0), _bind.read(cache, batch(), -1, torch.float16),
                _bind.append(x, x, cache, batch(), None, None, None, None, None, 1e-6, False, 1.0), _bind.append()):
        assert out is NotImplemented


@pytest.mark.parametrize("rows,heads,width,first", [(1, 4, 771, 0), (1, 1, 780, 64), (3, 1, 776, 0), (1, 2, 132, 1), (3, 2, 136, 0)])
def test_strides_of_single_rows_and_heads(library, rows, heads, width, first):
    """A slice of one row or head keeps strides that nothing goes by: odd ones are neither passed on nor a reason to decline."""
    cache = attention.new_cache(2, heads, 64, device="cpu")
    wide = torch.zeros(rows + 1, width, dtype=torch.float16)
    slices = [wide[:, first:first + 64 * heads].unflatten(1, (heads, 64))[:rows]]
    if heads == 1:
        slices += [torch.zeros(rows + 1, 3, 65, dtype=torch.float16)[:rows, at:at + 1, at:at + 64] for at in (0, 1)]
    for x in slices:
        attention.attend(x, cache, batch(rows))
        attention.norm_rope(x, x)
        attention.append(x, x, cache, batch(rows), q=x)
        assert len(library.calls) == 3
        for name, args in library.calls:
            for i in {"ishz_kv_attend": [0], "ishz_norm_rope": [0, 4], "ishz_kv_append": [0, 3, 22]}[name]:
                assert args[i] % 16 == 0 and args[i + 1] % 8 == 0 and args[i + 2] % 8 == 0
                if rows > 1 and x.stride(0) % 8 == 0:
                    assert args[i:i + 2] == (x.data_ptr(), x.stride(0))  # not copied
        library.calls.clear()


def test_launches_of_too_many_threads_are_declined():
    """A launch holds fewer than 2^32 threads, of 256 or 512 a workgroup."""
    tall = dict(heads=8, q_heads=64, sequences=4096, max_rows=8192, rows=8192 + 4095, max_length=8192)  # tiles of 512 threads
    assert attend(**tall) == _lib.DECLINED, _lib.last_error()
    many = dict(heads=8, q_heads=32, sequences=1 << 20, rows=1 << 20, max_length=640)  # eight waves
    assert attend(**many) == _lib.DECLINED, _lib.last_error()
    assert rope(rows=1 << 26) == rope(rows=(1 << 31) - 1) == _lib.DECLINED, _lib.last_error()
    assert append(rows=(1 << 31) - 1, max_rows=(1 << 31) - 1) == _lib.DECLINED, _lib.last_error()
    assert rope(q_heads=(1 << 31) - 1) == _lib.DECLINED, _lib.last_error()


def test_lengths_without_a_bound_are_split():
    """max_length may be as large as a host number gets: rows that take tiles are split as for any long cache."""
    size = _lib.lib().ishz_kv_attend_workspace_size
    assert size(70, 4, 1, 128, 1, 70, (1 << 31) - 1) == size(70, 4, 1, 128, 1, 70, 1 << 30) > 0
