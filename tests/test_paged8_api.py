"""The rotary, slot map and 8-bit cache operators on the CPU: dispatch signatures, refusals,
frequencies, the call cache and the C entry points' checks of arguments."""

from __future__ import annotations

import ctypes
import math

import pytest

from fakes import FakeDevice, FakeTensor, FakeTorch
from radeon_kernels import _native, rotary_frequencies
from radeon_kernels.ops._frontend import quick_call, remember_call
from radeon_kernels.ops.paged_cache_8bit.api import _execute_append, _execute_attention
from radeon_kernels.ops.paged_slots.api import _execute as execute_slots
from radeon_kernels.ops.rotary.api import _execute as execute_rotary


class Torch(FakeTorch):
    float64 = "float64"
    float32 = "float32"
    float8_e4m3fn = "float8_e4m3fn"
    int8 = "int8"


class Capture:
    def __init__(self, result=("a", "b")):
        self.call = None
        self.result = result

    def execute(self, **kwargs):
        self.call = kwargs
        return self.result


def T(shape, dtype="bfloat16", **kwargs):
    return FakeTensor(shape, dtype=dtype, **kwargs)


def _rotary_args():
    return dict(query=T((7, 8, 128)), key=T((7, 2, 128)), positions=T((7,), "int64"), frequencies=T((32,), "float64"),
                interleaved=False, amplitude=1.0)


def _slots_args():
    return dict(block_tables=T((4, 9), "int32"), context_lengths=T((4,), "int32"), new_lengths=T((4,), "int32"),
                free_blocks=T((20,), "int32"), num_tokens=6, block_size=16)


def _cache_args(kind="float8_e4m3fn"):
    return dict(key_cache=T((10, 16, 2, 128), kind), value_cache=T((10, 16, 2, 128), kind),
                key_scales=T((10, 2), "float32"), value_scales=T((10, 2), "float32"))


def _append_args(kind="float8_e4m3fn"):
    return dict(key=T((5, 2, 128)), value=T((5, 2, 128)), **_cache_args(kind), slot_mapping=T((5,), "int64"))


def _attention_args(kind="float8_e4m3fn"):
    return dict(query=T((3, 8, 128)), **_cache_args(kind), block_tables=T((3, 4), "int32"),
                context_lengths=T((3,), "int32"), scale=None)


EXECUTE = {"rotary": (execute_rotary, _rotary_args), "slots": (execute_slots, _slots_args),
           "append": (_execute_append, _append_args), "attention": (_execute_attention, _attention_args)}


def call(name, **changes):
    execute, arguments = EXECUTE[name]
    runtime = Capture("out" if name == "attention" else ("a", "b"))
    result = execute(**{**arguments(), **changes}, torch_module=Torch(), runtime=runtime)
    return runtime.call, result


def test_signatures_name_what_the_choice_depends_on():
    got, result = call("rotary")
    assert result == ("a", "b") and got["operator"] == "rotary_embedding" and got["semantic_version"] == "1.0"
    assert got["signature"] == {
        "dtype": "bf16", "query_heads": 8, "kv_heads": 2, "head_dim": 128, "rotary_dim": 64, "pairing": "halves",
        "index_dtype": "int64", "requires_grad": False,
    }
    assert got["native_arguments"][4:] == (False, 1.0) and got["fallback_selected"] == "cuda/rotary_embedding"
    got, _ = call("rotary", query=T((7, 8, 128), requires_grad=True), interleaved=True, amplitude=2)
    assert got["signature"]["requires_grad"] is True and got["signature"]["pairing"] == "interleaved"
    assert got["native_arguments"][4:] == (True, 2.0)
    got, _ = call("slots")
    assert got["signature"] == {"index_dtype": "int32", "block_size": 16, "contiguous": True}
    assert got["native_arguments"][-2:] == (6, 16) and got["fallback_selected"] == "cuda/paged_slots"
    got, _ = call("append")
    assert got["signature"] == {
        "dtype": "bf16", "cache_dtype": "e4m3", "kv_heads": 2, "head_dim": 128, "block_size": 16, "index_dtype": "int64",
        "cache_layout": "block_slot_head_dim", "requires_grad": False,
    }
    got, result = call("attention", **_cache_args("int8"), scale=2)
    assert result == "out" and got["signature"] == {
        "dtype": "bf16", "cache_dtype": "int8", "query_heads": 8, "kv_heads": 2, "head_dim": 128, "block_size": 16,
        "index_dtype": "int32", "cache_layout": "block_slot_head_dim", "scale_mode": "explicit", "contiguous": True,
        "requires_grad": False,
    }
    assert got["native_arguments"][-1] == 2.0
    got, _ = call("attention")
    assert got["native_arguments"][-1] == pytest.approx(128**-0.5) and got["signature"]["scale_mode"] == "default"


other = FakeDevice(1)
REFUSALS = [
    ("rotary", dict(query=3), TypeError, "query must be a PyTorch tensor"),
    ("rotary", dict(query=T((7, 8))), ValueError, "query must be rank 3"),
    ("rotary", dict(key=T((7, 2, 128), "float16")), TypeError, "same dtype"),
    ("rotary", dict(query=T((7, 8, 128), "float32")), TypeError, "supports torch.float16 and torch.bfloat16"),
    ("rotary", dict(key=T((6, 2, 128))), ValueError, "share tokens and head_dim"),
    ("rotary", dict(key=T((7, 2, 64))), ValueError, "share tokens and head_dim"),
    ("rotary", dict(positions=T((6,), "int64")), ValueError, "one position per token"),
    ("rotary", dict(positions=T((7,), "float64")), TypeError, "int32 or torch.int64"),
    ("rotary", dict(positions=T((7,), "int64", device=other)), ValueError, "same device"),
    ("rotary", dict(frequencies=T((65,), "float64")), ValueError, "1 to head_dim // 2 pairs"),
    ("rotary", dict(frequencies=T((0,), "float64")), ValueError, "1 to head_dim // 2 pairs"),
    ("rotary", dict(frequencies=T((32,), "float32")), TypeError, "torch.float64"),
    ("rotary", dict(frequencies=T((32, 1), "float64")), ValueError, "rank 1"),
    ("rotary", dict(frequencies=[0.1]), TypeError, "frequencies must be a PyTorch tensor"),
    ("rotary", dict(frequencies=T((32,), "float64", requires_grad=True)), ValueError, "must not require gradients"),
    ("rotary", dict(interleaved=1), TypeError, "interleaved must be bool"),
    ("rotary", dict(amplitude=True), TypeError, "amplitude must be a number"),
    ("rotary", dict(amplitude=math.nan), ValueError, "amplitude must be finite"),
    ("rotary", dict(query=T((7, 0, 128))), ValueError, "head counts"),
    ("rotary", dict(query=T((7, 8, 2048)), key=T((7, 2, 2048))), ValueError, "head_dim must be at most 1024"),
    ("slots", dict(context_lengths=T((3,), "int32")), ValueError, "one length per row"),
    ("slots", dict(new_lengths=T((4,), "int64")), TypeError, "same dtype"),
    ("slots", dict(free_blocks=T((20,), "int32", device=other)), ValueError, "same device"),
    ("slots", dict(block_tables=T((0, 9), "int32"), context_lengths=T((0,), "int32"), new_lengths=T((0,), "int32")),
     ValueError, "dimensions must be positive"),
    ("slots", dict(num_tokens=-1), ValueError, "num_tokens must be in"),
    ("slots", dict(num_tokens=2**31), ValueError, "num_tokens must be in"),
    ("slots", dict(num_tokens=2.0), TypeError, "num_tokens must be an int"),
    ("slots", dict(block_size=0), ValueError, "block_size must be positive"),
    ("slots", dict(block_size=True), TypeError, "block_size must be an int"),
    ("slots", dict(block_size=2**30), ValueError, "below 2"),
    ("slots", dict(block_tables=T((4, 9), "int32", contiguous=False)), ValueError, "contiguous"),
    ("append", dict(key=T((5, 2, 128), "float16")), TypeError, "same dtype"),
    ("append", dict(value=T((4, 2, 128))), ValueError, "same shape"),
    ("append", dict(key=T((5, 3, 128)), value=T((5, 3, 128))), ValueError, "must match the cache"),
    ("append", dict(key_cache=T((10, 16, 2, 128), "bfloat16")), TypeError, "float8_e4m3fn or torch.int8"),
    ("append", dict(value_cache=T((10, 16, 2, 128), "int8")), TypeError, "same dtype"),
    ("append", dict(value_cache=T((10, 8, 2, 128), "float8_e4m3fn")), ValueError, "same shape"),
    ("append", dict(key_scales=T((10, 2), "float64")), TypeError, "torch.float32"),
    ("append", dict(value_scales=T((2, 10), "float32")), ValueError, "[num_blocks, kv_heads]"),
    ("append", dict(slot_mapping=T((6,), "int64")), ValueError, "one slot per token"),
    ("append", dict(slot_mapping=T((5,), "int8")), TypeError, "int32 or torch.int64"),
    ("append", dict(key_cache=T((10, 16, 2, 128), "float8_e4m3fn", contiguous=False)), ValueError, "contiguous"),
    ("append", dict(key=T((5, 2, 128), requires_grad=True)), ValueError, "inference-only"),
    ("append", dict(**{**_cache_args(), "key_cache": T((10, 2048, 2, 128), "int8"),
                       "value_cache": T((10, 2048, 2, 128), "int8")}), ValueError, "block_size must be at most 1024"),
    ("append", dict(slot_mapping=T((5,), "int64", device=other)), ValueError, "same device"),
    ("append", (lambda a: dict(value_cache=a["key_cache"], key_cache=a["key_cache"]))(_cache_args()), ValueError,
     "caches and scales of their own"),
    ("append", (lambda a: dict(value_scales=a["key_scales"], key_scales=a["key_scales"]))(_cache_args()), ValueError,
     "caches and scales of their own"),
    ("attention", dict(query=T((3, 8))), ValueError, "query must be rank 3"),
    ("attention", dict(query=T((3, 7, 128))), ValueError, "divisible by kv_heads"),
    ("attention", dict(query=T((3, 8, 64))), ValueError, "head_dim must match cache"),
    ("attention", dict(block_tables=T((2, 4), "int32")), ValueError, "block_tables must have shape"),
    ("attention", dict(block_tables=T((3, 4), "int64")), TypeError, "same dtype"),
    ("attention", dict(context_lengths=T((4,), "int32")), ValueError, "one length per sequence"),
    ("attention", dict(block_tables=T((3, 2**27), "int32")), ValueError, "below 2"),
    ("attention", dict(query=T((3, 8, 128), contiguous=False)), ValueError, "must be contiguous"),
    ("attention", dict(key_scales=T((10, 2), "float32", requires_grad=True)), ValueError, "inference-only"),
    ("attention", dict(scale=0.0), ValueError, "scale must be positive"),
    ("attention", dict(scale=True), TypeError, "scale must be a number"),
    ("attention", dict(key_scales=T((10, 2), "float32", device=other)), ValueError, "same device"),
    ("attention", dict(query=T((3, 8, 128), device=other)), ValueError, "same device"),
]


@pytest.mark.parametrize("name, changes, error, message", REFUSALS, ids=[f"{r[0]}-{i}" for i, r in enumerate(REFUSALS)])
def test_refusals(name, changes, error, message):
    with pytest.raises(error) as caught:
        call(name, **changes)
    assert message in str(caught.value)


def test_frequencies():
    plain = rotary_frequencies(8, base=100.0, device="cpu").tolist()
    assert plain == pytest.approx([100.0 ** (-i / 4) for i in range(4)], rel=1e-15)
    assert rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu").tolist() == pytest.approx(
        [f / 4 for f in rotary_frequencies(8, device="cpu").tolist()], rel=1e-15)
    stretched, base = rotary_frequencies(64, scaling="ntk", factor=8.0, device="cpu"), rotary_frequencies(64, device="cpu")
    assert stretched[0] == 1.0 and (base[-1] / stretched[-1]).item() == pytest.approx(8.0, rel=1e-12)
    yarn = rotary_frequencies(128, scaling="yarn", factor=16.0, original_length=4096, device="cpu")
    ratio = (rotary_frequencies(128, device="cpu") / yarn).tolist()
    turns = [4096 * f / (2 * math.pi) for f in rotary_frequencies(128, device="cpu").tolist()]
    assert all(r == pytest.approx(1.0) for r, t in zip(ratio, turns) if t > 33)
    assert all(r == pytest.approx(16.0) for r, t in zip(ratio, turns) if t < 0.95)
    assert ratio == sorted(ratio)
    assert str(yarn.dtype) == "torch.float64" and yarn.shape == (64,)


@pytest.mark.parametrize("changes, error", [
    (dict(rotary_dim=7), ValueError), (dict(rotary_dim=0), ValueError), (dict(rotary_dim=8.0), TypeError),
    (dict(base=1.0), ValueError), (dict(base=math.inf), ValueError), (dict(factor=0.5), ValueError),
    (dict(scaling="other"), ValueError), (dict(scaling="yarn"), ValueError), (dict(rotary_dim=2, scaling="ntk"), ValueError),
    (dict(scaling="yarn", original_length=100, fast_turns=1.0, slow_turns=2.0), ValueError), (dict(factor=True), TypeError),
])
def test_frequencies_refuse(changes, error):
    with pytest.raises(error, match="rotary_frequencies"):
        rotary_frequencies(**{"rotary_dim": 8, "device": "cpu", **changes})


# ------------------------------------------------------------------------ the call cache
class Remembering:
    def __init__(self, error=None):
        self.calls, self.ran, self.error = {}, [], error

    def fast_key(self, operator, device, signature):
        return operator

    def fast_alias(self, key, signature_key):
        self.calls[key] = signature_key

    def fast_find(self, key):
        return self.calls.get(key)

    def fast_run(self, cached, arguments):
        self.ran.append((cached, arguments))
        if self.error is not None:
            raise self.error
        return "ran"


def test_calls_of_a_kind_go_straight_to_their_winner():
    runtime = Remembering()
    assert quick_call(runtime, ("op", 1), (2, 3)) is None and runtime.ran == []
    remember_call(runtime, ("op", 1), "op", 0, {})
    assert quick_call(runtime, ("op", 1), (2, 3)) == "ran" and runtime.ran == [("op", (2, 3))]
    assert quick_call(runtime, ("op", 2), (2, 3)) is None
    remember_call(runtime, None, "op", 0, {})  # a call that has no key
    for error in (RuntimeError("refused"), TypeError("no tensor"), ValueError("bad")):
        refusing = Remembering(error)
        remember_call(refusing, ("op", 1), "op", 0, {})
        assert quick_call(refusing, ("op", 1), ()) is None  # the front-end's checks speak
    with pytest.raises(KeyboardInterrupt):
        interrupted = Remembering(KeyboardInterrupt())
        remember_call(interrupted, ("op", 1), "op", 0, {})
        quick_call(interrupted, ("op", 1), ())


def test_the_call_cache_is_bounded(monkeypatch):
    from radeon_kernels.ops import _runtime

    monkeypatch.setattr(_runtime, "POSITIONAL_CALLS", 3)
    runtime = _runtime.OperatorRuntime(pack_roots=())
    runtime._fast["s"] = ("entry", {}, {})
    for i in range(10):
        runtime.fast_alias((i,), "s")
        assert runtime.fast_find((i,)) is not None and len(runtime._fast_positional) <= 3


# -------------------------------------------------------------------------- the C entries
def test_c_entries_check_their_arguments():
    lib, null = _native.library(), ctypes.c_void_p(0)
    bad, no, ok = _native.RK_ERR_INVALID_ARGUMENT, _native.RK_ERR_UNSUPPORTED, _native.RK_OK
    some = ctypes.c_void_p(256)  # never dereferenced: each call is refused before

    def rotary(tokens=1, hq=2, hk=1, dim=64, rotary=32, strides=(128, 64, 64, 64), amplitude=1.0, dt=1, bits=32, p=null):
        return lib.rk_rotary_embedding(p, p, p, p, p, p, tokens, hq, hk, dim, rotary, *strides, 0, 0, amplitude, dt, bits, null)

    assert rotary(tokens=0) == ok
    for changes in (dict(tokens=-1), dict(hq=0), dict(dim=1, rotary=2), dict(rotary=3), dict(rotary=0), dict(rotary=66),
                    dict(bits=16), dict(dt=2), dict(amplitude=math.inf), dict(amplitude=math.nan),
                    dict(strides=(-1, 64, 64, 64)), dict()):
        assert rotary(**changes) == bad, changes
    for changes in (dict(dim=2048), dict(hq=40000), dict(tokens=2**31)):
        assert rotary(**changes, p=some) == no

    def slots(batch=1, width=1, size=1, free=0, tokens=0, bits=32, p=null):
        return lib.rk_paged_slots(p, p, p, p, p, p, p, p, batch, width, size, free, tokens, bits, null)

    for changes in (dict(batch=0), dict(width=0), dict(size=0), dict(free=-1), dict(tokens=-1), dict(bits=8), dict()):
        assert slots(**changes) == bad, changes
    assert slots(width=2**20, size=2**11, p=some) == no

    def append(tokens=1, heads=1, dim=64, blocks=1, size=16, strides=(64, 64, 64, 64), dt=1, kind=0, bits=32, p=null):
        return lib.rk_paged_cache_append_8bit(p, p, p, p, p, p, p, tokens, heads, dim, blocks, size, *strides, dt, kind, bits,
                                              null, 0, null)

    assert append(tokens=0) == ok
    for changes in (dict(tokens=-1), dict(heads=0), dict(dim=32), dict(blocks=0), dict(size=0), dict(dt=5), dict(kind=2),
                    dict(bits=31), dict(strides=(64, 64, -8, 64)), dict()):
        assert append(**changes) == bad, changes
    for changes in (dict(size=1025), dict(tokens=2**30), dict(strides=(60, 64, 64, 64)), dict(p=ctypes.c_void_p(8))):
        assert append(**{"p": some, **changes}) == no, changes
    size = ctypes.c_size_t(5)
    assert lib.rk_paged_cache_append_8bit_workspace_size(-1, 4, ctypes.byref(size)) == bad and size.value == 0
    assert lib.rk_paged_cache_append_8bit_workspace_size(10, 1000, ctypes.byref(size)) == ok and size.value == 0
    assert lib.rk_paged_cache_append_8bit_workspace_size(100000, 1000, ctypes.byref(size)) == ok and size.value >= 4000
    assert lib.rk_paged_cache_append_8bit_workspace_size(10, 10, None) == bad

    def attention(batch=1, hq=2, hk=1, dim=64, blocks=1, size=16, width=1, scale=1.0, dt=1, kind=0, bits=32, p=null):
        return lib.rk_paged_attention_decode_8bit(p, p, p, p, p, p, p, p, batch, hq, hk, dim, blocks, size, width, scale, dt,
                                                  kind, bits, null, 0, null)

    for changes in (dict(batch=0), dict(hq=0), dict(hq=3, hk=2), dict(dim=96), dict(blocks=0), dict(size=0), dict(width=0),
                    dict(scale=0.0), dict(scale=math.inf), dict(scale=math.nan), dict(dt=-1), dict(kind=7), dict(bits=0),
                    dict()):
        assert attention(**changes) == bad, changes
    for changes in (dict(width=2**21, size=2**10), dict(p=ctypes.c_void_p(264 + 4))):
        assert attention(**{"p": some, **changes}) == no, changes
    def off(count, at, offset):
        pointers = [some] * count
        pointers[at] = ctypes.c_void_p(256 + offset)
        return pointers

    for at, offset in ((0, 4), (1, 8), (2, 8), (3, 2), (4, 1), (5, 4), (6, 4), (7, 8)):
        assert lib.rk_paged_attention_decode_8bit(*off(8, at, offset), 1, 2, 1, 64, 1, 16, 1, 1.0, 1, 0, 64, null, 0, null) == no, at
    for at, offset in ((0, 8), (1, 8), (2, 8), (3, 8), (4, 2), (5, 1), (6, 4)):
        assert lib.rk_paged_cache_append_8bit(*off(7, at, offset), 1, 1, 64, 1, 16, 64, 64, 64, 64, 1, 0, 64, null, 0, null) == no, at
    for at, offset in ((0, 1), (1, 1), (2, 4), (3, 4), (4, 1), (5, 1)):
        assert lib.rk_rotary_embedding(*off(6, at, offset), 1, 2, 1, 64, 32, 128, 64, 64, 64, 0, 0, 1.0, 1, 64, null) == no, at
    for at, offset in ((0, 4), (1, 4), (2, 4), (3, 4), (4, 4), (5, 4), (6, 4), (7, 4)):
        assert lib.rk_paged_slots(*off(8, at, offset), 1, 1, 1, 1, 1, 64, null) == no, at
    assert lib.rk_paged_attention_decode_8bit_workspace_size(3, 2, 64, ctypes.byref(size)) == bad and size.value == 0
    assert lib.rk_paged_attention_decode_8bit_workspace_size(2, 2, 64, None) == bad


def test_manifests_and_contracts_name_the_operators():
    from radeon_kernels.runtime.resources import builtin_contract, builtin_dispatch_registry

    registry = builtin_dispatch_registry()
    for operator in ("rotary_embedding", "paged_slots", "paged_cache_append_8bit", "paged_attention_decode_8bit"):
        assert builtin_contract(operator, "1.0")["operator"] == operator
        entries = registry.get(operator, "1.0").entries
        assert entries and all(e.winner.entrypoint == operator for e in entries)
