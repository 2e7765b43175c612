"""Decode-step operators without a GPU: what they refuse on the host, and the
library's own argument checks (all made before any CUDA call)."""
import ctypes as C
import re
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import miniep_b200 as M
from miniep_b200 import MEPError, _lib, build
from miniep_b200.model import GRANITE_1B_A400M, Engine, ModelConfig, Shard


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def test_host_tensors_are_refused():
    k = torch.zeros(1, 2, 2, 8, 64)
    with pytest.raises(MEPError, match="CUDA"):
        M.KVCache(k, k)
    with pytest.raises(MEPError, match="CUDA"):
        M.KVCache.empty(1, 2, 2, 8, 64, torch.float32, device="cpu")
    with pytest.raises(MEPError, match="CUDA"):
        M.SharedPrefix(k[0], k[0])
    with pytest.raises(MEPError, match="CUDA"):
        M.sample_tokens(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(MEPError, match="CUDA"):
        M.sample_tokens([1.0], torch.zeros(2))


def _store(lib, heads, cap=8, col=0):
    """mep_norm_rope_store with null tensors."""
    return lib.mep_norm_rope_store(_lib.STORE_ARGS.pack(
        *heads, *[0] * 12, 0, 0, 1e-6, 0, 0, 0, 8, 0, 0, 0, 0, 0, 0, 0, 0, cap, col, 0), None)


def _attend(lib, heads, cap=8, col=0):
    return lib.mep_cache_attention(_lib.ATTENTION_ARGS.pack(
        *heads, *[0] * 8, cap, 0, 0, col, 0, 0, 0, 0, 1.0, 0, 0, 0), None)


def _heads(dtype=1, cache=1, B=2, T=1, Hq=4, Hk=2, D=64):
    return [dtype, cache, B, T, Hq, Hk, D]


BAD_HEADS = [(dict(dtype=2), b"dtype"), (dict(dtype=3), b"dtype"), (dict(cache=0), b"cache"),
             (dict(B=-1), b"negative"), (dict(T=-1), b"negative"), (dict(Hq=3), b"multiple"),
             (dict(Hk=0), b"multiple"), (dict(D=24), b"head_dim"), (dict(D=144), b"head_dim"),
             (dict(D=0), b"head_dim"), (dict(B=1 << 20), b"batch")]


@pytest.mark.parametrize("bad,word", BAD_HEADS, ids=str)
def test_bad_heads(lib, bad, word):
    n = C.c_int64()
    assert lib.mep_cache_attention_workspace(*_heads(**bad), 8, 0, 0, C.byref(n)) == 1
    assert word in lib.mep_last_error(None)
    assert _store(lib, _heads(**bad)) == 1
    assert word in lib.mep_last_error(None)
    assert _attend(lib, _heads(**bad)) == 1
    assert word in lib.mep_last_error(None)


@pytest.mark.parametrize("B,T,Hq", [(14351, 149640, 1), (1, 1 << 21, 1023), (65535, 1 << 15, 1)],
                         ids=str)
def test_rows_that_round_up_past_32_bits(lib, B, T, Hq):
    """Rows are counted in tiles of up to 256: the last whole one has to fit 32 bits."""
    n = C.c_int64()
    rc = lib.mep_cache_attention_workspace(*_heads(B=B, T=T, Hq=Hq, Hk=1), T, 0, 0, C.byref(n))
    assert rc == (1 if B * T * Hq > 2 ** 31 - 1025 else 0)
    if rc:
        assert b"2^31" in lib.mep_last_error(None)


@pytest.mark.parametrize("col", [-1, 1 << 62, 1 << 63, 1 << 70, -(1 << 63) - 1])
def test_host_columns_past_64_bits(col):
    with pytest.raises(MEPError, match="column"):
        M.decode._column(col, None)


def test_columns_and_null_tensors(lib):
    for cap, col, word in ((8, 8, b"fit"), (8, -1, b"fit"), (-1, 0, b"capacity"), (8, 0, b"null")):
        assert _store(lib, _heads(), cap, col) == 1
        assert word in lib.mep_last_error(None)
        assert _attend(lib, _heads(), cap, col) == 1
        assert (b"null" if cap == 8 and col == 0 else b"") in lib.mep_last_error(None)
    for start, n in ((-1, 2), (0, 9), (8, 1), (3, -1)):
        assert lib.mep_kv_read(1, 2, 2, 64, None, None, None, None, 8, start, n, None, None,
                               None) == 1
        assert b"columns" in lib.mep_last_error(None)
    assert lib.mep_kv_read(1, 2, 2, 64, None, None, None, None, 8, 0, 0, None, None, None) == 0
    assert lib.mep_kv_read(1, 2, 2, 64, None, None, None, None, 8, 0, 1, None, None, None) == 1


def test_packed_arguments_match_the_header(lib):
    """The structs are 8-byte fields in the header's order."""
    text = (Path(__file__).resolve().parents[1] / "include" / "miniep_b200.h").read_text()
    for name, packed in (("store", _lib.STORE_ARGS), ("attention", _lib.ATTENTION_ARGS)):
        body = re.search(r"typedef struct mep_%s_args \{(.*?)\}" % name, text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [f for d in body.split(";") if d.strip() for f in d.split(",")]
        kinds = "".join("d" if "double" in f else "q" for f in fields)
        want = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", packed.format))
        assert kinds == want
        assert packed.size == 8 * len(fields)
    assert lib.mep_norm_rope_store(None, None) == 1
    assert lib.mep_cache_attention(None, None) == 1


def test_calls_without_rows_do_nothing(lib):
    """No token, no row: fine, and no CUDA call (none would work here)."""
    assert _store(lib, _heads(B=0)) == 0
    assert _store(lib, _heads(T=0), 8, 8) == 0
    assert _attend(lib, _heads(B=0)) == 0
    assert _attend(lib, _heads(T=0), 8, 8) == 0
    assert lib.mep_sample(0, None, 0, 5, 5, *[None] * 5, 1.0, 0, 1.0, 0.0, None, None, None) == 0


@pytest.mark.parametrize("args,word", [
    ((2, 2, 5, 5, 1.0, 0, 1.0, 0.0), b"dtype"), ((0, -1, 5, 5, 1.0, 0, 1.0, 0.0), b"rows"),
    ((0, 2, 0, 5, 1.0, 0, 1.0, 0.0), b"vocab"), ((0, 2, 1 << 25, 1 << 25, 1.0, 0, 1.0, 0.0), b"vocab"),
    ((0, 2, 5, -5, 1.0, 0, 1.0, 0.0), b"stride"), ((0, 2, 5, 5, -1.0, 0, 1.0, 0.0), b"temperature"),
    ((0, 2, 5, 5, float("nan"), 0, 1.0, 0.0), b"temperature"),
    ((0, 2, 5, 5, 1.0, -1, 1.0, 0.0), b"top_k"), ((0, 2, 5, 5, 1.0, 0, 0.0, 0.0), b"top_p"),
    ((0, 2, 5, 5, 1.0, 0, 1.0, 1.1), b"min_p"), ((0, 2, 5, 5, 1.0, 0, 1.0, 0.0), b"null")], ids=str)
def test_bad_sampling_arguments(lib, args, word):
    dtype, rows, vocab, stride, t, k, p, m = args
    assert lib.mep_sample(dtype, None, rows, vocab, stride, *[None] * 5, t, k, p, m, None, None,
                          None) == 1
    assert word in lib.mep_last_error(None)


def test_workspace_is_host_arithmetic(lib):
    n = C.c_int64(-1)
    assert lib.mep_cache_attention_workspace(*_heads(), 4096, 4000, 512, C.byref(n)) == 0
    assert n.value >= 0
    assert lib.mep_cache_attention_workspace(*_heads(), 4096, 4000, 512, None) == 1


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_scale_must_be_finite(lib, scale):
    args = _lib.ATTENTION_ARGS.pack(*_heads(), *[0] * 8, 8, 0, 0, 0, 0, 0, 0, 0, scale, 0, 0, 0)
    assert lib.mep_cache_attention(args, None) == 1
    assert b"scale" in lib.mep_last_error(None)


@pytest.mark.parametrize("start,n", [(2 ** 63 - 1, 2), (2 ** 63 - 1, 2 ** 63 - 1), (5, 2 ** 63 - 1)])
def test_columns_to_read_whose_end_passes_64_bits(lib, start, n):
    assert lib.mep_kv_read(1, 2, 2, 64, None, None, None, None, 8, start, n, None, None, None) == 1
    assert b"columns" in lib.mep_last_error(None)


class _NoForward:
    """A model that must not be reached."""
    cfg = ModelConfig.from_dict(dict(GRANITE_1B_A400M, num_hidden_layers=1))
    device, dtype = torch.device("cpu"), torch.float32

    def forward(self, *a, **k):
        raise AssertionError("a forward ran")


def test_an_empty_common_prompt_is_refused():
    with pytest.raises(ValueError, match="token"):
        Engine(_NoForward()).build_prefix([])


def test_replayed_steps_behind_the_cache_are_refused():
    m = _NoForward()
    shard = Shard([[1, 2, 3]], m.cfg, 2, "cpu", torch.float32)
    shard.used, shard.last_tokens = 3, torch.zeros(1, dtype=torch.long)
    with pytest.raises(ValueError, match="columns"):
        Engine(m).decode_graphed(shard, 3)
    assert shard.used == 3 and shard.generated == [[]]


def test_the_package_imports_on_a_torch_without_cuda():
    """Planners, oracle forms and the host side need no CUDA build of torch:
    without its bindings' private names the package still imports."""
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, n)\n"
            "import miniep_b200 as M\n"
            "M.plan_balanced, M.Placement, M.KVCache\n")
    root = Path(M.__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(root)!r})\n" + code],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
