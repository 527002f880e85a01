"""The reply controls' refusals, before anything is launched (no GPU needed), and their oracle on plain cases."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import dkv_hip
from oracle import logits_ref

P = 64  # a stand-in for a device pointer, never read here


def args(**change):
    a = dkv_hip.LogitsArgs()
    fields = dict(logits=P, out=P, pick=P, logits_row=1000, out_row=1000, dtype=2, rows=4, vocab=1000, token_bytes=8)
    fields.update(change)
    for name, value in fields.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code,words", [
    (dict(dtype=4), -1, "dtype 4"), (dict(rows=-1), -2, "bad shape"), (dict(rows=65536), -2, "65535"),
    (dict(vocab=0), -2, "bad shape"), (dict(vocab=2**31 - 1), -2, "bad shape"), (dict(history=-1), -2, "history=-1"),
    (dict(biases=-1), -2, "bad shape"), (dict(masks=-1), -2, "bad shape"), (dict(tokens=P), -1, "without lengths"),
    (dict(tokens=P, lengths=P, token_bytes=2), -1, "2 bytes"), (dict(biases=3), -1, "null bias"),
    (dict(biases=3, bias_ids=P, bias_values=P), -1, "null bias"), (dict(allowed=P, words=31, masks=4), -2, "31 mask words"),
    (dict(allowed=P, words=32, masks=3), -2, "3 masks"), (dict(logits=None), -1, "null pointer"),
    (dict(out=None), -1, "null pointer"), (dict(out=65), -1, "misaligned"), (dict(dtype=0, logits=66), -1, "misaligned"),
    (dict(logits_row=999), -2, "overlap"), (dict(out_row=0), -2, "overlap")])
def test_refused(change, code, words):
    a = args(**change)
    rc = dkv_hip.lib().dkv_adjust_logits(ctypes.addressof(a), P, 1 << 20, None)
    assert rc == code and words in dkv_hip.lib().dkv_last_error().decode()


def test_workspace():
    lib = dkv_hip.lib()
    a = args(vocab=100000, logits_row=100000, out_row=100000)
    need = lib.dkv_adjust_logits_workspace_bytes(ctypes.addressof(a))
    assert need >= 4 * 8 * 13
    for workspace, size, code in ((None, need, -1), (P, 8, -3), (68, need, -1)):
        assert lib.dkv_adjust_logits(ctypes.addressof(a), workspace, size, None) == code
    none = args(rows=0)
    assert lib.dkv_adjust_logits(ctypes.addressof(none), None, 0, None) == 0
    assert lib.dkv_adjust_logits(None, None, 0, None) == -1


def test_python_refusals():
    from reply_controls import ReplyControls

    for bad in (dict(rows=-1), dict(rows=70000), dict(vocab=0), dict(device="cpu")):
        with pytest.raises(ValueError):
            ReplyControls(**(dict(rows=2, vocab=10, device="cuda") | bad))
    logits = torch.zeros(4, 1000, dtype=torch.bfloat16)
    for given in (logits, logits[:3], logits.double()):  # on the CPU, too few rows, another type
        with pytest.raises(ValueError):
            dkv_hip.adjust_logits(args(), given)


def test_pack_allowed():
    from reply_controls import pack_allowed

    mask = torch.rand(3, 77) < 0.5
    words = pack_allowed(mask)
    assert words.dtype == torch.int32 and words.shape == (3, 3)
    for t in range(77):
        assert torch.equal((words[:, t // 32] >> (t % 32)) & 1, mask[:, t].int())
    assert not (words[:, 2] >> 13).any()


def test_oracle():
    x, pick = logits_ref.adjust([2.0, -2.0, 1.0, 0.5], [0, 1, 1, 9, 3], 2, 2.0, 0.25, 0.5, [(2, 1.0), (2, 3.0)])
    assert x.tolist() == [1.0, -4.75, 4.0, -0.5] and pick == 2
    assert logits_ref.adjust([1.0, 1.0], [], 0, 1, 0, 0)[1] == 0
    assert logits_ref.adjust([1.0, np.nan], [], 0, 1, 0, 0)[1] == 1
    assert logits_ref.adjust([1.0, np.nan], [], 0, 1, 0, 0, allowed=[False, False])[1] == -1


@pytest.mark.parametrize("change", [dict(tokens=P, lengths=P, history=2**31 - 2**16),
                                    dict(bias_ids=P, bias_values=P, bias_cu=P, biases=2**31 - 1)])
def test_longest_lists(change):
    a = args(**change)
    assert dkv_hip.lib().dkv_adjust_logits(ctypes.addressof(a), P, 1 << 20, None) == -2
    assert "2^31 - 2^16" in dkv_hip.lib().dkv_last_error().decode()
    a = args(**{k: v - 2**17 if type(v) is int and v > P else v for k, v in change.items()})
    assert dkv_hip.lib().dkv_adjust_logits_workspace_bytes(ctypes.addressof(a)) > 0


STRETCHES = """
#include "dkv_stretch.h"
// How often the stretches of a row count each token (seen), and how many of their counters lie outside a stretch.
extern "C" long count(long vocab, int line, int tokens, int shift, int* seen) {
  long outside = 0;
  for (int s = 0; s < dkv::stretches_of_row(vocab, line, tokens); ++s) {
    const long first = (long)s * tokens - shift;
    const dkv::TokenRange own = dkv::tokens_of_stretch(first, tokens, vocab);
    for (long id = -2; id < vocab + 2; ++id) {
      const uint32_t from = (uint32_t)id - own.lowest;
      if (from >= own.count) continue;
      const long at = (int)(from + (uint32_t)(own.lowest - first));
      if (id < 0 || id >= vocab || at < 0 || at >= tokens) ++outside;
      else ++seen[id];
    }
  }
  return outside;
}
"""


@pytest.fixture(scope="module")
def count(tmp_path_factory):
    import subprocess
    from pathlib import Path

    here = tmp_path_factory.mktemp("stretch")
    (here / "count.cpp").write_text(STRETCHES)
    csrc = Path(dkv_hip.__file__).resolve().parent / "csrc"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{csrc}", "-o", here / "count.so", here / "count.cpp"], check=True)
    call = ctypes.CDLL(str(here / "count.so")).count
    call.restype, call.argtypes = ctypes.c_long, [ctypes.c_long, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    return call


@pytest.mark.parametrize("line,tokens", [(8, 64), (4, 64), (8, 8192), (8, 16384), (4, 4096), (4, 16384)])
def test_stretches_count_their_own_tokens(count, line, tokens):
    """Every token of the vocabulary is counted once and inside its stretch, wherever in a line the row begins; so also
    where the last stretch begins past the vocabulary (a vocabulary just below a multiple of the stretch)."""
    some = range(1, 200) if tokens == 64 else [tokens - x for x in range(-9, 10)] + [1, 2 * tokens - 1, 2 * tokens - line + 2]
    for vocab in some:
        for shift in range(line):
            seen = np.zeros(vocab, np.int32)
            assert count(vocab, line, tokens, shift, seen.ctypes.data) == 0, (vocab, shift)
            assert (seen == 1).all(), (vocab, shift)


def test_rows_that_meet():
    """Shared memory of two sets of rows, other than row for row in place, against a count of every byte."""
    rng = np.random.RandomState(0)
    met = 0
    for _ in range(3000):
        rows, width = int(rng.randint(1, 5)), int(rng.randint(1, 6))
        a_row, b_row = (int(width + rng.randint(0, 8)) for _ in range(2))
        a, b = 100, int(100 + rng.randint(-30, 31))
        if rng.rand() < 0.3:
            b_row = a_row
        owner = {a + r * a_row + x: (r, x) for r in range(rows) for x in range(width)}
        same = a == b and a_row == b_row
        want = not same and any(b + r * b_row + x in owner for r in range(rows) for x in range(width))
        assert dkv_hip._rows_meet(a, a_row, b, b_row, rows, width) == want
        met += want
    assert 500 < met < 2500
