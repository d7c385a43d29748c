"""CPU: the serving entry points refuse bad arguments before they touch a device, and the ctypes mirror has the header's layout."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from pyc_b200 import abi, backend

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"pyc_b200_kv_plan_args": abi.KvPlanArgs, "pyc_b200_kv_write_args": abi.KvWriteArgs, "pyc_b200_paged_attention_args": abi.PagedAttentionArgs,
           "pyc_b200_token_logprobs_args": abi.TokenLogprobsArgs, "pyc_b200_token_logprobs_grad_args": abi.TokenLogprobsGradArgs}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "pyc_b200.h"', "int main(void) {"]
    for name, mirror in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT}/include", str(src), "-o", str(tmp_path / "layout")], check=True)
    said = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, mirror in STRUCTS.items():
        assert int(said[name]) == C.sizeof(mirror)
        for f, _ in mirror._fields_:
            assert int(said[f"{name}.{f}"]) == getattr(mirror, f).offset, f"{name}.{f}"


def fill(cls, **over):
    a = cls()
    for f, t in cls._fields_:
        setattr(a, f, 0x10000 if t is C.c_void_p else 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


PLAN = dict(requests=4, block_size=16, num_blocks=64, max_blocks=8, max_tokens=32, seq_lens=0x20000, free_count_out=None)
WRITE = dict(dtype=abi.DTYPE_BF16, tokens=4, kv_heads=2, head_dim=64, block_size=16, num_blocks=8)
ATTEND = dict(dtype=abi.DTYPE_BF16, requests=2, max_query=1, heads=4, kv_heads=2, head_dim=64, block_size=16, num_blocks=8, max_blocks=4, scale=0.1)
SCORE = dict(dtype=abi.DTYPE_F32, rows=3, vocab=10, top_k=2)
GRAD = dict(dtype=abi.DTYPE_F32, rows=3, vocab=10)


@pytest.mark.parametrize("bad, says", [
    (dict(context_lens=None), "NULL"), (dict(result=None), "NULL"), (dict(free_blocks=None), "NULL"), (dict(block_size=24), "block_size"),
    (dict(block_size=256), "block_size"), (dict(requests=0), "requests"), (dict(requests=16385), "requests"), (dict(num_blocks=0), "positive"),
    (dict(max_blocks=0), "positive"), (dict(max_tokens=0), "positive"), (dict(max_blocks=1 << 28), "2^31"), (dict(seq_lens=0x10000), "seq_lens")])
def test_plan_refusals(bad, says):
    L = backend.load()
    assert L.pyc_b200_kv_plan(C.byref(fill(abi.KvPlanArgs, **{**PLAN, **bad})), None) == -1
    assert says in backend.last_error()


def test_null_structs_are_refused():
    L = backend.load()
    for call in (L.pyc_b200_kv_plan, L.pyc_b200_kv_write, L.pyc_b200_token_logprobs, L.pyc_b200_token_logprobs_backward):
        assert call(None, None) == -1 and "NULL" in backend.last_error()
    assert L.pyc_b200_paged_attention(None, 0x10000, 1 << 30, None) == -1 and "NULL" in backend.last_error()


@pytest.mark.parametrize("at, value, says", [(0, 0, "requests"), (0, 16385, "requests"), (1, 17, "block_size"), (2, 0, "positive"), (3, 0, "positive"),
                                             (4, None, "NULL"), (8, None, "NULL")])
def test_release_refusals(at, value, says):
    args = [4, 16, 64, 8] + [0x10000] * 5 + [None]
    args[at] = value
    assert backend.load().pyc_b200_kv_release(*args) == -1 and says in backend.last_error()


@pytest.mark.parametrize("bad, says", [
    (dict(k=None), "NULL"), (dict(v_scale=None), "NULL"), (dict(slot_map=None), "NULL"), (dict(dtype=abi.DTYPE_F32), "bf16 or f16"),
    (dict(block_size=8), "block_size"), (dict(head_dim=96), "head_dim"), (dict(tokens=0), "positive"), (dict(kv_heads=0), "positive"),
    (dict(kv_heads=70000), "positive"), (dict(num_blocks=0), "positive"), (dict(k_stride=132), "strides"), (dict(v_stride=64), "strides"),
    (dict(k=0x10008), "aligned"), (dict(v_cache=0x10004), "aligned")])
def test_write_refusals(bad, says):
    assert backend.load().pyc_b200_kv_write(C.byref(fill(abi.KvWriteArgs, **{**WRITE, **bad})), None) == -1
    assert says in backend.last_error()


@pytest.mark.parametrize("bad, says", [
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(block_table=None), "NULL"), (dict(dtype=abi.DTYPE_F32), "bf16 or f16"),
    (dict(block_size=48), "block_size"), (dict(head_dim=256), "head_dim"), (dict(requests=0), "requests"), (dict(requests=20000), "requests"),
    (dict(max_query=0), "max_query"), (dict(num_blocks=0), "num_blocks"), (dict(heads=5), "heads"), (dict(kv_heads=0), "heads"),
    (dict(q_stride=260), "strides"), (dict(out_stride=128), "strides"), (dict(q=0x10002), "aligned"), (dict(k_cache=0x10008), "aligned")])
def test_attention_refusals(bad, says):
    a = fill(abi.PagedAttentionArgs, **{**ATTEND, **bad})
    assert backend.load().pyc_b200_paged_attention(C.byref(a), 0x10000, 1 << 30, None) == -1
    assert says in backend.last_error()


def test_attention_refuses_a_bad_workspace():
    L, a = backend.load(), fill(abi.PagedAttentionArgs, **ATTEND)
    need = backend.paged_attention_workspace_bytes(2, 1, 4, 2, 64)
    assert need > 0
    assert L.pyc_b200_paged_attention(C.byref(a), None, need, None) == -1 and "NULL" in backend.last_error()
    assert L.pyc_b200_paged_attention(C.byref(a), 0x10000, need - 1, None) == -1 and "workspace" in backend.last_error()
    assert L.pyc_b200_paged_attention(C.byref(a), 0x10010, need, None) == -1 and "256-byte" in backend.last_error()
    for bad in [(0, 1, 4, 2, 64), (1, 0, 4, 2, 64), (1, 1, 5, 2, 64), (1, 1, 4, 0, 64), (1, 1, 4, 2, 80)]:
        assert backend.paged_attention_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("bad, says", [
    (dict(logits=None), "NULL"), (dict(tokens=None), "NULL"), (dict(logprob=None), "NULL"), (dict(dtype=abi.DTYPE_I8), "dtype"), (dict(rows=0), "rows"),
    (dict(vocab=0), "rows"), (dict(vocab=1 << 31), "rows"), (dict(row_stride=9), "stride"), (dict(top_k=33), "top_k"), (dict(top_k=-1), "top_k"),
    (dict(top_k=11), "top_k"), (dict(top_ids=None), "top_ids")])
def test_score_refusals(bad, says):
    assert backend.load().pyc_b200_token_logprobs(C.byref(fill(abi.TokenLogprobsArgs, **{**SCORE, **bad})), None) == -1
    assert says in backend.last_error()


@pytest.mark.parametrize("bad, says", [
    (dict(lse=None), "NULL"), (dict(grad_logits=None), "NULL"), (dict(entropy=None), "entropy"), (dict(dtype=abi.DTYPE_I32), "dtype"),
    (dict(rows=0), "rows"), (dict(row_stride=9), "stride"), (dict(grad_stride=4), "stride"), (dict(row_stride=16), "in place")])
def test_score_gradient_refusals(bad, says):
    assert backend.load().pyc_b200_token_logprobs_backward(C.byref(fill(abi.TokenLogprobsGradArgs, **{**GRAD, **bad})), None) == -1
    assert says in backend.last_error()


def test_cache_class_refuses_what_it_cannot_hold():
    import torch
    from pyc_b200.kv_cache import PagedKvCache
    base = dict(requests=2, num_blocks=8, block_size=16, max_blocks=4, max_tokens=8, heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16, device="cpu")
    for bad in (dict(dtype=torch.float32), dict(block_size=20), dict(head_dim=96), dict(heads=3)):
        with pytest.raises(ValueError):
            PagedKvCache(torch, **{**base, **bad})
    c = PagedKvCache(torch, **base)                       # buffers on the host: the checks alone
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    assert c._rows("k", x, 128) == (4, 128) and c._rows("k", x.reshape(4, 128), 128) == (4, 128)
    wide = torch.zeros((4, 384), dtype=torch.bfloat16)
    assert c._rows("k", wide[:, 128:256], 128) == (4, 384)
    for bad in (x.float(), x.transpose(1, 2), x[:, :1], torch.zeros((9, 128), dtype=torch.bfloat16), x[:0]):
        with pytest.raises(ValueError):
            c._rows("k", bad, 128)
    with pytest.raises(ValueError):
        c.plan([1, 2, 3])
    c.result.copy_(torch.tensor([8, 0, 0, 3]))
    with pytest.raises(backend.BackendError, match="too few free blocks.*3 missing"):
        c.status()


def test_cache_class_refuses_overlapping_rows_and_steps_out_of_order(monkeypatch):
    import torch
    from pyc_b200.kv_cache import PagedKvCache
    c = PagedKvCache(torch, requests=2, num_blocks=8, block_size=16, max_blocks=4, max_tokens=8, heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16,
                     device="cpu")
    row = torch.zeros((1, 128), dtype=torch.bfloat16)
    for bad in (row.expand(4, 128), torch.zeros(4 * 132, dtype=torch.bfloat16).as_strided((4, 128), (132, 1)), torch.zeros(600, dtype=torch.bfloat16).as_strided((4, 128), (64, 1))):
        with pytest.raises(ValueError, match="values apart"):
            c._rows("k", bad, 128)
    with pytest.raises(ValueError, match="max_query"):
        c.attend(0, torch.zeros((8, 256), dtype=torch.bfloat16), max_query=9)
    monkeypatch.setattr(c, "_stream", lambda: 0)
    monkeypatch.setattr(backend, "kv_plan", lambda *a, **k: None)
    monkeypatch.setattr(backend, "kv_release", lambda *a, **k: None)
    c.plan([1, 1])
    with pytest.raises(RuntimeError):
        c.plan([1, 1])
    with pytest.raises(RuntimeError):
        c.release([1, 0])
    c.advance()
    c.release([1, 0])
    c.plan([1, 1])
    c.result.copy_(torch.tensor([8, 0, 0, 1]))             # could not be planned: another one may be
    with pytest.raises(backend.BackendError):
        c.status()
    c.plan([1, 0])


def test_attention_refuses_a_negative_number_of_rows():
    a = fill(abi.PagedAttentionArgs, **ATTEND, rows=-1)
    assert backend.load().pyc_b200_paged_attention(C.byref(a), 0x10000, 1 << 30, None) == -1
    assert "-1 rows" in backend.last_error()


if __name__ == "__main__":
    sys.exit(pytest.main([__file__, "-q"]))
