"""What the recurrent state's and the drafts' entries refuse, without a GPU: nothing is launched, a message says why."""
import ctypes as C
import subprocess

import pytest
import torch

from bundles_amd import _lib
from bundles_amd.qwen36_layer import gdn_fused
from bundles_amd.qwen36_lmhead8 import lmhead8
from test_abi import HEADER

BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def test_structures_match_the_header(tmp_path):
    structs = {"q36_gdn_commit_args": _lib.GdnCommitArgs, "q36_gdn_prompt_args": _lib.GdnPromptArgs,
               "q36_verify_drafts_args": _lib.VerifyDraftsArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for name, st in structs.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in st._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    out = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines()
    got = {tuple(o.split()[:2]): int(o.split()[2]) for o in out}
    for name, st in structs.items():
        assert got[name, "size"] == C.sizeof(st)
        for f, _ in st._fields_:
            assert got[name, f] == getattr(st, f).offset, f"{name}.{f}"


def test_entries_refuse_another_structure(L):
    for name, st in (("q36_gdn_ring_commit", _lib.GdnCommitArgs), ("q36_gdn_prompt", _lib.GdnPromptArgs),
                     ("q36_verify_drafts", _lib.VerifyDraftsArgs)):
        for wrong in (C.byref(_lib.MoeArgs()), bytes(C.sizeof(st)), 4096):
            with pytest.raises(C.ArgumentError):
                getattr(L, name)(wrong, None)
        assert getattr(L, name)(None, None) == _lib.Q36_EINVAL
        assert b"null" in L.q36_last_error()


P = 1 << 20  # an aligned address that no refused call reads


def _args(st, **kw):
    a = st()
    for n, t in st._fields_:
        if t is _lib.P:
            setattr(a, n, P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


COMMIT = dict(B=2, T=4, room=4, advance=1, slots=4, rslots=4, wslots=4, idx_i64=15, cs_slot=24576, win_slot=49152, d_slot=65536,
              dlo_slot=65536, k_slot=32768, klo_slot=32768, g_slot=512)
PROMPT = dict(B=2, rows=10, slots=4, cs_slot=24576, workspace_bytes=1 << 30, oq=None, oqs=None)
DRAFTS = dict(B=2, T=4, V=1000, ld=1000, workspace_bytes=1 << 30)


@pytest.mark.parametrize("entry,st,good,bad,word", [
    ("q36_gdn_ring_commit", _lib.GdnCommitArgs, COMMIT, bad, word) for bad, word in [
        (dict(B=-1), "B="), (dict(B=65536), "B="), (dict(T=0), "T="), (dict(T=9), "T="), (dict(room=17), "room"),
        (dict(room=-1), "room"), (dict(slots=0), "slots"), (dict(rslots=0), "rslots"), (dict(wslots=0), "wslots"),
        (dict(cs_slot=24575), "conv_state"), (dict(cs_slot=24580), "conv_state"), (dict(win_slot=49151), "window"),
        (dict(T=5), "window"), (dict(d_slot=65535), "d ring"), (dict(dlo_slot=65540), "d ring"), (dict(k_slot=32767), "k ring"),
        (dict(klo_slot=0), "k ring"), (dict(g_slot=511), "g ring"), (dict(g_slot=514), "g ring"), (dict(h0=None), "null"),
        (dict(window=None), "null"), (dict(accepted=None), "null"), (dict(write_pos=None), "null"), (dict(h0=P + 8), "aligned"),
        (dict(d_ring=P + 2), "aligned"), (dict(g_ring=P + 4), "aligned"), (dict(conv_state=P + 8), "aligned")]
] + [
    ("q36_gdn_prompt", _lib.GdnPromptArgs, PROMPT, bad, word) for bad, word in [
        (dict(B=-1), "B="), (dict(B=65536), "B="), (dict(rows=-1), "rows"), (dict(rows=(1 << 20) + 1), "rows"),
        (dict(slots=0), "slots"), (dict(cs_slot=24575), "stride"), (dict(cs_slot=24577), "stride"), (dict(mixed=None), "null"),
        (dict(qsl=None), "null"), (dict(state_idx=None), "null"), (dict(workspace=None), "null"), (dict(out=None), "null"),
        (dict(mixed=P + 2), "aligned"), (dict(h0=P + 4), "aligned"), (dict(out=P + 8), "aligned"), (dict(norm_w=P + 2), "aligned"), (dict(dt_bias=P + 2), "aligned"),
        (dict(oq=P), "together"), (dict(oqs=P), "together"), (dict(oq=P + 4, oqs=P), "aligned"), (dict(workspace_bytes=0), "workspace"),
        (dict(workspace=P + 128), "workspace")]
] + [
    ("q36_verify_drafts", _lib.VerifyDraftsArgs, DRAFTS, bad, word) for bad, word in [
        (dict(B=-1), "B="), (dict(B=65536), "B="), (dict(T=0), "T="), (dict(T=9), "T="), (dict(V=0), "V="),
        (dict(V=(1 << 24) + 1, ld=1 << 25), "V="), (dict(ld=999), "ld"), (dict(logits=None), "null"), (dict(drafts=None), "null"),
        (dict(uniforms=None), "null"), (dict(tokens=None), "null"), (dict(counts=None), "null"), (dict(workspace=None), "null"),
        (dict(workspace_bytes=10), "workspace"), (dict(workspace=P + 8), "aligned"), (dict(logits=P + 1), "misaligned"),
        (dict(logits=P + 2, logits_f32=1), "misaligned"),
        (dict(B=65535, T=8, V=1 << 24, ld=1 << 24, workspace_bytes=1 << 60), "too large")]
])
def test_entry_refusals(L, entry, st, good, bad, word):
    a = _args(st, **{**good, **bad})
    assert getattr(L, entry)(C.byref(a), None) == _lib.Q36_EINVAL
    assert word in L.q36_last_error().decode(), L.q36_last_error()


def test_empty_batches_launch_nothing(L):
    assert L.q36_gdn_ring_commit(C.byref(_args(_lib.GdnCommitArgs, **{**COMMIT, "B": 0})), None) == _lib.Q36_OK
    assert L.q36_gdn_prompt(C.byref(_args(_lib.GdnPromptArgs, **{**PROMPT, "B": 0})), None) == _lib.Q36_OK
    assert L.q36_gdn_prompt(C.byref(_args(_lib.GdnPromptArgs, **{**PROMPT, "rows": 0})), None) == _lib.Q36_OK
    assert L.q36_verify_drafts(C.byref(_args(_lib.VerifyDraftsArgs, **{**DRAFTS, "B": 0})), None) == _lib.Q36_OK


def test_workspace_sizes(L):
    assert L.q36_gdn_prompt_workspace_bytes(0, 1) == 0 and L.q36_gdn_prompt_workspace_bytes(1, 0) == 0
    assert L.q36_verify_drafts_workspace_bytes(1, 9, 10) == 0 and L.q36_verify_drafts_workspace_bytes(1, 0, 10) == 0
    for rows, B in ((1, 1), (1000, 7), (1 << 20, 65535)):
        n = L.q36_gdn_prompt_workspace_bytes(rows, B)
        assert n > 0 and n % 256 == 0
        assert L.q36_gdn_prompt_workspace_bytes(rows, B + 1) >= n <= L.q36_gdn_prompt_workspace_bytes(rows + 1, B)
    with pytest.raises(ValueError):
        gdn_fused.PromptWorkspace(0, 1, "cpu")
    with pytest.raises(ValueError):
        lmhead8.VerifyWorkspace(1, 9, 100, "cpu")


# ---- the wrappers, on CPU tensors: every check before the one that no tensor here passes (the device's) ----
def _prompt(**kw):
    rows, B, slots = 6, 2, 3
    a = dict(mixed=torch.zeros((rows, 8192), dtype=BF), z=torch.zeros((rows, 4096), dtype=BF), a=torch.zeros((rows, 32), dtype=BF),
             b=torch.zeros((rows, 32), dtype=BF), conv_state=torch.zeros((slots, 8192, 3), dtype=BF),
             conv_w=torch.zeros((8192, 4), dtype=BF), A_log=torch.zeros(32), dt_bias=torch.zeros(32),
             h0=torch.zeros((slots, 32, 128, 128)), qsl=torch.tensor([0, 2, 6], dtype=I32), state_idx=torch.tensor([0, 1]),
             norm_w=torch.zeros(128, dtype=BF), ws=gdn_fused.PromptWorkspace(rows, B, "cpu"))
    a.update(kw)
    return gdn_fused.gdn_prompt(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(mixed=torch.zeros((6, 8192))), "mixed"), (dict(mixed=torch.zeros((6, 8000), dtype=BF)), "mixed"),
    (dict(z=torch.zeros((5, 4096), dtype=BF)), "z must"), (dict(a=torch.zeros((6, 64), dtype=BF)[:, ::2]), "a must"),
    (dict(b=torch.zeros((6, 16), dtype=BF)), "b must"), (dict(qsl=torch.tensor([0, 2, 6])), "qsl"),
    (dict(qsl=torch.zeros(0, dtype=I32)), "qsl"), (dict(conv_state=torch.zeros((3, 3, 8192), dtype=BF)), "conv_state"),
    (dict(conv_w=torch.zeros((8192, 4))), "conv_w"), (dict(A_log=torch.zeros(16)), "A_log"),
    (dict(dt_bias=torch.zeros(32, dtype=torch.float16)), "dt_bias"), (dict(h0=torch.zeros((3, 32, 128, 128), dtype=BF)), "state"),
    (dict(state_idx=torch.tensor([0])), "state_idx"), (dict(state_idx=torch.tensor([0.0, 1.0])), "state_idx"),
    (dict(norm_w=torch.zeros(128)), "norm_w"), (dict(prefix=torch.zeros(3, dtype=I32)), "prefix"),
    (dict(prefix=torch.zeros(2, dtype=I64)), "prefix"), (dict(out=torch.zeros((5, 4096), dtype=BF)), "out"), (dict(), "not on the current GPU")])
def test_prompt_wrapper(kw, word):
    with pytest.raises(ValueError, match=word):
        _prompt(**kw)


def test_prompt_wrapper_empty():
    e = _prompt(mixed=torch.zeros((0, 8192), dtype=BF), z=torch.zeros((0, 4096), dtype=BF), a=torch.zeros((0, 32), dtype=BF),
                b=torch.zeros((0, 32), dtype=BF), qsl=torch.zeros(3, dtype=I32))
    assert e.shape == (0, 4096)
    assert _prompt(qsl=torch.zeros(1, dtype=I32), state_idx=torch.zeros(0, dtype=I64)).shape == (6, 4096)


def _drafts(**kw):
    B, T, V = 2, 3, 50
    a = dict(logits=torch.zeros((B * T, V), dtype=BF), drafts=torch.zeros((B, T - 1), dtype=I32), uniforms=torch.zeros((B, T)),
             ws=lmhead8.VerifyWorkspace(B, T, V, "cpu"))
    a.update(kw)
    return lmhead8.verify_drafts(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(logits=torch.zeros((2, 3, 50), dtype=BF)), "logits"), (dict(logits=torch.zeros((5, 50), dtype=BF)), "logits"),
    (dict(logits=torch.zeros((6, 50), dtype=torch.float16)), "logits"), (dict(logits=torch.zeros((6, 100), dtype=BF)[:, ::2]), "logits"),
    (dict(uniforms=torch.zeros(6)), "uniforms"), (dict(uniforms=torch.zeros((2, 3), dtype=torch.float64)), "uniforms"),
    (dict(uniforms=torch.zeros((2, 9))), "logits"), (dict(drafts=torch.zeros((2, 3), dtype=I32)), "drafts"),
    (dict(drafts=torch.zeros((2, 2), dtype=I64)), "drafts"), (dict(drafts=None), "drafts"),
    (dict(temperature=torch.zeros(3)), "temperature"), (dict(draft_probs=torch.zeros((2, 3, 50))), "draft_probs"),
    (dict(tokens=torch.zeros((2, 2), dtype=I32)), "tokens"), (dict(counts=torch.zeros(2, dtype=I64)), "counts"),
    (dict(), "not on the current GPU")])
def test_drafts_wrapper(kw, word):
    with pytest.raises(ValueError, match=word):
        _drafts(**kw)


def _commit(**kw):
    T, n = 4, 3
    a = dict(conv_state=torch.zeros((n, 8192, 3), dtype=BF), window=torch.zeros((n, 8192, T + 2), dtype=BF),
             h0=torch.zeros((n, 32, 128, 128)), d_ring=torch.zeros((n, 32, 16, 128), dtype=BF),
             dlo_ring=torch.zeros((n, 32, 16, 128), dtype=BF), k_ring=torch.zeros((n, 16, 16, 128), dtype=BF),
             klo_ring=torch.zeros((n, 16, 16, 128), dtype=BF), g_ring=torch.zeros((n, 32, 16)), state_idx=torch.tensor([0, 1]),
             replay_idx=torch.tensor([0, 1]), win_idx=torch.tensor([0, 1]), write_pos=torch.zeros(n, dtype=I32),
             cache_base=torch.zeros(n, dtype=I32), accepted=torch.ones(2, dtype=I32), T=T)
    a.update(kw)
    return gdn_fused.gdn_ring_commit(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(T=9), "window"), (dict(T=5), "window"), (dict(accepted=torch.ones((2, 1), dtype=I32)), "accepted"),
    (dict(accepted=torch.ones(2)), "accepted"), (dict(accepted=torch.ones(3, dtype=I32)), "state_idx"),
    (dict(conv_state=torch.zeros((3, 8192, 3))), "conv_state"), (dict(window=torch.zeros((3, 4, 8192, 3), dtype=BF)), "windows"),
    (dict(h0=torch.zeros((3, 32, 128, 64))), "checkpoint"), (dict(d_ring=torch.zeros((3, 32, 8, 128), dtype=BF)), "d ring"),
    (dict(klo_ring=torch.zeros((3, 16, 16, 128))), "k ring"), (dict(g_ring=torch.zeros((3, 16, 16))), "g ring"),
    (dict(win_idx=torch.tensor([0])), "win_idx"), (dict(write_pos=torch.zeros(2, dtype=I32)), "write_pos"),
    (dict(cache_base=torch.zeros(3, dtype=I64)), "cache_base"), (dict(), "not on the current GPU")])
def test_commit_wrapper(kw, word):
    with pytest.raises(ValueError, match=word):
        _commit(**kw)


def test_commit_wrapper_room():
    assert _lib.Q36_EINVAL == _lib.lib().q36_gdn_ring_commit(C.byref(_args(_lib.GdnCommitArgs, **{**COMMIT, "room": 99})), None)
