"""The prompt chunk's entries on the CPU: their argument structures match the C layout, and arguments that they do not
serve are refused, by the wrappers and by the library, before anything is launched."""
import ctypes as C
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "q36_abi.h")
BF, U8, I32, I64 = torch.bfloat16, torch.uint8, torch.int32, torch.int64


@pytest.fixture(scope="module")
def L():
    from bundles_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from bundles_amd import build
        build.build()
    return _lib.lib()


def _structs():
    from bundles_amd import _lib
    return {"q36_page_plan_args": (_lib.PagePlanArgs, _lib.pack_plan), "q36_attn_front_args": (_lib.AttnFrontArgs, _lib.pack_front),
            "q36_chunk_args": (_lib.ChunkArgs, _lib.pack_chunk)}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for cname, (st, _) in _structs().items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in st._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for cname, (st, _) in _structs().items():
        assert got[(cname, "size")] == C.sizeof(st), cname
        for f, _ in st._fields_:
            assert got[(cname, f)] == getattr(st, f).offset, f"{cname}.{f}"


def test_packed_arguments_are_the_filled_structure():
    for st, pack in _structs().values():
        ref, flat = st(), []
        for i, (f, t) in enumerate(st._fields_):
            flat.append(0.5 + i if t is C.c_float else 3 + 7 * i)
            setattr(ref, f, flat[-1])
        assert pack(*flat) == bytes(ref)


def test_entries_take_their_own_structure(L):
    from bundles_amd import _lib
    for name, st in (("q36_page_plan", _lib.PagePlanArgs), ("q36_attn_front", _lib.AttnFrontArgs), ("q36_attn_chunk", _lib.ChunkArgs)):
        for wrong in (C.byref(_lib.MoeArgs()), bytes(C.sizeof(st)), 4096):
            with pytest.raises(C.ArgumentError):
                getattr(L, name)(wrong, None)
        assert getattr(L, name)(None, None) == _lib.Q36_EINVAL


# A call's arguments that pass every check (addresses that are never used), and one change each that is refused.
PLAN = dict(B=2, T=8, page_size=4, table_rows=2, table_width=4, free_count=3, pt_width=9, whole=1, cached=4096, new_tokens=4096,
            req=0, table=4096, free_pages=4096, qsl=4096, seqlens=4096, positions=4096, out_loc=4096, used=4096, page_table=4096)
PLAN_BAD = [dict(B=0), dict(B=65536), dict(T=-1), dict(page_size=0), dict(page_size=3), dict(page_size=2048), dict(table_rows=0),
            dict(table_rows=1), dict(table_width=0), dict(free_count=-1), dict(pt_width=0), dict(cached=0), dict(new_tokens=0),
            dict(table=0), dict(free_pages=0), dict(qsl=0), dict(seqlens=0), dict(positions=0), dict(out_loc=0), dict(used=0)]
FRONT = dict(T=4, max_pos=10, axes=3, q_e4m3=1, qkv_ld=9216, pos_stride=4, axis_map=0b100100, num_slots=7, qkv=4096, q_norm_w=4096,
             k_norm_w=4096, cos_sin=4096, positions=4096, q=4096, gate=4096, out_loc=4096, k_cache=4096, v_cache=4096, eps=1e-6)
FRONT_BAD = [dict(T=0), dict(T=(1 << 20) + 1), dict(max_pos=0), dict(axes=0), dict(axes=5), dict(axes=2), dict(axes=1),
             dict(axis_map=-1), dict(pos_stride=3), dict(qkv_ld=9208), dict(qkv_ld=9220), dict(qkv=0), dict(q_norm_w=0),
             dict(k_norm_w=0), dict(cos_sin=0), dict(positions=0), dict(q=0), dict(out_loc=0), dict(k_cache=0), dict(v_cache=0),
             dict(num_slots=0), dict(num_slots=1 << 31), dict(qkv=4104), dict(cos_sin=4100), dict(gate=4098), dict(q=4100),
             dict(q_e4m3=0, q=4104), dict(k_cache=4100), dict(v_cache=4100), dict(q_norm_w=4098), dict(k_norm_w=4098)]
CHUNK = dict(B=2, T=8, HQ=16, HKV=2, D=256, page_size=16, pt_stride=5, q_e4m3=1, num_slots=100, q=4096, k_cache=4096, v_cache=4096,
             page_table=4096, seqlens=4096, qsl=4096, out=4096, workspace=4096, workspace_bytes=1 << 40, scale=0.0625)
CHUNK_BAD = [dict(B=0), dict(B=65536), dict(T=0), dict(T=(1 << 20) + 1), dict(HQ=32), dict(HKV=4), dict(D=128), dict(page_size=0),
             dict(page_size=24), dict(page_size=2048), dict(pt_stride=0), dict(pt_stride=(1 << 23) + 1), dict(num_slots=0),
             dict(num_slots=1 << 31), dict(q=0), dict(k_cache=0), dict(v_cache=0), dict(page_table=0), dict(seqlens=0), dict(qsl=0),
             dict(out=0), dict(workspace=0), dict(workspace_bytes=100), dict(q=4104), dict(k_cache=4104), dict(v_cache=4104),
             dict(out=4104), dict(workspace=4224)]


@pytest.mark.parametrize("entry,base,bad", [("q36_page_plan", PLAN, b) for b in PLAN_BAD] + [("q36_attn_front", FRONT, b) for b in FRONT_BAD] +
                         [("q36_attn_chunk", CHUNK, b) for b in CHUNK_BAD], ids=str)
def test_the_library_refuses(L, entry, base, bad):
    from bundles_amd import _lib
    st = {"q36_page_plan": _lib.PagePlanArgs, "q36_attn_front": _lib.AttnFrontArgs, "q36_attn_chunk": _lib.ChunkArgs}[entry]
    a = st()
    for k, v in {**base, **bad}.items():
        setattr(a, k, v)
    assert getattr(L, entry)(C.byref(a), None) == _lib.Q36_EINVAL
    assert L.q36_last_error().startswith(entry.encode())


def z(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


def plan_call(**over):
    from bundles_amd.qwen36_layer import paging
    a = dict(cached=z(3), new=z(3), table=z(4, 5), free=z(6), T=7, req=z(3), page_table=z(3, 9), plan=paging.PagePlan.alloc(3, 7, "cpu"))
    a.update(over)
    return paging.plan_pages(**a)


def front_call(**over):
    from bundles_amd.qwen36_layer import attn_fused
    a = dict(qkv=z(5, 9216, dtype=BF), q_norm_w=z(256, dtype=BF), k_norm_w=z(256, dtype=BF), eps=1e-6, cos_sin=z(10, 64, dtype=torch.float32),
             positions=z(5), cache=(z(8, 2, 256, dtype=U8), z(8, 2, 256, dtype=U8), z(5, dtype=I64)))
    a.update(over)
    return attn_fused.attn_front(**a)


class _Space:
    buf = z(256, dtype=U8)


def chunk_call(**over):
    from bundles_amd.qwen36_layer import attn_fused
    a = dict(q=z(5, 16, 256, dtype=U8), k_cache=z(8, 2, 256, dtype=U8), v_cache=z(8, 2, 256, dtype=U8), page_table=z(2, 8),
             seqlens=z(2), qsl=z(3), scale=0.0625, ws=_Space())
    a.update(over)
    return attn_fused.attn_chunk(**a)


def other_plan(**over):
    from bundles_amd.qwen36_layer import paging
    p = paging.PagePlan.alloc(3, 7, "cpu")
    for k, v in over.items():
        setattr(p, k, v)
    return p


def three():
    from bundles_amd.qwen36_layer import attn_fused
    return attn_fused.RopeAxes((11, 11, 10))


@pytest.mark.parametrize("call,over,text", [
    (plan_call, lambda: dict(), "not on the current GPU"),
    (plan_call, lambda: dict(cached=z(3, dtype=I64)), "cached"), (plan_call, lambda: dict(cached=z(3, 1)), "cached"),
    (plan_call, lambda: dict(new=z(4)), "new"), (plan_call, lambda: dict(table=z(4)), "table"),
    (plan_call, lambda: dict(table=z(5, 4).t()), "table"), (plan_call, lambda: dict(free=z(6, 1)), "free"),
    (plan_call, lambda: dict(free=z(12)[::2]), "free"), (plan_call, lambda: dict(req=z(2)), "req"),
    (plan_call, lambda: dict(req=z(3, dtype=I64)), "req"), (plan_call, lambda: dict(page_table=z(2, 9)), "page_table"),
    (plan_call, lambda: dict(page_table=z(3, 18)[:, ::2]), "page_table"), (plan_call, lambda: dict(T=6), "positions"),
    (plan_call, lambda: dict(plan=other_plan(out_loc=z(7))), "out_loc"), (plan_call, lambda: dict(plan=other_plan(qsl=z(3))), "qsl"),
    (front_call, lambda: dict(), "not on the current GPU"), (front_call, lambda: dict(qkv=z(5, 9216)), "qkv"),
    (front_call, lambda: dict(qkv=z(5, 9000, dtype=BF)), "qkv"), (front_call, lambda: dict(qkv=z(9216, 5, dtype=BF).t()), "qkv"),
    (front_call, lambda: dict(qkv=z(5, 9217, dtype=BF)[:, :9216]), "stride"), (front_call, lambda: dict(qkv=z(1, 9216, dtype=BF).expand(5, 9216)), "stride"),
    (front_call, lambda: dict(q_norm_w=z(256)), "q_norm_w"), (front_call, lambda: dict(k_norm_w=z(128, dtype=BF)), "k_norm_w"),
    (front_call, lambda: dict(cos_sin=z(10, 32, dtype=torch.float32)), "cos_sin"), (front_call, lambda: dict(positions=z(3, 5)), "positions"),
    (front_call, lambda: dict(positions=z(5), axes=three()), "positions"), (front_call, lambda: dict(positions=z(2, 5), axes=three()), "positions"),
    (front_call, lambda: dict(positions=z(1, 5).expand(3, 5), axes=three()), "positions"),
    (front_call, lambda: dict(positions=z(5, dtype=I64)), "positions"), (front_call, lambda: dict(q_dtype=torch.float16), "q_dtype"),
    (front_call, lambda: dict(q=z(5, 16, 256, dtype=U8)), "q must"), (front_call, lambda: dict(gate=z(4, 16, 256, dtype=BF)), "gate"),
    (front_call, lambda: dict(cache=(z(8, 2, 128, dtype=U8), z(8, 2, 256, dtype=U8), z(5, dtype=I64))), "k_cache"),
    (front_call, lambda: dict(cache=(z(8, 2, 256, dtype=U8), z(9, 2, 256, dtype=U8), z(5, dtype=I64))), "differ"),
    (front_call, lambda: dict(cache=(z(8, 2, 256, dtype=U8), z(8, 2, 256, dtype=U8), z(4, dtype=I64))), "out_loc"),
    (front_call, lambda: dict(cache=(z(8, 2, 256, dtype=U8), z(8, 2, 256, dtype=U8), z(5))), "out_loc"),
    (chunk_call, lambda: dict(), "not on the current GPU"), (chunk_call, lambda: dict(q=z(5, 16, 256, dtype=torch.float16)), "q must"),
    (chunk_call, lambda: dict(q=z(5, 16, 128, dtype=U8)), "q must"), (chunk_call, lambda: dict(q=z(5, 8, 256, dtype=U8)), "q must"),
    (chunk_call, lambda: dict(q=z(10, 16, 256, dtype=U8)[::2]), "q must"), (chunk_call, lambda: dict(k_cache=z(8, 2, 256)), "k_cache"),
    (chunk_call, lambda: dict(v_cache=z(8, 4, 256, dtype=U8)), "v_cache"), (chunk_call, lambda: dict(v_cache=z(9, 2, 256, dtype=U8)), "differ"),
    (chunk_call, lambda: dict(page_table=z(2, 8, dtype=I64)), "page_table"), (chunk_call, lambda: dict(page_table=z(8, 2).t()), "page_table"),
    (chunk_call, lambda: dict(seqlens=z(3)), "seqlens"), (chunk_call, lambda: dict(qsl=z(2)), "qsl"),
    (chunk_call, lambda: dict(out=z(5, 16, 256)), "out must"), (chunk_call, lambda: dict(out=z(4, 16, 256, dtype=BF)), "out must"),
])
def test_the_wrappers_refuse(call, over, text):
    with pytest.raises(ValueError, match=text):
        call(**over())


@pytest.mark.parametrize("sections,woven", [((32,), False), ((8, 8, 8, 4, 4), False), ((11, 11, 11), False), ((40, -8), False),
                                            ((10, 11, 11), True), ((0, 32), True)])
def test_axes_that_are_none(sections, woven):
    from bundles_amd.qwen36_layer import attn_fused
    with pytest.raises(ValueError, match="RopeAxes"):
        attn_fused.RopeAxes(sections, woven)
    assert attn_fused.RopeAxes((8, 8, 8, 8), True).map < 0  # the last pair's axis sets the top bits


@pytest.mark.parametrize("bad", [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=2e6),
                                 dict(T=1 << 20, B=65535, pt_stride=(1 << 27) // 16)], ids=str)
def test_the_library_refuses_scales_and_too_long_lines(L, bad):
    from bundles_amd import _lib
    a = _lib.ChunkArgs()
    for k, v in {**CHUNK, **bad}.items():
        setattr(a, k, v)
    assert L.q36_attn_chunk(C.byref(a), None) == _lib.Q36_EINVAL
    assert L.q36_last_error().startswith(b"q36_attn_chunk")


def test_the_layer_node_asks_the_engine_for_prompt_batches(monkeypatch):
    """Which batches the attention mixer hands to the chunk path: bf16 rows that its positions fit, of a layer that is
    served, where the engine has a chunk_view that takes them; stock's are the others."""
    import types
    from bundles_amd.qwen36_layer import attn_fused, engine, layer
    m = object.__new__(layer._AttnMixer)
    asked = []
    view = engine.EngineView()
    view.chunk_view = lambda layer_id, fb: asked.append(layer_id)
    m.engine, m.refusal, m.layer_id, m.replica, m.axes, m.max_tokens = view, None, 7, object(), attn_fused.RopeAxes((11, 11, 10)), 8
    m.stock = lambda replica, positions, x, fb: "stock"
    x, fb = z(5, 2048, dtype=BF), types.SimpleNamespace()
    for positions, hidden, n in ((z(5), x, 1), (z(3, 5), x, 2), (z(4), x, 2), (z(2, 5), x, 2), (z(3, 4), x, 2), (z(5), x.float(), 2),
                                 (z(0), x[:0], 2), (z(5, dtype=I64), x, 3)):
        assert m(positions, hidden, fb) == "stock" and asked == [7] * n
    m.axes = None
    assert m(z(3, 5), x, fb) == "stock" and len(asked) == 3
    m.refusal = "a logit cap"
    assert m(z(5), x, fb) == "stock" and len(asked) == 3
    m.refusal, m.engine = None, types.SimpleNamespace(kv_view=lambda *a: None)
    assert m(z(5), x, fb) == "stock"
    assert engine.EngineView().chunk_view(7, fb) is None and engine.SglangView().chunk_view(7, fb) is None


def test_rope_axes_of_a_rotary_embedding():
    import types
    from bundles_amd.qwen36_layer import layer
    assert layer._rope_axes(types.SimpleNamespace()) is None
    assert layer._rope_axes(types.SimpleNamespace(mrope_section=None)) is None
    assert layer._rope_axes(types.SimpleNamespace(mrope_section=[16, 24, 24])) is None  # not 32 pairs: such positions are stock's
    r = layer._rope_axes(types.SimpleNamespace(mrope_section=[11, 11, 10], mrope_interleaved=True))
    assert r.axes == 3 and r.axis_of[:4] == [0, 1, 2, 0]
    assert layer._rope_axes(types.SimpleNamespace(mrope_section=[11, 11, 10])).axis_of[:4] == [0, 0, 0, 0]


def test_the_workspace_entry_refuses(L):
    from bundles_amd import _lib
    need = L.q36_attn_chunk_workspace_bytes()
    for at, size in ((0, need), (4096 + 16, need), (4096, need - 1), (4096, 0)):
        assert L.q36_attn_chunk_workspace_init(at, size, None) == _lib.Q36_EINVAL
        assert L.q36_last_error().startswith(b"q36_attn_chunk_workspace_init")
