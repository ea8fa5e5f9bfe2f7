"""Refusals of the attention step over the 4-bit cache: everything that is decided before a launch, without a GPU; and the
storage formulas against one another."""
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import baracuda_b200 as bq
from baracuda_b200 import _lib
import kv4_reference as ref

P = 16  # any pointer that is aligned; nothing here launches


def test_page_bytes(qlib):
    f = qlib.baracuda_kernels_kv4_page_bytes
    assert f(16, 1, 64) == 1152 and f(64, 8, 128) == 4 * 8 * 2304 and f(32, 2, 256) == 2 * 2 * 4608
    for bad in ((0, 1, 64), (8, 1, 64), (24, 1, 64), (16, 0, 64), (16, 1, 96), (16, 1, 512), (-16, 1, 64)):
        assert f(*bad) == 0
    assert bq.Kv4CacheDescriptor(5, 64, 8, 128).page_bytes == 73728


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_every_channel_of_a_tile_has_a_nibble_of_its_own(dim):
    t, d = torch.arange(16)[:, None], torch.arange(dim)[None]
    for values in (0, 1):
        byte, nib = ref.byte_of(t, d, values, dim)
        seen = (byte * 2 + nib).flatten()
        assert len(seen.unique()) == 16 * dim
        assert int(byte.min()) == 8 * dim * values and int(byte.max()) == 8 * dim * (values + 1) - 1


@pytest.mark.parametrize("dim,page,heads", [(64, 16, 1), (128, 48, 2), (256, 32, 3)])
def test_reference_fills_and_unpacks(dim, page, heads):
    g = torch.Generator().manual_seed(dim)
    k, v = (torch.randn(40, heads, dim, generator=g).to(torch.bfloat16) for _ in range(2))
    cache = torch.full((4, heads * (page // 16) * 18 * dim + 16), 255, dtype=torch.uint8)
    slots = torch.randperm(4 * page, generator=g)[:40]
    ref.fill(cache, page, heads, dim, slots, k, v)
    codes, s, m = ref.unpack(cache, page, heads, dim)
    for i, x in enumerate((k, v)):
        c, sc, mn = ref.quantize(x)
        assert torch.equal(codes[i, slots], c) and torch.equal(s[i, slots], sc) and torch.equal(m[i, slots], mn)
        # half a step, and what rounding s and m to f16 adds: 15 codes of s, and m
        step = sc.repeat_interleave(64, -1)
        off = (ref.values(c, sc, mn) - x.double()).abs()
        assert torch.all(off <= step * (0.5 + 15 * ref.HALF_F16) + x.double().abs().amax(-1, keepdim=True) * 2 * ref.HALF_F16)


def _norm(lib, tokens=4, hq=4, hkv=2, dim=128, q=P, ldq=512, k=P, ldk=256, qw=P, kw=P, eps=1e-6, table=P, rot=128, max_pos=10, positions=P,
          pos_stride=4, axes=1, axis=None, qo=P, ldqo=512, ko=P, ldko=256):
    return lib.baracuda_kernels_qk_norm_rope_bf16_sm100a_run(tokens, hq, hkv, dim, q, ldq, k, ldk, qw, kw, eps, table, rot, max_pos, 0, positions,
                                                             pos_stride, axes, axis, qo, ldqo, ko, ldko, None, 0, None)


def test_norm_rope_statuses(qlib):
    can = qlib.baracuda_kernels_qk_norm_rope_bf16_sm100a_can_implement
    assert can(1, 32, 8, 128, 128, 1) == 0 and can(0, 1, 1, 64, 0, 3) == 0 and can(7, 0, 1, 256, 8, 8) == 0
    for bad, status in (((-1, 1, 1, 64, 64, 1), 2), ((1, -1, 1, 64, 64, 1), 2), ((1, 1, 0, 64, 64, 1), 2), ((1, 1, 1, 0, 0, 1), 2),
                        ((1, 1, 1, 80, 64, 1), 3), ((1, 1, 1, 64, 128, 1), 2), ((1, 1, 1, 64, 20, 1), 3), ((1, 1, 1, 64, 64, 0), 2),
                        ((1, 1, 1, 64, 64, 9), 3), ((1, 1, 1, 64, -8, 1), 2)):
        assert can(*bad) == status, bad
    assert qlib.baracuda_kernels_qk_norm_rope_bf16_sm100a_workspace_size(9, 32, 8, 128) == 0
    assert _norm(qlib, tokens=0, q=None, k=None, qo=None, ko=None) == 0
    for kw, status in ((dict(q=None), 2), (dict(k=None), 2), (dict(qo=None), 2), (dict(ko=None), 2), (dict(ldq=511), 2), (dict(ldk=255), 2),
                       (dict(ldqo=500), 2), (dict(ldko=1), 2), (dict(q=20), 1), (dict(k=18), 1), (dict(ldq=513), 1), (dict(ldko=258), 1),
                       (dict(qw=20), 1), (dict(eps=-1.0), 2), (dict(eps=float("nan")), 2), (dict(table=None), 2), (dict(table=24), 1),
                       (dict(max_pos=0), 2), (dict(positions=None), 2), (dict(positions=18), 1), (dict(axes=2, pos_stride=3), 2)):
        assert _norm(qlib, **kw) == status, kw
    axis = (np.arange(64) % 3).astype(np.uint8)
    assert _norm(qlib, axes=2, axis=axis.ctypes.data) == 2  # names a third axis


def _append(lib, tokens=4, hkv=2, dim=128, k=P, ldk=256, v=P, ldv=256, cache=P, stride=4608, pages=4, page=16, slots=P):
    return lib.baracuda_kernels_kv4_append_bf16_sm100a_run(tokens, hkv, dim, k, ldk, v, ldv, cache, stride, pages, page, slots, None, 0, None)


def _read(lib, tokens=4, hkv=2, dim=128, k=P, ldk=256, v=P, ldv=256, cache=P, stride=4608, pages=4, page=16, slots=P):
    return lib.baracuda_kernels_kv4_read_bf16_sm100a_run(tokens, hkv, dim, cache, stride, pages, page, slots, k, ldk, v, ldv, None, 0, None)


@pytest.mark.parametrize("call", [_append, _read])
def test_append_and_read_statuses(qlib, call):
    assert call(qlib, tokens=0, k=None, v=None, cache=None, slots=None) == 0
    for kw, status in ((dict(tokens=-1), 2), (dict(hkv=0), 2), (dict(dim=32), 3), (dict(page=8), 3), (dict(page=0), 2), (dict(cache=None), 2),
                       (dict(cache=8), 1), (dict(stride=4600), 2), (dict(stride=4616), 1), (dict(pages=-1), 2), (dict(k=None), 2),
                       (dict(v=None), 2), (dict(ldk=255), 2), (dict(ldv=250), 2), (dict(k=18), 1), (dict(ldv=258), 1), (dict(slots=None), 2),
                       (dict(slots=20), 1)):
        assert call(qlib, **kw) == status, kw
    if call is _read:
        assert call(qlib, k=24) == 1 and call(qlib, ldk=260) == 1


def _attend(lib, batch=2, total=2, max_q=1, max_kv=100, hq=8, hkv=2, dim=128, q=P, ldq=1024, cu=P, cache=P, stride=4608, pages=20, page=16, table=P,
            ldt=7, lens=P, scale=0.1, causal=1, window=0, out=P, ldo=1024, lse=None, ws=P, ws_bytes=1 << 40):
    return lib.baracuda_kernels_attention_kv4_bf16_sm100a_run(batch, total, max_q, max_kv, hq, hkv, dim, q, ldq, cu, cache, stride, pages, page, table,
                                                              ldt, lens, scale, causal, window, out, ldo, lse, ws, ws_bytes, None)


def test_attention_statuses(qlib):
    can = qlib.baracuda_kernels_attention_kv4_bf16_sm100a_can_implement
    assert can(1, 1, 1, 8, 1, 128, 16) == 0 and can(0, 0, 0, 1, 1, 64, 16) == 0 and can(4, 100000, 1 << 20, 64, 8, 256, 128) == 0
    for bad, status in (((-1, 1, 1, 8, 1, 128, 16), 2), ((1, -1, 1, 8, 1, 128, 16), 2), ((1, 1, -1, 8, 1, 128, 16), 2), ((1, 1, 1, 8, 3, 128, 16), 2),
                        ((1, 1, 1, 0, 1, 128, 16), 2), ((1, 1, 1, 8, 1, 96, 16), 3), ((1, 1, 1, 8, 1, 128, 17), 3), ((1, 2 ** 31 - 1, 1, 8, 1, 128, 16), 3)):
        assert can(*bad) == status, bad
    assert _attend(qlib, batch=0, q=None) == 0 and _attend(qlib, total=0, q=None) == 0 and _attend(qlib, max_q=0, q=None) == 0
    for kw, status in ((dict(total=-1), 2), (dict(window=-1), 2), (dict(scale=float("inf")), 2), (dict(scale=float("nan")), 2), (dict(q=None), 2),
                       (dict(out=None), 2), (dict(cu=None), 2), (dict(lens=None), 2), (dict(table=None), 2), (dict(cache=None), 2),
                       (dict(ldq=1023), 2), (dict(ldo=1000), 2), (dict(ldt=6), 2), (dict(q=24), 1), (dict(out=8), 1), (dict(ldq=1028), 1),
                       (dict(cu=18), 1), (dict(lens=18), 1), (dict(table=18), 1), (dict(lse=18), 1), (dict(cache=8), 1), (dict(stride=4607), 2)):
        assert _attend(qlib, **kw) == status, kw
    size = qlib.baracuda_kernels_attention_kv4_bf16_sm100a_workspace_size
    need = size(1, 1, 100000, 8, 1, 128)
    assert need > 0
    big = dict(batch=1, max_kv=100000, hkv=1, ldt=6250, stride=2304, pages=6250)
    assert _attend(qlib, **big, ws=None, ws_bytes=0) == 4 and _attend(qlib, **big, ws_bytes=need - 1) == 4 and _attend(qlib, **big, ws=P + 8) == 1
    assert size(0, 1, 100, 8, 1, 128) == 0 and size(1, 0, 100, 8, 1, 128) == 0


def test_plans_refuse_before_they_call(qlib):
    cache = bq.Kv4CacheDescriptor(4, 16, 2, 128)
    with pytest.raises(bq.Unsupported):
        bq.Kv4AppendPlan.select(None, bq.Kv4AppendDescriptor(1, bq.Kv4CacheDescriptor(4, 24, 2, 128)))
    with pytest.raises(bq.InvalidProblem):
        bq.Kv4ReadPlan.select(None, bq.Kv4ReadDescriptor(-1, cache))
    with pytest.raises(bq.InvalidProblem):
        bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(1, 8, 4, 128, cache=cache))  # another number of kv heads
    with pytest.raises(bq.InvalidProblem):
        bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(1, 8, 2, 128, axis_of_pair=[0] * 63))
    with pytest.raises(bq.InvalidProblem):
        bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(1, 1, 10, 3, cache))
    with pytest.raises(bq.InvalidProblem):
        bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(1, 1, 10, 8, cache, scale=float("nan")))
    with pytest.raises(bq.Unsupported):
        bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(1, 1, 1 << 20, 8, cache), bq.PlanPreference(max_workspace_bytes=1))
    plan = bq.Kv4AppendPlan.select(None, bq.Kv4AppendDescriptor(1, cache))
    x, buf, slots = torch.zeros(1, 256, dtype=torch.bfloat16), torch.zeros(4, cache.page_bytes, dtype=torch.uint8), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(bq.InvalidProblem):
        plan.run(None, None, bq.Kv4AppendArgs(k=x, v=x, cache=buf, slots=slots))  # host buffers
    bq.Kv4AppendPlan.select(None, bq.Kv4AppendDescriptor(0, cache)).run(None, None, bq.Kv4AppendArgs(k=x, v=x, cache=buf, slots=slots))


def test_attention_plan_refuses_missing_and_host_queries(qlib):
    cache = bq.Kv4CacheDescriptor(4, 16, 2, 128)
    plan = bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(1, 1, 10, 8, cache))
    some = torch.zeros(1, dtype=torch.int32)
    for q in (None, torch.zeros(1, 1024, dtype=torch.bfloat16), torch.zeros((), dtype=torch.bfloat16)):
        with pytest.raises(bq.InvalidProblem):
            plan.run(None, None, bq.Kv4AttentionArgs(q=q, cu_q=some, kv_lens=some, page_table=some, cache=some, out=q))


def test_cpp_plans(qlib, tmp_path):
    """Compiles and runs the host-only checks of include/baracuda_kernels_kv4_plan.hpp against the library."""
    root = Path(__file__).resolve().parents[1]
    exe, lib = tmp_path / "kv4_plan_host_test", _lib.LIB_PATH.parent
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", str(root / "include"), str(root / "tests" / "cpp" / "kv4_plan_host_test.cpp"),
                    "-o", str(exe), "-L", str(lib), "-lbaracuda_kernels_q", f"-Wl,-rpath,{lib}"], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0 and "kv4_plan_host_test ok" in res.stdout, res.stdout + res.stderr


def test_rust_declarations_name_the_headers_symbols():
    """The -sys declarations have the header's symbols with as many parameters."""
    root = Path(__file__).resolve().parents[1]
    strip = lambda text: re.sub(r"/\*.*?\*/|//[^\n]*", "", text, flags=re.S)  # noqa: E731
    header = strip((root / "include" / "baracuda_kernels_q.h").read_text())
    rust = strip((root / "rust" / "baracuda-kernels-sys" / "src" / "sm100a_q.rs").read_text())
    names = re.findall(r"\b(baracuda_kernels_(?:qk_norm_rope|kv4|attention_kv4)\w*)\(([^)]*)\)", header)
    assert len(names) == 16
    for name, params in names:
        found = re.search(rf"fn {name}\(([^)]*)\)", rust)
        assert found, name
        assert len([x for x in found.group(1).split(",") if x.strip()]) == len(params.split(",")), name


def test_the_self_test_of_the_waits_takes_limits_that_let_copies_arrive(qlib):
    f = qlib.baracuda_kernels_q_selftest_kv4_waits
    for limit in (-1, 1, (1 << 20) - 1, (1 << 28) + 1, 1 << 40):
        assert f(limit) == 2
    for limit in (1 << 20, 1 << 28, 0):
        assert f(limit) == 0


def test_plans_refuse_numbers_that_leave_their_types(qlib):
    """Sizes beyond int32 are not taken modulo 2^32, a head size of zero is refused as such, a scale has to fit f32."""
    wrap = 1 << 32
    for cache in (bq.Kv4CacheDescriptor(4, wrap + 16, 2, 128), bq.Kv4CacheDescriptor(wrap, 16, 2, 128)):
        with pytest.raises(bq.InvalidProblem):
            bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(1, 8, 2, 128, cache=cache))
        with pytest.raises(bq.InvalidProblem):
            bq.Kv4AppendPlan.select(None, bq.Kv4AppendDescriptor(1, cache))
        with pytest.raises(bq.InvalidProblem):
            bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(1, 1, 10, 8, cache))
    for sizes in ((4, wrap + 16, 2, 128), (4, 16, wrap + 2, 128), (4, 16, 2, wrap + 128)):
        assert bq.Kv4CacheDescriptor(*sizes).page_bytes == 0
    for head_dim in (0, -64):
        with pytest.raises(bq.InvalidProblem):
            bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(1, 1, 10, 8, bq.Kv4CacheDescriptor(4, 16, 2, head_dim)))
    for scale in (1e39, -1e39, float("inf")):
        with pytest.raises(bq.InvalidProblem):
            bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(1, 1, 10, 8, bq.Kv4CacheDescriptor(4, 16, 2, 128), scale=scale))
