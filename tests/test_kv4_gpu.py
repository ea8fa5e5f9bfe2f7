"""The attention step over the 4-bit cache on the GPU, through the plans: against tests/kv4_reference.py in 64 bits."""
import math

import pytest
import torch

import baracuda_b200 as bq
import kv4_reference as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _cache(pages, page, heads, dim, pad=0, fill=255):
    desc = bq.Kv4CacheDescriptor(pages, page, heads, dim)
    return desc, torch.full((pages, desc.page_bytes + pad), fill, dtype=torch.uint8, device="cuda")


def _angles(longest, rot):
    a = torch.arange(longest, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(rot // 2, device="cuda").double() / max(rot // 2, 1))
    return torch.cat([a.cos(), a.sin()], 1).float()


# ------------------------------------------------------------------------------------------------ append and read
def _append(desc, cache, k, v, slots):
    bq.Kv4AppendPlan.select(None, bq.Kv4AppendDescriptor(k.shape[0], desc)).run(None, None, bq.Kv4AppendArgs(k=k, v=v, cache=cache, slots=slots))


@pytest.mark.parametrize("dim,heads,page,tokens,pad", [(64, 1, 16, 1, 0), (64, 3, 48, 77, 16), (128, 8, 64, 500, 0), (128, 2, 16, 33, 48),
                                                       (256, 4, 32, 130, 0), (256, 1, 128, 1, 32)])
def test_append_writes_the_formats_bytes_and_nothing_else(dim, heads, page, tokens, pad):
    g = _gen(tokens + dim)
    pages = -(-tokens // page) + 3
    desc, cache = _cache(pages, page, heads, dim, pad, fill=0xA5)
    wide = _randn(g, tokens, 2 * heads * dim + 12).to(BF16)  # keys and values as columns of a wider matrix
    k, v = wide[:, 4 : 4 + heads * dim], wide[:, 8 + heads * dim : 8 + 2 * heads * dim]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[tokens // 2] = -1 if tokens > 1 else slots[tokens // 2]
    want = ref.fill(cache.clone(), page, heads, dim, slots[slots >= 0], *(x.reshape(tokens, heads, dim)[slots >= 0] for x in (k, v)))
    _append(desc, cache, k, v, slots)
    torch.cuda.synchronize()
    assert bq.device_status() == 0
    assert torch.equal(cache, want)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_append_edge_values(dim):
    """Constant groups, zeros, ties between codes, the largest and smallest numbers; NaN and infinities stay in their group."""
    g = _gen(dim)
    desc, cache = _cache(2, 16, 1, dim)
    rows = [torch.zeros(dim), torch.full((dim,), 3.0), torch.full((dim,), -1e30), torch.linspace(-1, 1, dim),
            torch.arange(dim).float() % 31 * 0.5, torch.cat([torch.full((dim - 1,), 1e-30), torch.tensor([2e-30])]),
            torch.cat([torch.full((dim - 1,), 100.0), torch.tensor([100.5])]), torch.full((dim,), 3e38) * (-1.0) ** torch.arange(dim)]
    x = torch.stack(rows).cuda().to(BF16)
    bad = _randn(g, 3, dim).to(BF16)
    bad[0, 5], bad[1, 6], bad[2, 7] = math.nan, math.inf, -math.inf
    x = torch.cat([x, bad])
    slots = torch.arange(len(x), device="cuda")
    _append(desc, cache, x, x.flip(0).contiguous(), slots)
    codes, s, m = ref.unpack(cache, 16, 1, dim)
    for which, y in ((0, x), (1, x.flip(0))):
        wc, ws, wm = ref.quantize(y.unsqueeze(1))
        live = ~torch.isnan(ws)
        assert torch.equal(torch.isnan(s[which, : len(x)]), torch.isnan(ws))
        assert torch.equal(s[which, : len(x)][live], ws[live]) and torch.equal(m[which, : len(x)].nan_to_num(), wm.nan_to_num())
        keep = live.repeat_interleave(64, -1)
        assert torch.equal(codes[which, : len(x)][keep], wc[keep])
    assert bq.device_status() == 0


@pytest.mark.parametrize("dim,heads,page,tokens", [(64, 3, 32, 45), (128, 8, 64, 1), (128, 1, 16, 700), (256, 2, 48, 99)])
def test_read_gives_the_values(dim, heads, page, tokens):
    g = _gen(tokens)
    pages = -(-tokens // page) + 2
    desc, cache = _cache(pages, page, heads, dim, 32)
    cache.random_(0, 256, generator=g)
    codes, s, m = ref.unpack(cache, page, heads, dim)
    slots = torch.randint(0, pages * page, (tokens,), generator=g, device="cuda")  # the same slot twice among them
    out = torch.full((tokens, 2 * heads * dim + 16), 7.0, dtype=BF16, device="cuda")
    k, v = out[:, : heads * dim], out[:, heads * dim + 8 : 2 * heads * dim + 8]
    if tokens > 2:
        slots[1] = -5
    bq.Kv4ReadPlan.select(None, bq.Kv4ReadDescriptor(tokens, desc)).run(None, None, bq.Kv4ReadArgs(cache=cache, slots=slots, k=k, v=v))
    torch.cuda.synchronize()
    for which, got in ((0, k), (1, v)):
        s32, m32, c32 = (x[which].float() for x in (s, m, codes))
        want = (c32 * s32.repeat_interleave(64, -1) + m32.repeat_interleave(64, -1)).to(BF16)[slots.clamp(min=0)].flatten(1)
        want[slots < 0] = 7.0
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert torch.all(out[:, heads * dim : heads * dim + 8] == 7) and torch.all(out[:, 2 * heads * dim + 8 :] == 7)
    assert bq.device_status() == 0


def test_slots_beyond_the_cache_are_reported_and_left_out():
    g = _gen(1)
    desc, cache = _cache(2, 16, 2, 128)
    before = cache.clone()
    k, v = _randn(g, 2, 256).to(BF16), _randn(g, 2, 256).to(BF16)
    slots = torch.tensor([32, 1 << 40], device="cuda")
    _append(desc, cache, k, v, slots)
    torch.cuda.synchronize()
    assert bq.device_status() == 402 and bq.device_status() == 0
    assert torch.equal(cache, before)
    back = torch.zeros_like(k)
    bq.Kv4ReadPlan.select(None, bq.Kv4ReadDescriptor(2, desc)).run(None, None, bq.Kv4ReadArgs(cache=cache, slots=slots, k=back, v=back.clone()))
    torch.cuda.synchronize()
    assert bq.device_status() == 402 and not back.any()


# ------------------------------------------------------------------------------------------------ norm and rotation
NORM_CASES = [
    # tokens, heads_q, heads_kv, dim, rot, interleaved, axes (None: one), norm
    (1, 32, 8, 128, 128, False, None, True),
    (5, 5, 1, 64, 32, True, None, True),
    (33, 3, 3, 256, 256, False, None, True),
    (700, 32, 8, 128, 128, False, 3, True),
    (513, 40, 8, 64, 64, True, 2, True),
    (9, 7, 1, 128, 40, False, 3, True),
    (17, 4, 2, 256, 8, True, None, True),
    (65, 4, 4, 128, 0, False, None, True),
    (65, 4, 2, 128, 64, False, None, False),
]


def _norm_inputs(tokens, hq, hkv, dim, rot, axes, seed):
    g = _gen(seed)
    qkv = (_randn(g, tokens, (hq + 2 * hkv) * dim) * torch.exp(_randn(g, (hq + 2 * hkv) * dim))).to(BF16)
    if tokens > 1:
        qkv[1] = 0  # a row of zeros: eps alone under the root
    weights = [1 + 0.5 * _randn(g, dim), 1 + 0.5 * _randn(g, dim)]
    n_axes = axes or 1
    positions = torch.randint(0, 1000, (n_axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    table = None if axes is None else torch.randint(0, axes, (rot // 2,), generator=g, device="cuda").tolist()
    if table:
        table[-1] = axes - 1
    return qkv, weights, positions, table, _angles(1000, rot) if rot else None


@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,interleaved,axes,norm", NORM_CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_and_rotation(tokens, hq, hkv, dim, rot, interleaved, axes, norm, in_place):
    qkv, (wq, wk), positions, table, angles = _norm_inputs(tokens, hq, hkv, dim, rot, axes, tokens + rot)
    if not norm:
        wq = wk = None
    before = qkv.clone()
    q, k = qkv[:, : hq * dim], qkv[:, hq * dim : (hq + hkv) * dim]
    q_out, k_out = (q, k) if in_place else (torch.empty_like(q), torch.empty_like(k))
    plan = bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(tokens, hq, hkv, dim, rot_dim=rot, interleaved=interleaved,
                                                                  axis_of_pair=table, eps=1e-5))
    plan.run(None, None, bq.QkNormRopeArgs(q=q, k=k, q_out=q_out, k_out=k_out, q_weight=wq, k_weight=wk, cos_sin=angles,
                                           positions=positions if axes else positions[0]))
    torch.cuda.synchronize()
    assert bq.device_status() == 0
    for x, got, heads, w in ((before[:, : hq * dim], q_out, hq, wq), (before[:, hq * dim : (hq + hkv) * dim], k_out, hkv, wk)):
        want, tol = ref.norm_rope(x, heads, dim, w, 1e-5, angles, positions, table, rot, interleaved)
        err = (got.double().reshape(want.shape) - want).abs()
        assert torch.all(err <= tol), f"off by {float((err / tol).max())} of what the roundings allow"
    if in_place:
        assert torch.equal(qkv[:, (hq + hkv) * dim :], before[:, (hq + hkv) * dim :])
    else:
        assert torch.equal(qkv, before)


@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,interleaved,axes,norm", NORM_CASES)
def test_the_one_launch_form_leaves_the_bits_of_the_two_launches(tokens, hq, hkv, dim, rot, interleaved, axes, norm):
    qkv, (wq, wk), positions, table, angles = _norm_inputs(tokens, hq, hkv, dim, rot, axes, tokens + rot + 1)
    if not norm:
        wq = wk = None
    q, k, v = qkv[:, : hq * dim], qkv[:, hq * dim : (hq + hkv) * dim], qkv[:, (hq + hkv) * dim :]
    page = 32
    desc, one = _cache(-(-tokens // page) + 1, page, hkv, dim)
    two = one.clone()
    slots = torch.randperm(one.shape[0] * page, device="cuda", generator=_gen(3))[:tokens]
    slots[0] = -1 if tokens > 4 else slots[0]
    kw = dict(rot_dim=rot, interleaved=interleaved, axis_of_pair=table)
    turn = dict(q=q, k=k, q_weight=wq, k_weight=wk, cos_sin=angles, positions=positions if axes else positions[0])
    q1, q2, k2 = torch.empty(tokens, hq * dim, dtype=BF16, device="cuda"), torch.empty(tokens, hq * dim, dtype=BF16, device="cuda"), torch.empty(tokens, hkv * dim, dtype=BF16, device="cuda")
    bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(tokens, hq, hkv, dim, cache=desc, **kw)).run(
        None, None, bq.QkNormRopeArgs(q_out=q1, v=v, cache=one, slots=slots, **turn))
    bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(tokens, hq, hkv, dim, **kw)).run(
        None, None, bq.QkNormRopeArgs(q_out=q2, k_out=k2, **turn))
    _append(desc, two, k2, v, slots)
    torch.cuda.synchronize()
    assert torch.equal(q1, q2) and torch.equal(one, two)
    want = ref.fill(torch.full_like(one, 255), page, hkv, dim, slots[slots >= 0], *(x.reshape(tokens, hkv, dim)[slots >= 0] for x in (k2, v)))
    assert torch.equal(one, want)


def test_positions_out_of_range_are_cut_and_reported():
    qkv, (wq, wk), _, _, angles = _norm_inputs(2, 1, 1, 64, 64, None, 5)
    q, k = qkv[:, :64], qkv[:, 64:128]
    plan = bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(2, 1, 1, 64))
    got = []
    for p in ([-3, 1000], [0, 999]):
        args = bq.QkNormRopeArgs(q=q, k=k, q_out=torch.empty_like(q), k_out=torch.empty_like(k), cos_sin=angles,
                                 positions=torch.tensor(p, dtype=torch.int32, device="cuda"))
        plan.run(None, None, args)
        torch.cuda.synchronize()
        got.append((args.q_out, args.k_out, bq.device_status()))
    assert got[0][2] == 401 and got[1][2] == 0
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


# ------------------------------------------------------------------------------------------------ attention
class Problem:
    """A batch over a cache whose unused places hold 0xFF (NaN scales) and whose page table holds -1 where nothing is."""

    def __init__(self, lens, heads_q, heads_kv, dim, page, seed=0, causal=True, window=0, scale=None, pad_rows=3, max_q=None, max_kv=None,
                 q_gain=1.5):
        g = _gen(seed)
        self.dim, self.page, self.heads_q, self.heads_kv, self.causal, self.window = dim, page, heads_q, heads_kv, causal, window
        self.scale = dim ** -0.5 if scale is None else scale
        self.q_lens, self.lens = [n for n, _ in lens], [n for _, n in lens]
        rows = sum(self.q_lens)
        counts = [-(-n // page) for n in self.lens]
        self.max_q, self.max_kv = max_q or max(self.q_lens), max_kv or max(self.lens)
        width = max(1, -(-self.max_kv // page))
        pages = sum(counts) + 2
        self.desc, self.cache = _cache(pages, page, heads_kv, dim, 16)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), width + 1), -1, dtype=torch.int32, device="cuda")
        at, slots = 0, []
        for i, n in enumerate(self.lens):
            self.table[i, : counts[i]] = order[at : at + counts[i]]
            at += counts[i]
            place = torch.arange(n, device="cuda")
            slots.append(self.table[i].long()[place // page] * page + place % page)
        slots = torch.cat(slots)
        if len(slots):
            k = (_randn(g, len(slots), heads_kv, dim) + 0.5 * _randn(g, heads_kv, dim)).to(BF16)
            v = (_randn(g, len(slots), heads_kv, dim) * torch.exp(_randn(g, len(slots), 1, 1))).to(BF16)
            ref.fill(self.cache, page, heads_kv, dim, slots, k, v)
        self.cu_q = torch.tensor([sum(self.q_lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.rows, self.total = rows, rows + pad_rows
        wide = (q_gain * _randn(g, self.total, heads_q * dim + 8)).to(BF16)
        self.q = wide[:, : heads_q * dim]

    def plan(self):
        return bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(len(self.lens), self.max_q, self.max_kv, self.heads_q, self.desc,
                                                                          causal=self.causal, window=self.window, scale=self.scale))

    def run(self, stream=None, lse=True):
        plan = self.plan()
        out = torch.full((self.total, self.heads_q * self.dim + 16), 7.0, dtype=BF16, device="cuda")
        args = bq.Kv4AttentionArgs(q=self.q, cu_q=self.cu_q, kv_lens=self.kv_lens, page_table=self.table, cache=self.cache,
                                   out=out[:, : self.heads_q * self.dim],
                                   lse=torch.full((self.total, self.heads_q), 7.0, device="cuda") if lse else None)
        workspace = torch.full((plan.workspace_size(),), 255, dtype=torch.uint8, device="cuda")
        plan.run(stream, workspace, args)
        return args

    def check(self, args):
        torch.cuda.synchronize()
        assert bq.device_status() == 0
        assert torch.all(args.out[self.rows :] == 7) and torch.all(args.out._base[:, self.heads_q * self.dim :] == 7)
        want, lse, tol, lse_tol = ref.attention(self.q[: self.rows], self.cu_q, self.kv_lens, self.table, self.cache, self.page, self.heads_kv,
                                                self.dim, self.scale, self.causal, self.window)
        got = args.out[: self.rows].double().reshape(want.shape)
        assert torch.isfinite(got).all()
        err = (got - want).abs()
        assert torch.all(err <= tol), f"off by {float((err / tol).max())} of what the roundings allow"
        # all roundings together, as independent ones: bf16 (at most 2^-8 / sqrt 3 of each value) and a few of 2^-11
        if float(want.norm()) > 0:
            assert float(err.norm() / want.norm()) <= 2.0 ** -8 / math.sqrt(3.0) + 4 * 2.0 ** -11
        if args.lse is not None:
            got = args.lse[: self.rows].double()
            assert torch.equal(torch.isinf(got), torch.isinf(lse)) and torch.all(got[torch.isinf(got)] < 0)
            live = ~torch.isinf(lse)
            assert torch.all((got - lse).abs()[live] <= lse_tol[live])
            assert torch.all(args.lse[self.rows :] == 7)


ATTENTION_CASES = [
    # (rows, cached) of each sequence, heads_q, heads_kv, dim, page, causal, window
    ([(1, 1)], 1, 1, 64, 16, True, 0),
    ([(1, 17)], 32, 8, 128, 16, True, 0),
    ([(1, 300), (1, 31), (1, 32), (1, 33)], 8, 1, 128, 64, True, 0),
    ([(1, 1000), (0, 500), (1, 0), (1, 129)], 16, 2, 64, 32, True, 0),
    ([(1, 513), (1, 64)], 10, 2, 256, 48, True, 0),
    ([(1, 2500)], 4, 4, 128, 128, True, 0),
    ([(1, 700), (1, 90)], 12, 4, 128, 16, True, 100),
    ([(5, 400), (3, 3), (8, 8), (1, 77)], 8, 2, 128, 32, True, 0),
    ([(4, 2), (7, 5), (2, 0)], 4, 2, 64, 16, True, 0),
    ([(6, 90), (2, 35)], 3, 1, 256, 16, True, 20),
    ([(3, 130), (9, 70)], 20, 4, 128, 64, False, 0),
    ([(2, 40), (5, 300)], 4, 1, 64, 16, False, 33),
    ([(16, 333)], 16, 1, 128, 32, True, 1),
    ([(100, 100), (37, 260)], 4, 2, 128, 16, True, 0),
    ([(70, 200), (33, 33), (0, 9)], 5, 1, 64, 32, True, 50),
    ([(65, 65), (130, 300)], 4, 2, 256, 64, True, 0),
    ([(50, 20), (200, 150)], 2, 1, 128, 16, True, 0),
    ([(129, 257)], 7, 7, 128, 16, False, 0),
]


@pytest.mark.parametrize("lens,heads_q,heads_kv,dim,page,causal,window", ATTENTION_CASES)
def test_attention(lens, heads_q, heads_kv, dim, page, causal, window):
    p = Problem(lens, heads_q, heads_kv, dim, page, seed=len(lens) + dim, causal=causal, window=window)
    p.check(p.run())


@pytest.mark.parametrize("dim,heads_q,heads_kv,rows", [(128, 8, 2, 1), (64, 64, 2, 1), (256, 4, 2, 3), (128, 16, 1, 2)])
def test_attention_joins_many_slices(dim, heads_q, heads_kv, rows):
    p = Problem([(rows, 9000), (rows, 40)], heads_q, heads_kv, dim, 32, seed=dim)
    assert p.plan().workspace_size() > 0
    p.check(p.run())


@pytest.mark.parametrize("rows", [1, 4, 150])
@pytest.mark.parametrize("gain", [0.0, 1e-30, 40.0, 3e4])
def test_attention_query_sizes(rows, gain):
    """Queries of no size, of almost none, of scores up to some hundreds (one key takes all), and of many thousands."""
    p = Problem([(rows, 600)], 4, 1, 128, 16, seed=9, q_gain=gain, scale=128 ** -0.5 if gain < 1e4 else 1e-4)
    p.check(p.run())


@pytest.mark.parametrize("rows", [1, 140])
def test_attention_value_sizes(rows):
    """Keys whose values differ by many orders, and a first token that takes the attention and says nothing."""
    p = Problem([(rows, 900)], 8, 2, 128, 16, seed=4)
    g = _gen(8)
    size = torch.exp(3.0 * _randn(g, 900, 2, 1))
    v = (_randn(g, 900, 2, 128) * size).to(BF16)
    k = _randn(g, 900, 2, 128)
    k[0] = p.q[0, :128].float() * 2
    v[0] = 0
    place = torch.arange(900, device="cuda")
    ref.fill(p.cache, 16, 2, 128, p.table[0].long()[place // 16] * 16 + place % 16, k.to(BF16), v)
    p.check(p.run())


@pytest.mark.parametrize("rows,dim", [(1, 128), (3, 64), (160, 128), (140, 256)])
def test_keys_that_no_row_may_see_can_hold_anything(rows, dim):
    """Tokens after a row's own, and before its window, hold NaN and infinity: they change nothing."""
    p = Problem([(rows, 400)], 4, 1, dim, 16, seed=2, window=64)
    clean = p.run()
    p.check(clean)
    first_seen = 400 - rows - 64 + 1
    if first_seen > 0:
        place = torch.arange(first_seen, device="cuda")
        slots = p.table[0].long()[place // 16] * 16 + place % 16
        bad = torch.full((first_seen, 1, dim), math.nan, device="cuda").to(BF16)
        ref.fill(p.cache, 16, 1, dim, slots, bad, bad)
    # the last token: seen by the last row alone
    slot = p.table[0].long()[399 // 16] * 16 + 399 % 16
    bad = torch.full((1, 1, dim), math.nan, device="cuda").to(BF16)
    ref.fill(p.cache, 16, 1, dim, slot.reshape(1), bad, bad)
    got = p.run()
    torch.cuda.synchronize()
    assert torch.equal(got.out[: rows - 1], clean.out[: rows - 1]) and torch.equal(got.lse[: rows - 1], clean.lse[: rows - 1])
    assert got.out[rows - 1].isnan().all()


@pytest.mark.parametrize("rows", [1, 150])
def test_attention_is_the_same_every_time_and_on_any_stream(rows):
    p = Problem([(rows, 3000), (rows, 200)], 8, 2, 128, 32, seed=6)
    first = p.run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = p.run()
    third = p.run(stream=stream)
    torch.cuda.synchronize()
    for other in (second, third):
        assert torch.equal(first.out, other.out) and torch.equal(first.lse, other.lse)
    p.check(first)


def test_pages_beyond_four_gigabytes():
    """A cache of which only pages behind 2^32 bytes are used: offsets are 64 bits wide."""
    dim, heads, page = 128, 8, 64
    desc = bq.Kv4CacheDescriptor(130000, page, heads, dim)
    cache = torch.empty((desc.num_pages, desc.page_bytes), dtype=torch.uint8, device="cuda")
    assert 60000 * desc.page_bytes > 2 ** 32
    p = Problem([(1, 200), (3, 64)], 16, heads, dim, page, seed=12)
    used = torch.tensor([129999, 70001, 100000, 65000], device="cuda")
    small = p.table.clone()
    new = torch.full_like(small, -1)
    k, v = torch.empty(264, heads * dim, dtype=BF16, device="cuda"), torch.empty(264, heads * dim, dtype=BF16, device="cuda")
    slots = torch.cat([small[0].long()[torch.arange(200, device="cuda") // page] * page + torch.arange(200, device="cuda") % page,
                       small[1].long()[torch.zeros(64, dtype=torch.long, device="cuda")] * page + torch.arange(64, device="cuda")])
    new[0, :4] = used.to(torch.int32)
    cache[used] = 255
    cache[used, :] = torch.stack([p.cache[int(x), : desc.page_bytes] for x in small[0, :4]])
    other = 64000
    cache[other] = p.cache[int(small[1, 0]), : desc.page_bytes]
    new[1, 0] = other
    want = p.run()
    args = bq.Kv4AttentionArgs(q=p.q, cu_q=p.cu_q, kv_lens=p.kv_lens, page_table=new, cache=cache, out=torch.empty(p.total, 16 * dim, dtype=BF16, device="cuda"))
    plan = bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(2, p.max_q, p.max_kv, 16, desc, scale=p.scale))
    plan.run(None, torch.empty(plan.workspace_size(), dtype=torch.uint8, device="cuda"), args)
    torch.cuda.synchronize()
    assert torch.equal(args.out[: p.rows], want.out[: p.rows])
    # append there and read it back
    far = torch.tensor([129999 * page + 63, 70001 * page], device="cuda")
    x = _randn(_gen(1), 2, heads * dim).to(BF16)
    _append(desc, cache, x, x, far)
    bq.Kv4ReadPlan.select(None, bq.Kv4ReadDescriptor(2, desc)).run(None, None, bq.Kv4ReadArgs(cache=cache, slots=far, k=k[:2], v=v[:2]))
    codes, s, m = ref.quantize(x.reshape(2, heads, dim))
    torch.cuda.synchronize()
    assert torch.equal(k[:2].reshape(2, heads, dim), ref.values(codes, s, m).float().to(BF16)) and torch.equal(k[:2], v[:2])
    assert bq.device_status() == 0


def test_bad_lengths_and_pages_are_reported():
    p = Problem([(1, 100), (1, 100)], 4, 1, 64, 16, seed=3)
    good = p.run()
    p.check(good)
    lens = p.kv_lens.clone()
    p.kv_lens[0] = 500  # beyond max_kv
    got = p.run()
    torch.cuda.synchronize()
    assert bq.device_status() == 403
    assert torch.equal(got.out[:2], good.out[:2])  # cut to max_kv = 100
    p.kv_lens.copy_(lens)
    for bad in (-1, p.desc.num_pages, 2 ** 31 - 1):
        table = p.table.clone()
        p.table[0, 6] = bad  # the last, partly filled page of the first sequence: 96 keys are left
        got = p.run()
        torch.cuda.synchronize()
        assert bq.device_status() == 404
        p.table.copy_(table)
        assert torch.equal(got.out[1], good.out[1])
        want, *_ = ref.attention(p.q[:1], p.cu_q[:2], torch.tensor([96]), p.table, p.cache, 16, 1, 64, p.scale, True, 0)
        assert (got.out[0].double() - want[0].flatten()).norm() <= 5e-3 * want.norm()
    assert bq.device_status() == 0


@pytest.mark.parametrize("rows", [1, 140])
def test_attention_in_a_captured_graph(rows):
    """Captured with its bounds; replayed after lengths, pages and queries changed, a sequence of no rows and one of no keys among them."""
    p = Problem([(rows, 700), (rows, 30), (rows, 64)], 8, 2, 128, 16, seed=5, max_kv=900)
    plan = p.plan()
    out = torch.zeros(p.total, 8 * 128, dtype=BF16, device="cuda")
    lse = torch.zeros(p.total, 8, device="cuda")
    args = bq.Kv4AttentionArgs(q=p.q, cu_q=p.cu_q, kv_lens=p.kv_lens, page_table=p.table, cache=p.cache, out=out, lse=lse)
    workspace = torch.empty(plan.workspace_size(), dtype=torch.uint8, device="cuda")
    plan.run(None, workspace, args)  # warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(None, workspace, args)
    for cu, lens in (([0, rows, rows, 2 * rows], [650, 30, 64]), ([0, rows, 2 * rows, 3 * rows], [700, 0, 17])):
        p.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))
        p.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        p.q.copy_(p.q.flip(0).clone())
        out.fill_(7.0)
        lse.fill_(7.0)
        graph.replay()
        n = cu[-1]
        want, want_lse, tol, _ = ref.attention(p.q[:n], p.cu_q, p.kv_lens, p.table, p.cache, 16, 2, 128, p.scale, True, 0)
        torch.cuda.synchronize()
        assert bq.device_status() == 0
        assert torch.all((out[:n].double().reshape(want.shape) - want).abs() <= tol)
        assert torch.equal(torch.isinf(lse[:n]), torch.isinf(want_lse))
        assert torch.all(out[n:] == 7) and torch.all(lse[n:] == 7)


# ------------------------------------------------------------------------------------------------ together
def test_a_layers_attention_step_between_its_quantized_projections():
    """Prompt, then drafted tokens, then single tokens: qkv projection, norm + rotation + append, attention, output projection."""
    hidden, hq, hkv, dim, page = 1024, 8, 2, 128, 32
    g = _gen(21)
    qkv_cols = (hq + 2 * hkv) * dim
    weight = {"qkv": torch.randint(-127, 128, (qkv_cols, hidden), generator=g, device="cuda", dtype=torch.int8),
              "o": torch.randint(-127, 128, (hidden, hq * dim), generator=g, device="cuda", dtype=torch.int8)}
    wscale = {n: torch.rand(w.shape[0], generator=g, device="cuda") * 0.002 + 1e-4 for n, w in weight.items()}
    qw, kw = 1 + 0.1 * _randn(g, dim), 1 + 0.1 * _randn(g, dim)
    angles = _angles(512, dim)
    longest = 400
    desc, cache = _cache(2 * -(-longest // page) + 1, page, hkv, dim)
    table = torch.randperm(desc.num_pages, generator=g, device="cuda")[: 2 * -(-longest // page)].reshape(2, -1).to(torch.int32)

    def linear(name, x):
        m, k = x.shape
        n = weight[name].shape[0]
        plan = bq.QuantizedLinearPlan.select(None, bq.QuantizedLinearDescriptor(m, n, k))
        y = torch.empty(m, n, dtype=BF16, device="cuda")
        plan.run(None, torch.empty(max(plan.workspace_size(), 16), dtype=torch.uint8, device="cuda"),
                 bq.QuantizedLinearArgs(x, weight[name], wscale[name], y, torch.empty(m, k, dtype=torch.int8, device="cuda"),
                                        torch.empty(m, dtype=torch.float32, device="cuda")))
        return y

    have = [0, 0]
    held = [[], []]  # the keys and values that each sequence should have in the cache
    for step in ([130, 57], [4, 4], [1, 1], [1, 1]):
        t = sum(step)
        x = _randn(g, t, hidden).to(BF16)
        qkv = linear("qkv", x)
        q, k, v = qkv[:, : hq * dim], qkv[:, hq * dim : (hq + hkv) * dim], qkv[:, (hq + hkv) * dim :]
        place = torch.cat([torch.arange(have[i], have[i] + step[i], device="cuda") for i in range(2)])
        seq = torch.repeat_interleave(torch.arange(2, device="cuda"), torch.tensor(step, device="cuda"))
        slots = table[seq, place // page].long() * page + place % page
        q_out = torch.empty(t, hq * dim, dtype=BF16, device="cuda")
        positions = place.to(torch.int32)
        bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(t, hq, hkv, dim, cache=desc)).run(None, None, bq.QkNormRopeArgs(
            q=q, k=k, v=v, q_out=q_out, q_weight=qw, k_weight=kw, cos_sin=angles, positions=positions, cache=cache, slots=slots))
        have = [a + b for a, b in zip(have, step)]
        kv_lens = torch.tensor(have, dtype=torch.int32, device="cuda")
        cu_q = torch.tensor([0, step[0], t], dtype=torch.int32, device="cuda")
        plan = bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(2, max(step), longest, hq, desc))
        out = torch.empty(t, hq * dim, dtype=BF16, device="cuda")
        plan.run(None, torch.empty(plan.workspace_size(), dtype=torch.uint8, device="cuda"), bq.Kv4AttentionArgs(
            q=q_out, cu_q=cu_q, kv_lens=kv_lens, page_table=table, cache=cache, out=out))
        y = linear("o", out)
        torch.cuda.synchronize()
        assert bq.device_status() == 0
        want_q, tol_q = ref.norm_rope(q, hq, dim, qw, 1e-6, angles, positions[None], None, dim, False)
        assert torch.all((q_out.double().reshape(want_q.shape) - want_q).abs() <= tol_q)
        # the cache holds every token so far: values by the format, keys within a code of the 64-bit ones
        want_k, _ = ref.norm_rope(k, hkv, dim, kw, 1e-6, angles, positions[None], None, dim, False)
        codes, s, m = ref.unpack(cache, page, hkv, dim)
        vc, vs, vm = ref.quantize(v.reshape(t, hkv, dim))
        assert torch.equal(codes[1, slots], vc) and torch.equal(s[1, slots], vs) and torch.equal(m[1, slots], vm)
        got_k = ref.values(codes[0, slots], s[0, slots], m[0, slots])
        assert torch.all((got_k - want_k).abs() <= s[0, slots].repeat_interleave(64, -1) * 0.51 + want_k.abs() * 2 * ref.HALF_BF16 + want_k.abs().amax(-1, keepdim=True) * 2 * ref.HALF_BF16)
        want, _, tol, _ = ref.attention(q_out, cu_q, kv_lens, table, cache, page, hkv, dim, dim ** -0.5, True, 0)
        assert torch.all((out.double().reshape(want.shape) - want).abs() <= tol)
        assert torch.isfinite(y).all() and y.abs().amax() > 0


def test_norm_and_rotation_round_step_by_step():
    """The stated f32 steps of the keys, each rounded once, in plain torch operations: the same bits (the cache's codes depend on them)."""
    t, heads, dim = 3000, 8, 128
    g = _gen(17)
    x = (_randn(g, t, (heads + 1) * dim) * torch.exp(_randn(g, (heads + 1) * dim))).to(BF16)
    k, q = x[:, : heads * dim], x[:, heads * dim :]
    w = 1 + 0.3 * _randn(g, dim)
    angles = _angles(1000, dim)
    positions = torch.randint(0, 1000, (t,), generator=g, device="cuda", dtype=torch.int32)
    for interleaved in (False, True):
        for weight in (w, None):
            q_out, k_out = torch.empty_like(q), torch.empty_like(k)
            bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(t, 1, heads, dim, interleaved=interleaved, eps=1e-6)).run(
                None, None, bq.QkNormRopeArgs(q=q, k=k, q_out=q_out, k_out=k_out, q_weight=weight, k_weight=weight, cos_sin=angles, positions=positions))
            y = k.reshape(t, heads, dim)
            if weight is not None:
                mean = (y.double().square().sum(-1, keepdim=True) / dim).float()
                y = y.float() * (1.0 / torch.sqrt(mean + 1e-6)) * weight
            y = y.float()
            c, s = angles[positions.long()][:, None].chunk(2, -1)
            a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else y.chunk(2, -1)
            one, two = a * c - b * s, b * c + a * s
            want = torch.stack([one, two], -1).flatten(-2) if interleaved else torch.cat([one, two], -1)
            assert torch.equal(k_out.reshape(t, heads, dim), want.to(BF16))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_without_keys(dim):
    """Whole blocks of rows that see nothing, many of them at once and again and again: zeros, every time."""
    p = Problem([(200, 30), (150, 0), (140, 20), (300, 64)], 8, 2, dim, 16, seed=31)
    first = p.run()
    p.check(first)
    for _ in range(30):
        again = p.run()
        assert torch.equal(again.out, first.out) and torch.equal(again.lse, first.lse)


@pytest.mark.parametrize("dim,page,start,tokens", [(64, 16, 0, 16), (128, 32, 5, 100), (128, 64, 15, 1), (256, 48, 33, 300), (64, 128, 127, 130), (128, 16, 8, 8)])
def test_read_of_a_sequences_tokens(dim, page, start, tokens):
    """Slots of a sequence, beginning and ending inside tiles, its pages in no order: the values, and the rows beside them untouched."""
    g = _gen(start + tokens)
    heads = 3
    pages = -(-(start + tokens) // page) + 2
    desc, cache = _cache(pages, page, heads, dim)
    cache.random_(0, 256, generator=g)
    codes, s, m = ref.unpack(cache, page, heads, dim)
    order = torch.randperm(pages, generator=g, device="cuda")
    place = torch.arange(start, start + tokens, device="cuda")
    slots = order[place // page] * page + place % page
    out = torch.full((2, tokens + 2, heads * dim), 7.0, dtype=BF16, device="cuda")
    bq.Kv4ReadPlan.select(None, bq.Kv4ReadDescriptor(tokens, desc)).run(None, None, bq.Kv4ReadArgs(cache=cache, slots=slots, k=out[0, 1:-1], v=out[1, 1:-1]))
    torch.cuda.synchronize()
    for which in (0, 1):
        want = ref.values(codes[which], s[which], m[which]).float().to(BF16)[slots].flatten(1)
        got = out[which, 1:-1]
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        assert torch.all(out[which, 0] == 7) and torch.all(out[which, -1] == 7)
    assert bq.device_status() == 0


# ------------------------------------------------------------------------------------------------ large batches, holes, two at once
@pytest.mark.parametrize("batch,dim,heads_q,heads_kv,most_rows", [(33, 128, 4, 1, 1), (128, 64, 2, 2, 3), (129, 256, 2, 1, 2), (300, 128, 16, 2, 2), (1000, 64, 1, 1, 1)])
def test_many_sequences(batch, dim, heads_q, heads_kv, most_rows):
    """More sequences than a warp, and than a block, looks at in one go, of very different lengths; some without rows, some without keys."""
    g = torch.Generator().manual_seed(batch)
    rows = torch.randint(0, most_rows + 1, (batch,), generator=g).tolist()
    lens = (torch.rand(batch, generator=g) ** 4 * 900).int().tolist()
    rows[0] = rows[-1] = most_rows
    p = Problem(list(zip(rows, lens)), heads_q, heads_kv, dim, 16, seed=batch)
    p.check(p.run())


def test_many_prompts():
    p = Problem([(40 + 37 * i % 100, 30 + 91 * i % 400) for i in range(40)], 4, 2, 64, 16, seed=40)
    p.check(p.run())


@pytest.mark.parametrize("rows,dim", [(1, 64), (1, 128), (3, 256), (20, 128), (100, 128), (200, 128), (160, 64), (20, 64), (140, 256)])
def test_pages_that_are_missing_inside_leave_their_keys_out(rows, dim):
    """Of 400 keys the pages of 48..79 and 320..335 have no number: what is seen is the rest."""
    page, heads_q, heads_kv = 16, 4, 2
    p = Problem([(rows, 400)], heads_q, heads_kv, dim, page, seed=rows)
    keys = [j for j in range(400) if j // page not in (3, 4, 20)]
    values = ref.values(*(x[:, p.table[0].long()[torch.tensor(keys, device="cuda") // page] * page + torch.tensor(keys, device="cuda") % page]
                          for x in ref.unpack(p.cache, page, heads_kv, dim))).double()
    table = p.table.clone()
    p.table[0, 3], p.table[0, 4], p.table[0, 20] = -1, p.desc.num_pages, 2 ** 31 - 1
    got = p.run()
    torch.cuda.synchronize()
    assert bq.device_status() == 404 and bq.device_status() == 0
    k, v = (x.repeat_interleave(heads_q // heads_kv, 1) for x in values)
    q = p.q[:rows].double().reshape(rows, heads_q, dim)
    score = torch.einsum("ihd,jhd->hij", q, k) * p.scale
    seen = torch.tensor(keys, device="cuda")[None, :] <= 400 - rows + torch.arange(rows, device="cuda")[:, None]
    weight = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
    want = torch.einsum("hij,jhd->ihd", weight, v)
    # all roundings together: bf16 of the output, f16 of keys, values and weights
    err = (got.out[:rows].double().reshape(want.shape) - want).norm() / want.norm()
    assert float(err) <= 2.0 ** -8 / math.sqrt(3.0) + 4 * 2.0 ** -11
    p.table.copy_(table)
    p.check(p.run())


@pytest.mark.parametrize("rows,dim", [(1, 64), (1, 128), (3, 256), (20, 128), (200, 128), (160, 64), (140, 256)])
@pytest.mark.parametrize("what", ["key", "value"])
def test_a_nan_reaches_the_rows_that_see_it_and_no_other(rows, dim, what):
    page, at = 16, 400 - rows + rows // 2
    p = Problem([(rows, 400), (rows, 30)], 2, 1, dim, page, seed=rows + dim)
    clean = p.run()
    codes, s, m = ref.unpack(p.cache, page, 1, dim)
    slot = p.table[0].long()[at // page] * page + at % page
    k, v = (ref.values(codes[i], s[i], m[i])[slot].reshape(1, 1, dim).to(BF16) for i in (0, 1))
    (k if what == "key" else v)[0, 0, 5] = math.nan
    ref.fill(p.cache, page, 1, dim, slot.reshape(1), k, v)
    got = p.run()
    torch.cuda.synchronize()
    sees = 400 - rows + torch.arange(rows, device="cuda") >= at
    out, before = (x.out[:rows].reshape(rows, 2, dim) for x in (got, clean))
    assert out[sees][:, :, :64].isnan().all()
    assert what == "value" or out[sees].isnan().all()
    assert torch.equal(out[~sees], before[~sees])
    assert torch.equal(got.out[rows:], clean.out[rows:])
    assert bq.device_status() == 0


def test_two_streams_at_once():
    """Calls on two streams, each with a workspace of its own, leave what they leave one after the other."""
    problems = [Problem([(1, 5000), (2, 3000)], 8, 2, 128, 32, seed=1), Problem([(150, 2000)], 8, 2, 128, 32, seed=2)]
    alone = [p.run() for p in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    plans = [p.plan() for p in problems]
    spaces = [torch.empty(max(1, plan.workspace_size()), dtype=torch.uint8, device="cuda") for plan in plans]
    outs = [[torch.zeros_like(a.out) for _ in range(10)] for a in alone]
    torch.cuda.synchronize()
    for i in range(10):
        for p, plan, stream, space, out in zip(problems, plans, streams, spaces, outs):
            plan.run(stream, space, bq.Kv4AttentionArgs(q=p.q, cu_q=p.cu_q, kv_lens=p.kv_lens, page_table=p.table, cache=p.cache, out=out[i]))
    torch.cuda.synchronize()
    for p, a, out in zip(problems, alone, outs):
        assert all(torch.equal(o[: p.rows], a.out[: p.rows]) for o in out)
    assert bq.device_status() == 0


@pytest.mark.parametrize("lens,heads_q,heads_kv,dim,window", [([(600, 3000), (300, 2500), (500, 1100)], 16, 2, 256, 900),
                                                              ([(700, 700), (200, 2000)], 8, 2, 256, 0),
                                                              ([(12, 1000 + 37 * i) for i in range(60)], 16, 2, 128, 0),
                                                              ([(16, 900 + 41 * i) for i in range(50)], 12, 2, 64, 0),
                                                              ([(900, 1500), (400, 1900)], 16, 2, 128, 600)])
def test_blocks_whose_warps_run_apart_agree_every_time(lens, heads_q, heads_kv, dim, window):
    """Many blocks of many steps: the warps of a block drift apart by a step, and no row may be taken before its last product."""
    p = Problem(lens, heads_q, heads_kv, dim, 16, seed=dim, window=window)
    first = p.run()
    p.check(first)
    for _ in range(25):
        again = p.run()
        assert torch.equal(again.out, first.out) and torch.equal(again.lse, first.lse)


@pytest.mark.parametrize("dim,rot,interleaved", [(64, 64, False), (128, 128, True), (256, 64, False)])
@pytest.mark.parametrize("tokens", [1, 37, 1500])
@pytest.mark.parametrize("weights", ["q", "k"])
def test_norm_of_one_side_keys_alone_and_rows_on_eight_bytes(tokens, dim, rot, interleaved, weights):
    """Only queries or only keys are normed; no queries at all; matrices that begin and step by 8 bytes."""
    hq, hkv = 9, 3
    qkv, (wq, wk), positions, _, angles = _norm_inputs(tokens, hq, hkv, dim, rot, None, tokens + dim)
    wide = torch.full((tokens, qkv.shape[1] + 12), 3.0, dtype=BF16, device="cuda")
    wide[:, 4:-8] = qkv
    q, k = wide[:, 4 : 4 + hq * dim], wide[:, 4 + hq * dim : 4 + (hq + hkv) * dim]
    wq, wk = (wq, None) if weights == "q" else (None, wk)
    out = torch.full((tokens, (hq + hkv) * dim + 4), 7.0, dtype=BF16, device="cuda")
    args = bq.QkNormRopeArgs(q=q, k=k, q_out=out[:, 4 : 4 + hq * dim], k_out=out[:, 4 + hq * dim :], q_weight=wq, k_weight=wk, cos_sin=angles, positions=positions)
    bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(tokens, hq, hkv, dim, rot_dim=rot, interleaved=interleaved)).run(None, None, args)
    alone = torch.empty(tokens, hkv * dim, dtype=BF16, device="cuda")
    bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(tokens, 0, hkv, dim, rot_dim=rot, interleaved=interleaved)).run(
        None, None, bq.QkNormRopeArgs(q=None, k=k, k_out=alone, k_weight=wk, cos_sin=angles, positions=positions))
    torch.cuda.synchronize()
    assert bq.device_status() == 0
    for x, got, heads, w in ((q, args.q_out, hq, wq), (k, args.k_out, hkv, wk), (k, alone, hkv, wk)):
        want, tol = ref.norm_rope(x, heads, dim, w, 1e-6, angles, positions, None, rot, interleaved)
        assert torch.all((got.double().reshape(want.shape) - want).abs() <= tol)
    assert torch.equal(alone, args.k_out) and torch.all(out[:, :4] == 7) and torch.all(wide[:, :4] == 3) and torch.all(wide[:, -8:] == 3)


def test_a_captured_step_with_a_padded_batch():
    """Norm, rotation and append, then attention, captured once; replayed with other tokens, positions, slots and lengths, and rows of
    padding: they write nothing to the cache and get zeros."""
    hq, hkv, dim, page, batch = 8, 2, 128, 16, 6
    desc, cache = _cache(40, page, hkv, dim)
    qkv, (wq, wk), positions, _, angles = _norm_inputs(batch, hq, hkv, dim, dim, None, 8)
    q, k, v = qkv[:, : hq * dim], qkv[:, hq * dim : (hq + hkv) * dim], qkv[:, (hq + hkv) * dim :]
    slots, lens = torch.full((batch,), -1, device="cuda"), torch.zeros(batch, dtype=torch.int32, device="cuda")
    table = torch.arange(36, dtype=torch.int32, device="cuda").reshape(batch, 6)
    q_out, out = torch.empty(batch, hq * dim, dtype=BF16, device="cuda"), torch.empty(batch, hq * dim, dtype=BF16, device="cuda")
    rope = bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(batch, hq, hkv, dim, cache=desc))
    attend = bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(batch, 1, 6 * page, hq, desc))
    space = torch.empty(attend.workspace_size(), dtype=torch.uint8, device="cuda")
    rope_args = bq.QkNormRopeArgs(q=q, k=k, v=v, q_out=q_out, q_weight=wq, k_weight=wk, cos_sin=angles, positions=positions, cache=cache, slots=slots)
    attend_args = bq.Kv4AttentionArgs(q=q_out, cu_q=torch.arange(batch + 1, dtype=torch.int32, device="cuda"), kv_lens=lens, page_table=table,
                                      cache=cache, out=out)

    def step():
        rope.run(None, None, rope_args)
        attend.run(None, space, attend_args)

    step()
    torch.cuda.synchronize()
    empty = cache.clone()
    assert torch.all(cache == 255) and not out.any()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = _gen(77)
    held = torch.zeros(batch, dtype=torch.long)
    for i in range(20):
        live = torch.tensor([(i + b) % 3 != 0 and b != 4 for b in range(batch)])  # sequence 4 is padding throughout
        qkv.copy_(_randn(g, *qkv.shape).to(BF16))
        slots.copy_(torch.where(live, table[:, 0].cpu().long() * page + held, -1))
        held += live
        positions[0].copy_(held.to(torch.int32))
        lens.copy_(torch.where(live, held, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert bq.device_status() == 0
        want, _, tol, _ = ref.attention(q_out, attend_args.cu_q, lens, table, cache, page, hkv, dim, dim ** -0.5, True, 0)
        assert torch.all((out.double().reshape(want.shape) - want).abs() <= tol)
        assert not out[~live.cuda()].any()
    assert torch.equal(cache[24:30], empty[24:30]) and torch.equal(cache[36:], empty[36:])


# ------------------------------------------------------------------------------------------------ far ends of the ranges
@pytest.mark.parametrize("rows,dim", [(60, 64), (160, 64), (60, 128), (200, 128), (140, 256)])
def test_a_nan_key_reaches_every_row_wherever_it_lies_in_its_tile(rows, dim):
    """Each of the 16 places, in a step that all rows see in full and that comes when the softmax's reference has settled; the values are numbers."""
    page, first = 16, 256
    p = Problem([(rows, 700)], 2, 1, dim, page, seed=rows + dim)
    p.check(p.run())
    clean = p.cache.clone()
    codes, s, m = ref.unpack(p.cache, page, 1, dim)
    for place in range(16):
        slot = p.table[0].long()[first // page] * page + place
        k, v = (ref.values(codes[i], s[i], m[i])[slot].reshape(1, 1, dim).to(BF16) for i in (0, 1))
        k[0, 0, 7] = math.nan
        p.cache.copy_(clean)
        ref.fill(p.cache, page, 1, dim, slot.reshape(1), k, v)
        got = p.run()
        torch.cuda.synchronize()
        assert got.out[:rows].isnan().all() and got.lse[:rows].isnan().all(), place
    assert bq.device_status() == 0


@pytest.mark.parametrize("lens,heads_q,heads_kv,dim,statuses", [([(1, 600)] * 300, 4, 2, 128, (411,)), ([(3, 400 + 31 * i) for i in range(40)], 4, 4, 64, (411,)),
                                                                ([(2, 20000)], 2, 1, 256, (411,)), ([(200, 900), (150, 400)], 4, 2, 128, range(412, 417)),
                                                                ([(60, 2000)], 2, 1, 64, range(412, 417)), ([(140, 700), (40, 300)], 2, 1, 256, range(412, 417))])
def test_waits_that_run_out_are_reported(qlib, lens, heads_q, heads_kv, dim, statuses):
    """Barriers that nothing completes: the call ends with a status, whatever the workspace held, writes to its sequences' rows alone, and
    the next call is as good as any."""
    p = Problem(lens, heads_q, heads_kv, dim, 16, seed=len(lens))
    good = p.run()
    p.check(good)
    plan = p.plan()
    g = _gen(2)
    for fill in (0, 0x7F, 0x80, 0xFF, None):
        space = torch.full((max(1, plan.workspace_size()),), fill or 0, dtype=torch.uint8, device="cuda")
        if fill is None:
            space.random_(0, 256, generator=g)
        out, lse = torch.full_like(good.out._base, 7.0), torch.full_like(good.lse, 7.0)
        args = bq.Kv4AttentionArgs(q=p.q, cu_q=p.cu_q, kv_lens=p.kv_lens, page_table=p.table, cache=p.cache, out=out[:, : heads_q * dim], lse=lse)
        assert qlib.baracuda_kernels_q_selftest_kv4_waits(1 << 21) == 0  # about a millisecond
        try:
            plan.run(None, space, args)
        finally:
            assert qlib.baracuda_kernels_q_selftest_kv4_waits(0) == 0
        torch.cuda.synchronize()
        assert bq.device_status() in statuses and bq.device_status() == 0
        assert torch.all(out[p.rows :] == 7) and torch.all(lse[p.rows :] == 7) and torch.all(out[:, heads_q * dim :] == 7)
    again = p.run()
    p.check(again)
    assert torch.equal(again.out, good.out) and torch.equal(again.lse, good.lse)


@pytest.mark.parametrize("lens,heads_q,dim", [([(9, 4), (1, 30)], 2, 128), ([(6, 1), (7, 70)], 3, 64), ([(5, 0), (8, 2)], 2, 256),
                                              ([(100, 60), (30, 90)], 4, 128), ([(90, 7), (140, 300)], 2, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_window_of_any_size_and_fewer_keys_than_rows(lens, heads_q, dim, causal):
    """Windows up to the largest number limit nothing, also where the first rows come before the first key."""
    p = Problem(lens, heads_q, 1, dim, 16, seed=dim, causal=causal)
    free = p.run()
    p.check(free)
    for window in (300, 2 ** 31 - 9, 2 ** 31 - 1):
        p.window = window
        got = p.run()
        p.check(got)
        assert torch.equal(got.out, free.out) and torch.equal(got.lse, free.lse)


@pytest.mark.parametrize("rows,dim", [(1, 64), (1, 128), (3, 256), (20, 128), (160, 64), (200, 128), (140, 256)])
def test_pages_before_every_rows_window_need_not_exist(rows, dim):
    """A sequence gives up the pages that no row sees any more: neither their keys nor their numbers are looked at."""
    page, length, window = 16, 730, 100
    p = Problem([(rows, length), (1, 50)], 4, 2, dim, page, seed=rows, window=window)
    clean = p.run()
    p.check(clean)
    gone = (length - rows - window + 1) // page
    for number in (-1, p.desc.num_pages, 2 ** 31 - 1):
        p.table[0, :gone] = number
        got = p.run()
        torch.cuda.synchronize()
        assert bq.device_status() == 0
        assert torch.equal(got.out, clean.out) and torch.equal(got.lse, clean.lse)
    p.table[0, gone] = -1  # the first of which something is seen
    p.run()
    torch.cuda.synchronize()
    assert bq.device_status() == 404


@pytest.mark.parametrize("dim,interleaved", [(64, False), (128, True), (256, False)])
@pytest.mark.parametrize("tokens", [7, 1500])
def test_norm_of_heads_beyond_the_range(tokens, dim, interleaved):
    """A sum of squares beyond f32 is infinite: the head's numbers become 0, an infinite channel and its partner in the rotation NaN; a NaN
    takes the whole head.  Queries and keys alike, and nothing of it reaches another head."""
    heads = 12
    g = _gen(dim)
    x = _randn(g, tokens, 2 * heads, dim).to(BF16)
    for at in (0, heads):  # some heads of a token among ordinary ones
        x[3, at] = 3e38
        x[3, at + 2, 5] = math.inf
        x[3, at + 4, dim - 1] = -math.inf
        x[3, at + 5] = 1e19
        x[3, at + 7, 9] = 2e19
        x[3, at + 8, 11] = math.nan
    x = x.flatten(1)
    q, k = x[:, : heads * dim], x[:, heads * dim :]
    w = 1 + 0.3 * _randn(g, dim)
    angles = _angles(1000, dim)
    positions = torch.randint(0, 1000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(tokens, heads, heads, dim, interleaved=interleaved)).run(
        None, None, bq.QkNormRopeArgs(q=q, k=k, q_out=q_out, k_out=k_out, q_weight=w, k_weight=w, cos_sin=angles, positions=positions))
    torch.cuda.synchronize()
    for given, got in ((q, q_out), (k, k_out)):
        y = given.reshape(tokens, heads, dim).float()
        y = y * (1.0 / torch.sqrt(y.square().sum(-1, keepdim=True) / dim + 1e-6)) * w
        c, s = angles[positions.long()][:, None].chunk(2, -1)
        a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else y.chunk(2, -1)
        one, two = a * c - b * s, b * c + a * s
        want = torch.stack([one, two], -1).flatten(-2) if interleaved else torch.cat([one, two], -1)
        got = got.reshape(want.shape).float()
        assert torch.equal(got.isnan(), want.isnan())
        assert not got[3, 0].any() and not got[3, 5].any() and not got[3, 7].any() and got[3, 8].isnan().all()
        assert int(got[3, 2].isnan().sum()) == 2 and int(got[3, 4].isnan().sum()) == 2
        # the ordinary heads: 8 roundings of f32 and one of bf16 over two terms, as in the tests above
        live = torch.tensor([h for h in range(heads) if h not in (0, 2, 4, 5, 7, 8)], device="cuda")
        true, tol = ref.norm_rope(given.reshape(tokens, heads, dim)[:, live].flatten(1), len(live), dim, w, 1e-6, angles, positions, None, dim, interleaved)
        assert torch.all((got[:, live].double() - true).abs() <= tol)


@pytest.mark.parametrize("rows,dim", [(1, 64), (1, 128), (2, 256), (60, 128), (150, 64), (150, 128), (140, 256)])
@pytest.mark.parametrize("gain", [1e5, 1e8, 1e12, 1e33])
@pytest.mark.parametrize("length", [1, 400])
def test_attention_of_far_scores_takes_one_key(rows, dim, gain, length):
    """Scores far beyond what f32 holds to a unit, of either sign: where one is ahead its value comes out; of a single key, always."""
    p = Problem([(rows, length)], 2, 1, dim, 16, seed=dim, q_gain=1.0, causal=False)
    p.q.copy_(p.q.float() * gain)
    got = p.run()
    codes, s, m = ref.unpack(p.cache, 16, 1, dim)
    place = torch.arange(length, device="cuda")
    slots = p.table[0].long()[place // 16] * 16 + place % 16
    k, v = (ref.values(codes[i, slots, 0], s[i, slots, 0], m[i, slots, 0]) for i in (0, 1))
    x, mag = p.q[:rows].double().reshape(rows, 2, dim), ref.values(codes[0, slots, 0], s[0, slots, 0], m[0, slots, 0].abs())
    top, best = torch.nn.functional.pad(x @ k.T, (0, 1), value=-math.inf).topk(2, -1)
    # ahead by more than the roundings of two scores (as the reference counts them) and 40 nats
    off = (x.abs() @ mag.T).amax(-1) * ((dim + 8) * 2.0 ** -23 + 2 * ref.HALF_F16)
    sure = (top[..., 0] - top[..., 1] - 2 * off) * p.scale > 40.0
    assert sure.any()
    torch.cuda.synchronize()
    want = v[best[..., 0]]
    # one weight of 1: codes, scale and minimum in f16 products and f32 sums, one rounding to f16 at most, then bf16
    err = (got.out[:rows].double().reshape(want.shape) - want).abs()
    assert torch.isfinite(got.out[:rows]).all() and torch.all(err[sure] <= (2.0 ** -8 * want.abs() + 2.0 ** -10 * v.abs().amax())[sure])
    lse = top[..., 0] * p.scale
    assert torch.all((got.lse[:rows].double() - lse).abs()[sure] <= (off * p.scale + 2.0 ** -20 * lse.abs())[sure])
    assert bq.device_status() == 0


@pytest.mark.parametrize("rows,dim", [(1, 64), (2, 128), (3, 256), (150, 64), (150, 128), (140, 256)])
@pytest.mark.parametrize("gain,scale", [(1e36, 1e-37), (5e37, 2e-38), (2e34, 1e-35)])
def test_attention_of_the_largest_queries(rows, dim, gain, scale):
    """Queries up to the largest bf16 numbers, under a scale that makes ordinary scores of them."""
    p = Problem([(rows, 300)], 4, 2, dim, 16, seed=rows, q_gain=1.0, scale=scale)
    p.q.copy_((p.q.float() * gain).clamp(-3.3e38, 3.3e38))
    p.q[0, :5] = 3.3e38 if gain == 5e37 else p.q[0, :5]
    p.check(p.run())


@pytest.mark.parametrize("rows,dim", [(1, 64), (1, 128), (2, 256), (150, 64), (150, 128), (140, 256)])
def test_the_largest_queries_over_a_single_key(rows, dim):
    """Queries of 1e36 under the usual scale, scores of either sign: of one key the value comes out."""
    p = Problem([(rows, 1)], 2, 1, dim, 16, seed=dim, q_gain=1.0, causal=False)
    p.q.copy_(p.q.float() * 1e36)
    got = p.run(lse=False)
    codes, s, m = ref.unpack(p.cache, 16, 1, dim)
    slot = p.table[0, 0].long() * 16
    want = ref.values(codes[1, slot, 0], s[1, slot, 0], m[1, slot, 0])
    torch.cuda.synchronize()
    err = (got.out[:rows].double().reshape(rows, 2, dim) - want).abs()
    assert torch.all(err <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * want.abs().amax())
    assert bq.device_status() == 0
