"""GPU: fragment attention (ai2bmd_amd/attention.py) against its formula in 64 bits, fragment by fragment.

Tolerances come with the reference: next to every value it sums, in 64 bits, what float32 arithmetic and the roundings to
the rows' type may do to it (first order, times 1.1).  e = 2^-24 is half a float32 step, u = eps(T) / 2 half a step of T.
  score      e_s  = e ((D + 4) scale sum|q k| + 6 slope r + |table| + 2 |s|)          products, root, sums
  P          e_p  = e_s + max_j e_s + e (3 |s - m| + n / 16 + 40), relative           exponent, sum over n keys
  a product  each factor P, dS rounded to T first (u, float32: 0), then sums of n terms in n / 16 + 8 steps
  float16    what lies under 2^-14 has an absolute step: 2^-25 of P in the forward product, 2^-39 in the backward one,
             2^-38 of a column's largest dS; and a result under 2^-14 is a multiple of 2^-24: off by up to 2^-25"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def unit(t):
    return torch.finfo(t).eps / 2


class Case:
    def __init__(self, sizes, T, heads=8, kv=None, dim=32, slope=True, lut=None, queries=None, extra=0, seed=0, spread=1.0, buckets=None):
        self.T, self.heads, self.kv, self.dim = T, heads, kv or heads, dim
        gen = torch.Generator(device="cuda").manual_seed(seed + 1000 * dim + heads)
        normal = lambda *s, t=T, by=1.0: (torch.randn(*s, generator=gen, device="cuda") * by).to(t)
        self.end = np.cumsum(sizes)
        self.start = self.end - np.asarray(sizes)
        self.apart = queries is not None
        self.q_end = np.cumsum(queries) if self.apart else self.end
        self.q_start = self.q_end - np.asarray(queries) if self.apart else self.start
        nk, nq = int(self.end[-1]) + extra, int(self.q_end[-1]) + extra
        self.q, self.k, self.v = normal(nq, heads, dim, by=spread), normal(nk, self.kv, dim), normal(nk, self.kv, dim)
        self.dout = normal(nq, heads, dim)
        self.terms = {}
        f32 = torch.float32
        if slope:
            self.terms.update(pos=normal(nk, 3, t=f32, by=6.0), slope=torch.linspace(0.02, 0.6, heads, device="cuda"))
            if self.apart:
                self.terms["query_pos"] = normal(nq, 3, t=f32, by=4.0)
        self.lut = lut
        if lut is not None:
            self.buckets = int(max(lut)) + 1 if buckets is None else buckets
            self.terms.update(residue=(torch.arange(nk, device="cuda") // 5).int(), table=normal(heads, self.buckets, t=f32, by=0.7))
            if self.apart:
                self.terms["query_residue"] = torch.randint(0, 20, (nq,), generator=gen, device="cuda", dtype=torch.int32)

    def plan(self, **more):
        from ai2bmd_amd.attention import FragmentAttention
        if self.apart:
            more.update(query_start=self.q_start, query_end=self.q_end)
        if self.lut is not None:
            more.update(buckets=self.lut, num_buckets=self.buckets)
        return FragmentAttention(self.start, self.end, self.heads, self.dim, num_kv_heads=self.kv, **more)

    def reference(self, scale=None):
        """{name: (value, bound)}, both float64"""
        T, H, share, D = self.T, self.heads, self.heads // self.kv, self.dim
        scale = D ** -0.5 if scale is None else scale
        t = {n: (x.double() if x.is_floating_point() else x) for n, x in self.terms.items()}
        u, up, half = unit(T), (0.0 if T == torch.float32 else unit(T)), T == torch.float16
        zero = lambda *s: [torch.zeros(*s, dtype=torch.float64, device="cuda") for _ in range(2)]
        res = {"out": zero(*self.q.shape), "dq": zero(*self.q.shape), "dk": zero(*self.k.shape), "dv": zero(*self.k.shape)}
        if "pos" in t:
            res.update(dslope=zero(H), dpos=zero(self.k.shape[0], 3))
            if self.apart:
                res["dquery_pos"] = zero(self.q.shape[0], 3)
        if "table" in t:
            res["dtable"] = zero(H, self.buckets)
        for f in range(len(self.end)):
            a, b, c, d = int(self.q_start[f]), int(self.q_end[f]), int(self.start[f]), int(self.end[f])
            n, m_ = d - c, b - a
            if n == 0 or m_ == 0:
                continue
            q, do = self.q[a:b].double().transpose(0, 1), self.dout[a:b].double().transpose(0, 1)
            k = self.k[c:d].double().transpose(0, 1).repeat_interleave(share, 0)
            v = self.v[c:d].double().transpose(0, 1).repeat_interleave(share, 0)
            kt, vt = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
            s = scale * (q @ kt)
            es = (D + 4) * scale * (q.abs() @ kt.abs())
            if "pos" in t:
                off = t.get("query_pos", t["pos"])[a:b, None] - t["pos"][None, c:d]
                r = off.pow(2).sum(-1).sqrt()
                s = s - t["slope"][:, None, None] * r
                es = es + 6 * t["slope"].abs()[:, None, None] * r
            if "table" in t:
                R = len(self.lut) // 2
                here = t.get("query_residue", t["residue"])[a:b].long()
                kind = torch.as_tensor(np.asarray(self.lut), device="cuda").long()[(t["residue"][c:d].long()[None] - here[:, None]).clamp(-R, R) + R]
                s = s + t["table"][:, kind]
                es = es + torch.nan_to_num(t["table"][:, kind].abs(), posinf=0.0)
            fine = torch.isfinite(s)
            es = E * (es + 2 * torch.where(fine, s.abs(), 0.0))
            top = s.amax(-1, keepdim=True)
            top = torch.where(torch.isinf(top), 0.0, top)
            p = (s - top).exp()
            l = p.sum(-1, keepdim=True)
            p = p / torch.where(l == 0, 1.0, l)
            steps = E * (n / 16 + 8)
            ep = es + es.amax(-1, keepdim=True) + E * (3 * torch.where(fine, (s - top).abs(), 0.0) + n / 16 + 40)
            out = p @ v
            eo = (p * (up + ep + steps)) @ v.abs() + (2.0 ** -25 * v.abs().sum(1, keepdim=True) if half else 0)
            res["out"][0][a:b], res["out"][1][a:b] = out.transpose(0, 1), (eo + u * out.abs()).transpose(0, 1)
            dp = do @ vt
            edp = E * (D + 4) * (do.abs() @ vt.abs())
            delta = (p * dp).sum(-1, keepdim=True)
            edelta = (p * (dp.abs() * (ep + steps) + edp)).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            eds = p * ((dp.abs() + delta.abs()) * (ep + 4 * E) + edp + edelta)
            dq = scale * (ds @ k)
            edq = scale * ((eds + ds.abs() * (up + steps)) @ k.abs())
            if half:
                edq = edq + scale * 2.0 ** -38 * ds.abs().amax(-1, keepdim=True) * k.abs().sum(1, keepdim=True)
            res["dq"][0][a:b], res["dq"][1][a:b] = dq.transpose(0, 1), (edq + u * dq.abs()).transpose(0, 1)
            qsteps = E * (m_ * share / 16 + 8)
            dst, edst = ds.transpose(1, 2).contiguous(), (eds + ds.abs() * (up + qsteps)).transpose(1, 2).contiguous()
            dk, edk = scale * (dst @ q), scale * (edst @ q.abs())
            dv = p.transpose(1, 2).contiguous() @ do
            edv = (p * (up + ep + qsteps)).transpose(1, 2).contiguous() @ do.abs()
            if half:
                edk = edk + scale * 2.0 ** -38 * ds.abs().amax(1)[..., None] * q.abs().sum(1, keepdim=True)
                edv = edv + 2.0 ** -39 * do.abs().sum(1, keepdim=True)
            for name, x, e in (("dk", dk, edk), ("dv", dv, edv)):
                x, e = (y.view(self.kv, share, n, D).sum(1).transpose(0, 1) for y in (x, e))
                res[name][0][c:d], res[name][1][c:d] = x, e + u * x.abs()
            total = E * (n + 300)  # steps of the sums that run over many rows
            if "pos" in t:
                res["dslope"][0] -= (ds * r).sum((1, 2))
                res["dslope"][1] += ((eds + ds.abs() * total) * r).sum((1, 2))
                way = off / torch.where(r == 0, 1.0, r)[..., None]
                pull = -(t["slope"][:, None, None] * ds).sum(0)[..., None] * way
                epull = (t["slope"].abs()[:, None, None] * (eds + ds.abs() * total)).sum(0)[..., None] * (way.abs() + 4 * E)
                mine = res["dquery_pos" if self.apart else "dpos"]
                mine[0][a:b] += pull.sum(1)
                mine[1][a:b] += epull.sum(1)
                res["dpos"][0][c:d] -= pull.sum(0)
                res["dpos"][1][c:d] += epull.sum(0)
            if "table" in t:
                flat, eflat = ds.reshape(H, -1), (eds + ds.abs() * total).reshape(H, -1)
                for b_ in range(self.buckets):
                    hit = (kind == b_).reshape(-1)
                    res["dtable"][0][:, b_] += flat[:, hit].sum(1)
                    res["dtable"][1][:, b_] += eflat[:, hit].sum(1)
        return res

    def results(self, plan=None, scale=None):
        plan = plan or self.plan()
        out, stats = plan.forward(self.q, self.k, self.v, save=True, scale=scale, **self.terms)
        g = plan.backward(self.dout, self.q, self.k, self.v, stats, scale=scale, **self.terms)
        got = {"out": out, **{n: x for n, x in g._asdict().items() if x is not None}}
        return got

    def check(self, plan=None, scale=None):
        got, want = self.results(plan, scale), self.reference(scale)
        assert set(got) == set(want)
        for name, (value, bound) in want.items():
            off = (got[name].double() - value).abs()
            limit = 1.1 * bound + (2.0 ** -25 if got[name].dtype == torch.float16 else 1e-30)
            bad = ~(off <= limit)
            assert not bad.any(), (name, int(bad.sum()), float((off / limit)[bad].max()), float(off.max()), float(value.abs().max()))
            assert got[name].dtype == (self.T if name in ("out", "dq", "dk", "dv") else torch.float32)
        return got


CLIP = list(range(9))                      # reach 4, a bucket each
COARSE = [0, 0, 1, 1, 2, 3, 3, 4, 4]       # reach 4, shared buckets
ONE_LENGTHS = [[1], [2], [5], [31], [32], [33], [0, 5, 0], [22, 12, 28], [64, 65], [44, 1, 0, 36], [129, 1, 200]]


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("sizes", ONE_LENGTHS, ids=str)
def test_lengths(T, sizes):
    Case(sizes, T, slope=True).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("slope,lut", [(False, None), (False, CLIP), (True, COARSE), (True, [0])], ids=["plain", "table", "both", "one"])
def test_terms(T, slope, lut):
    Case([22, 12, 70, 33], T, slope=slope, lut=lut).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 8), (3, 1, 16), (4, 2, 24), (8, 2, 40), (5, 5, 64), (6, 3, 96), (4, 1, 128), (12, 12, 32)])
def test_heads(T, heads, kv, dim):
    Case([19, 75, 3], T, heads=heads, kv=kv, dim=dim, lut=CLIP).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 8), (3, 1, 16), (4, 2, 40), (6, 3, 96), (4, 1, 128), (8, 8, 64)])
def test_heads_of_one_tile_fragments(T, heads, kv, dim):
    Case([19, 3, 32, 1, 16, 17], T, heads=heads, kv=kv, dim=dim, lut=CLIP).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("kv", [4, 2])
def test_many_one_tile_fragments(T, kv):
    """more than 512: a wave walks all heads and writes the positions' gradient itself"""
    sizes = [1 + (7 * i) % 32 for i in range(520)]
    Case(sizes, T, heads=4, kv=kv, dim=16, lut=COARSE).check()
    Case(sizes, T, heads=4, kv=kv, dim=16, lut=CLIP, queries=[1 + (5 * i) % 32 for i in range(520)]).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_few_one_tile_fragments_with_queries_of_their_own(T):
    Case([12, 32, 1, 30], T, lut=CLIP, queries=[3, 1, 32, 2]).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("dim,kv", [(32, 8), (64, 8), (32, 4)])
def test_all_kinds_of_fragments_together(T, dim, kv):
    Case([12, 30, 0, 33, 64] * 14 + [150, 300, 97], T, dim=dim, kv=kv, lut=COARSE, extra=3).check()


def test_nothing_at_all():
    for queries in (None, [0, 0]):
        got = Case([0, 0], torch.float32, lut=CLIP, queries=queries).check()
        assert not got["dslope"].any() and not got["dtable"].any() and got["out"].numel() == 0


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_queries_of_their_own(T):
    """one row per fragment; several; none; and fragments without keys, whose rows are 0"""
    Case([300, 1, 0, 45, 64], T, queries=[1, 1, 1, 1, 1], lut=CLIP).check()
    got = Case([30, 0, 70, 9], T, queries=[3, 40, 0, 33], kv=4, lut=COARSE).check()
    assert not got["out"][3:43].any() and not got["dq"][3:43].any() and not got["dk"][30:100].any()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_split_keys(T, dim):
    """few rows over many keys: the runs of keys are split and joined"""
    Case([1700, 1, 513, 0, 700], T, dim=dim, kv=2, queries=[1, 1, 2, 1, 35], lut=CLIP).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("dim,kv", [(32, 8), (64, 4), (128, 8)])
def test_workgroups_that_share_tiles(T, dim, kv):
    Case([150, 12, 130, 65, 64, 260] * 4, T, dim=dim, kv=kv, lut=COARSE).check()


def test_wide_table_and_far_residues():
    """reach at its largest; residue numbers at the ends of int32, whose difference saturates"""
    lut = (np.arange(2047) // 16).tolist()
    case = Case([90, 40], torch.float32, heads=3, dim=16, lut=lut, buckets=200)
    case.terms["residue"] = torch.randint(-600, 600, (130,), device="cuda", dtype=torch.int32)
    case.terms["residue"][::17] = 2 ** 31 - 1
    case.terms["residue"][5::17] = -2 ** 31
    got = case.check()
    assert not got["dtable"][:, 128:].any()


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_forbidden_buckets_and_lowest_values(T):
    case = Case([50, 7, 33], T, slope=False, lut=CLIP)
    case.terms["table"][:, 3] = -float("inf")
    case.terms["table"][:, 5] = torch.finfo(torch.float32).min / 2
    case.check()
    case = Case([50, 7, 33], T, slope=False, lut=CLIP)
    case.terms["table"][2:4] = -float("inf")  # two heads with nothing left
    got = case.check()
    assert not got["out"][:, 2:4].any() and not got["dq"][:, 2:4].any()
    # every score at the lowest value: the rounding swallows q.k, what is left is the mean over the keys
    case = Case([50, 7, 33], T, slope=False, lut=[0])
    case.terms["table"][:] = torch.finfo(torch.float32).min
    got = case.results()
    mean = torch.cat([case.v[a:b].double().mean(0, keepdim=True).expand(b - a, -1, -1) for a, b in zip(case.start, case.end)])
    # (1 / n is rounded to T, and n equal terms of it are summed)
    assert ((got["out"].double() - mean).abs() <= 3 * unit(T) * case.v.double().abs().amax() + 1e-6).all()
    assert all(torch.isfinite(x).all() for x in got.values())


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_large_scores_keep_their_precision(T):
    """scores of some hundreds: e_s of the tolerance grows with them, nothing else does"""
    Case([60, 9], T, spread=40.0, lut=CLIP).check()
    Case([60, 9], T, lut=CLIP).check(scale=20.0)


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [[20, 45, 12, 200], [20, 28, 12, 30], [20, 100, 12, 30] + [9] * 40], ids=["tiles", "small", "mixed"])
def test_nothing_leaks_between_fragments_or_from_behind(T, sizes):
    case = Case(sizes, T, lut=CLIP, extra=7)
    last, used = int(case.end[1]), int(case.end[-1])
    plan = case.plan()
    before = case.results(plan)
    for x in (case.q, case.k, case.v, case.dout, case.terms["pos"]):
        x[20:last] = float("nan")
        x[used:] = float("inf")
    case.terms["residue"][used:] = -2 ** 31
    after = case.results(plan)
    rows = torch.ones(used + 7, dtype=torch.bool, device="cuda")
    rows[20:last] = False
    rows[used:] = False
    for name in ("out", "dq", "dk", "dv", "dpos"):
        assert torch.equal(after[name][rows], before[name][rows]), name
        assert not after[name][used:].any()
    assert torch.isnan(after["out"][20:last]).all()


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_given_output_keeps_rows_behind_the_last_fragment(T):
    case = Case([20, 45], T, extra=5)
    plan = case.plan()
    want = plan.forward(case.q, case.k, case.v, **case.terms)
    wide = torch.full((70, 8, 64), 3.0, dtype=T, device="cuda")
    out = wide[:, :, 16:48]
    assert plan.forward(case.q, case.k, case.v, out=out, **case.terms) is out
    assert torch.equal(out[:65], want[:65]) and (out[65:] == 3).all() and (wide[:, :, :16] == 3).all() and (wide[:, :, 48:] == 3).all()


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_strides_alignment_and_orders(T):
    case = Case([20, 45, 100], T, lut=CLIP)
    plan = case.plan()
    want = case.results(plan)
    packed = torch.stack([case.q, case.k, case.v], 1)                       # [rows, 3, heads, dim]
    views = [tuple(packed[:, i] for i in range(3)),
             tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (case.q, case.k, case.v)),
             tuple(torch.cat([x, x[..., :3]], -1)[..., :32] for x in (case.q, case.k, case.v)),            # odd steps: copied
             tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (case.q, case.k, case.v))]      # last axis apart
    for q, k, v in views:
        out, stats = plan.forward(q, k, v, save=True, **case.terms)
        g = plan.backward(case.dout.transpose(0, 1).contiguous().transpose(0, 1), q, k, v, stats, **case.terms)
        assert torch.equal(out, want["out"])
        assert all(torch.equal(getattr(g, n), want[n]) for n in ("dq", "dk", "dv", "dpos", "dslope", "dtable"))
    # broadcast inputs: one row for all, one head for all
    case.k = case.k[:1].expand(165, -1, -1)
    case.v = case.v[:, :1].expand(-1, 8, -1)
    case.dout = torch.ones(1, 1, 1, dtype=T, device="cuda").expand(165, 8, 32)
    case.check(plan)


@pytest.mark.parametrize("size", [1e-7, 1.0, 3e4])
def test_float16_gradients_of_any_size(size):
    """dS of float16 rows stays precise where the gradients are tiny or near the type's largest (dv stays below 65504:
    P sums to at most the fragment's queries here, times |dout| of 3e4 / 60)"""
    case = Case([50, 20, 90], torch.float16, lut=CLIP)
    case.dout = (case.dout.float() * (size if size <= 1 else size / 60)).half()
    got = case.results()
    want = case.reference()
    for name, (value, bound) in want.items():
        # half a step of the smallest float16 numbers (2^-24) on top, where the result itself is that small
        extra = 2.0 ** -25 if got[name].dtype == torch.float16 else 0.0
        assert ((got[name].double() - value).abs() <= 1.1 * bound + extra + 1e-30).all(), name


def test_gradients_against_differences():
    """central differences in 64 bits of sum(out dout), step 1e-4: their own error is below 1e-7 of O(1) third
    derivatives; the float32 gradients are within 1e-4 by the bounds above"""
    case = Case([9, 14], torch.float32, heads=2, dim=8, lut=COARSE)
    got = case.results()
    leaves = {"dq": case.q, "dk": case.k, "dv": case.v, "dpos": case.terms["pos"], "dslope": case.terms["slope"], "dtable": case.terms["table"]}
    names = {"dpos": "pos", "dslope": "slope", "dtable": "table"}
    def value():
        return (case.reference()["out"][0] * case.dout.double()).sum()
    for name, leaf in leaves.items():
        wide = leaf.double()
        if name in names:
            case.terms[names[name]] = wide
        else:
            setattr(case, name[1:], wide)
        flat = wide.view(-1)
        for at in range(0, flat.numel(), max(1, flat.numel() // 5)):
            flat[at] += 1e-4
            up = value()
            flat[at] -= 2e-4
            down = value()
            flat[at] += 1e-4
            assert abs((up - down) / 2e-4 - got[name].view(-1)[at].double()) < 2e-4, (name, at)
        if name in names:
            case.terms[names[name]] = leaf
        else:
            setattr(case, name[1:], leaf)


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("dim", [32, 128])
def test_repeats_streams_and_graph_replays(T, dim):
    case = Case([150, 12, 130, 65, 64, 260] * 4 + [20] * 30, T, lut=CLIP, dim=dim)
    rows = Case([1700, 40, 900], T, queries=[1, 1, 1], kv=2, dim=dim)
    plan, plan_rows = case.plan(), rows.plan()
    first, first_rows = case.results(plan), rows.results(plan_rows)
    same = lambda a, b: all(torch.equal(a[n], b[n]) for n in b)
    for _ in range(3):
        assert same(case.results(plan), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):  # two calls of one plan at once
        with torch.cuda.stream(side):
            there, there_rows = case.results(plan), rows.results(plan_rows)
        here, here_rows = case.results(plan), rows.results(plan_rows)
        torch.cuda.synchronize()
        assert same(here, first) and same(there, first) and same(here_rows, first_rows) and same(there_rows, first_rows)
    graphs = []
    for _ in range(2):  # two captured graphs with workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = case.results(plan), rows.results(plan_rows)
        graphs.append((graph, held))
    for seed in (31, 32, 33):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for c in (case, rows):
            c.q.copy_(torch.randn(c.q.shape, generator=gen, device="cuda"))
            c.terms["pos"].copy_(torch.randn(c.terms["pos"].shape, generator=gen, device="cuda") * 5)
        want = case.results(plan), rows.results(plan_rows)
        torch.cuda.synchronize()
        for graph, held in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert same(held[0], want[0]) and same(held[1], want[1])


def test_a_norm_and_attention_block_trains_like_its_64_bit_form():
    """layer norm -> q, k, v -> attention -> residual, forward and backward, as a layer over a fragment batch runs them.
    Bound: a float32 block of O(1) values, three products of 64 terms and the operators' own bounds: 2e-4 of each
    gradient's largest value; the difference seen by a wrong term is O(1)."""
    from ai2bmd_amd.attention import FragmentAttention, relative_buckets
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    gen = torch.Generator(device="cuda").manual_seed(5)
    normal = lambda *s, by=1.0: torch.randn(*s, generator=gen, device="cuda") * by
    sizes = [22, 12, 28, 12, 41]
    end = np.cumsum(sizes)
    start, n = end - sizes, int(end[-1])
    x, w, b, proj = normal(n, 64), 1 + normal(64, by=0.1), normal(64, by=0.1), normal(192, 64, by=0.125)
    pos, slope, table = normal(n, 3, by=4.0), torch.full((4,), 0.2, device="cuda"), normal(4, 9, by=0.5)
    residue, dy = (torch.arange(n, device="cuda") // 6).int(), normal(n, 64)
    lut = relative_buckets(9, 4)
    plan = FragmentAttention(start, end, 4, 16, buckets=lut)
    h, ln = layer_norm(x, w, b)
    q, k, v = (h @ proj.t()).view(n, 3, 4, 16).unbind(1)
    terms = dict(pos=pos, slope=slope, residue=residue, table=table)
    out, stats = plan.forward(q, k, v, save=True, **terms)
    y = x + out.reshape(n, 64)
    g = plan.backward(dy.view(n, 4, 16), q, k, v, stats, **terms)
    dqkv = torch.stack([g.dq, g.dk, g.dv], 1).reshape(n, 192)
    dx, dw, db = layer_norm_backward(dqkv @ proj, x, ln, w, b)
    got = [y, dx + dy, dw, db, dqkv.t() @ h, g.dpos, g.dslope, g.dtable]
    leaves = [t.double().requires_grad_() for t in (x, w, b, proj, pos, slope, table)]
    X, W, B, P, R, S, TB = leaves
    H = torch.nn.functional.layer_norm(X, (64,), W, B)
    Q, K, V = (H @ P.t()).view(n, 3, 4, 16).unbind(1)
    rows = []
    for a, z in zip(start, end):
        d2 = (R[a:z, None] - R[None, a:z]).pow(2).sum(-1)
        far = torch.where(d2 > 0, torch.where(d2 > 0, d2, 1.0).sqrt(), 0.0)
        kind = torch.as_tensor(lut, device="cuda").long()[(residue[a:z][None] - residue[a:z, None]).clamp(-4, 4).long() + 4]
        s = torch.einsum("ihd,jhd->hij", Q[a:z], K[a:z]) / 4 - S[:, None, None] * far + TB[:, kind]
        rows.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), V[a:z]))
    Y = X + torch.cat(rows).reshape(n, 64)
    want = [Y, *torch.autograd.grad(Y, leaves, dy.double())]
    for a, b_ in zip(got, want):
        assert (a.double() - b_).abs().max() <= 2e-4 * b_.abs().max()


def test_refusals():
    from ai2bmd_amd.attention import FragmentAttention
    case = Case([20, 45], torch.bfloat16, lut=CLIP)
    plan = case.plan()
    t = case.terms
    out, stats = plan.forward(case.q, case.k, case.v, save=True, **t)
    q, k, v = case.q, case.k, case.v
    without = {n: x for n, x in t.items() if n != "slope"}
    for bad in (lambda: plan.forward(q[:64], k, v, **t), lambda: plan.forward(q, k.half(), v, **t), lambda: plan.forward(q, k, v[:, :4], **t),
                lambda: plan.forward(q.double(), k, v, **t), lambda: plan.forward(q.cpu(), k, v, **t), lambda: plan.forward(q, k, v, **without),
                lambda: plan.forward(q, k, v, **{**t, "table": t["table"][:, :8]}), lambda: plan.forward(q, k, v, **{**t, "residue": t["residue"].long()}),
                lambda: plan.forward(q, k, v, **{**t, "pos": t["pos"][:64]}), lambda: plan.forward(q, k, v, query_pos=t["pos"], **t),
                lambda: plan.forward(q, k, v, out=torch.empty(65, 8, 33, dtype=torch.bfloat16, device="cuda")[..., :32], **t),
                lambda: plan.backward(case.dout.float(), q, k, v, stats, **t), lambda: plan.backward(case.dout, q, k, v, stats[:, :64], **t),
                lambda: FragmentAttention(case.start, case.end, 8, 32, device="cuda:0").forward(q, k, v, residue=t["residue"], table=t["table"])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="failed"):  # an output whose rows run into one another
        plan.forward(q, k, v, out=torch.empty(1, 8, 32, dtype=torch.bfloat16, device="cuda").expand(65, -1, -1), **t)
    with pytest.raises(RuntimeError, match="autograd"):
        plan.forward(q, k, v, **{**t, "table": t["table"].requires_grad_()})
