"""Windowed attention on the GPU where single rows go wrong: maxima that keep growing, rows and columns that
hold what is not finite, rows that a bias masks throughout, extreme arguments."""

import sys

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from gdl_b200.functional import window_attention

from .attention_ref import buckets, check, reference, visible
from .test_gpu_window_attention import DT, call, make, verify

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 72, 96, 128])
@pytest.mark.parametrize("window,sinks", [((-1, -1), 0), ((-1, 0), 0), ((150, 40), 9)])
def test_maxima_that_grow_all_along(dt, dim, window, sinks):
    """Logits rise by 16 with every 32 keys, so that a row's reference of the exponents moves in each half of
    every tile: what was written before (P of the other half, the output) is rescaled again and again."""
    c = make(40, [300, 77], 2, 1, dim, DT[dt])
    c["q"][..., 0] = dim ** 0.5
    c["k"][..., 0] = torch.cat([torch.arange(300), torch.arange(77)]).cuda()[:, None] * 0.5
    verify(c, window, sinks)


def test_bucket_sums_beside_keys_of_minus_infinity():
    """Keys with a component of -inf where every query is positive have logits of -inf: weight 0. dQ of the rows
    that see one is 0 times infinity, so the gradients' second pass runs; the bucket sums are those of the
    other keys, the same bits each time."""
    c = make(41, [700, 130], 2, 1, 64, torch.bfloat16, buckets=16)
    c["q"][..., 0] = 1.0
    at = torch.tensor([35, 45, 60, 63, 100, 127, 400, 700 + 50, 700 + 120])
    c["k"][at.cuda(), :, 0] = -float("inf")
    first = None
    for _ in range(5):
        got = call(c, (90, 70), 3)
        want = reference(c["q"], c["k"], c["v"], c["ptr_q"].tolist(), c["ptr_k"].tolist(), 90, 70, 3, 0.125, c["bias"],
                         c["pos_q"], c["pos_k"], 0.4, 4, c["dout"], True) if first is None else want
        for n in ("out", "dk", "dv", "dbias"):
            check(got[n], want[n], n)
        first = got if first is None else first
        assert torch.equal(got["dbias"], first["dbias"])


# ------------------------------------------------------------------ plain: row by row, in 64 bits
def plain(c, window, sinks, buckets_of=None, logits32=False):
    """{name: value} from the definition, each row from the keys that it sees alone; `logits32`: logits are held
    in 32 bits. `sees` [Nq, Nk] is returned too."""
    f = lambda t: t.detach().cpu().double()  # noqa: E731
    q, k, v, do = (f(c[n]) for n in ("q", "k", "v", "dout"))
    H, G, D = q.shape[1], q.shape[1] // k.shape[1], q.shape[2]
    r = {"out": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    if "bias" in c:
        r["dbias"] = torch.zeros(c["bias"].shape, dtype=torch.float64)
    sees = torch.zeros(len(q), len(k), dtype=torch.bool)
    pq, pk = c["ptr_q"].tolist(), c["ptr_k"].tolist()
    for q0, q1, k0, k1 in zip(pq[:-1], pq[1:], pk[:-1], pk[1:]):
        ok = visible(q1 - q0, k1 - k0, *window, sinks)
        sees[q0:q1, k0:k1] = ok
        for i in range(q1 - q0):
            j = k0 + torch.nonzero(ok[i]).flatten()
            for h in range(H):
                s = (k[j, h // G] @ q[q0 + i, h]) / D ** 0.5
                if "bias" in c:
                    b = buckets_of[q0 + i, j]
                    s = s + f(c["bias"])[h, b]
                s = s.float().double() if logits32 else s
                top = s.max() if len(j) else torch.tensor(0.0)
                p = torch.exp(s - (0.0 if top == -float("inf") else top))
                p = p / p.sum() if p.sum() != 0 else p
                o = (p[:, None] * v[j, h // G]).sum(0)
                ds = p * (v[j, h // G] @ do[q0 + i, h] - (do[q0 + i, h] * o).sum())
                r["out"][q0 + i, h] = o
                r["dq"][q0 + i, h] = (ds[:, None] * k[j, h // G]).sum(0) / D ** 0.5
                r["dk"][j, h // G] += ds[:, None] * q[q0 + i, h] / D ** 0.5
                r["dv"][j, h // G] += p[:, None] * do[q0 + i, h]
                if "bias" in c:
                    r["dbias"][h].index_add_(0, b, ds)
    return r, sees


def pair_buckets(c, radius, steps):
    return buckets(c["pos_q"].cpu().numpy(), c["pos_k"].cpu().numpy(), radius, c["bias"].shape[1], steps)


def bounds(c, n, extra=0.0):
    """Worst-case errors: of a weight (e: logits of D products, bfloat16 roundings of P, dS and a result; `extra`
    for the logits' own size), on the largest values that meet in each result; a key is seen by at most n rows."""
    big = {m: float(torch.nan_to_num(c[m].float(), 0.0, 0.0, 0.0).abs().max()) for m in ("q", "k", "v", "dout")}
    D, bf16 = c["q"].shape[2], c["q"].dtype == torch.bfloat16
    e = 8 * 2.0 ** -8 if bf16 else 8 * (D + 8) * 2.0 ** -24 * max(1.0, big["q"] * big["k"] * D ** 0.5) + 2.0 ** -18
    e += extra
    ds = 2 * D * big["dout"] * big["v"]
    return {"out": e * big["v"], "dq": e * ds * big["k"] / D ** 0.5, "dk": e * ds * big["q"] / D ** 0.5 * n,
            "dv": e * big["dout"] * n, "dbias": e * ds * len(c["q"])}


PATHS = {  # type, head size, queries: tensor cores, f32 tiles (two sizes), bf16 in those, few rows (all forwards; three backwards)
    "mma": (torch.bfloat16, 64, None), "mma wide": (torch.bfloat16, 96, None), "tiles": (torch.float32, 24, None),
    "tiles wide": (torch.float32, 72, None), "tiles bf16": (torch.bfloat16, 20, None), "few": (torch.bfloat16, 64, [9, 6]),
    "few f32": (torch.float32, 32, [9, 6])}


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("name", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("whole", [True, False])
def test_what_is_not_finite_reaches_what_sees_it(path, name, bad, whole):
    """Where the definition gives a finite value so do the kernels, and where it does not, neither do they. (A row of
    a gradient that sums over a value that is not finite may come out NaN as a whole on the tensor cores.)"""
    dt, dim, lens_q = PATHS[path]
    window, sinks = (20, 12), 2
    for at in (0, 70, 99 + 3):  # a sink, a row in the middle, one of the second cloud
        c = make(42, [99, 61], 2, 1, dim, dt, lens_q=lens_q, buckets=8)
        rows = c[name].shape[0]
        row = min(at, rows - 1) if lens_q is None or name in ("k", "v") else at % rows
        c[name][row, 0, slice(None) if whole else slice(0, 1)] = bad
        got = call(c, window, sinks)
        want, sees = plain(c, window, sinks, pair_buckets(c, 0.4, 4))
        tol = bounds(c, len(c["q"]))
        loose = {n: torch.zeros(len(want[n]), dtype=torch.bool) for n in want if n != "dbias"}
        if "tiles" not in path and path != "few f32":
            if name == "k":
                loose["dq"] = sees[:, row]
            if name in ("q", "dout"):
                loose["dk"] = loose["dv"] = sees[row]
        for n in want:
            g = got[n].detach().cpu().double()
            fine = torch.isfinite(want[n])
            assert not bool(torch.isfinite(g[~fine]).any()), (n, at, "finite where the definition is not")
            here = fine if n == "dbias" else fine & ~loose[n][:, None, None]
            assert bool(torch.isfinite(g[here]).all()), (n, at, "not finite where the definition is")
            assert bool(((g - want[n])[here].abs() <= tol[n]).all()), (n, at)


@pytest.mark.parametrize("path", ["tiles", "tiles wide", "tiles bf16", "few f32"])
def test_keys_of_minus_infinity_take_no_part(path):
    """As above where the tiles run without tensor cores: such a key's own dK and dV are 0."""
    dt, dim, lens_q = PATHS[path]
    c = make(48, [99, 61], 2, 1, dim, dt, lens_q=lens_q, buckets=8)
    c["q"][..., 0] = 1.0
    at = torch.tensor([1, 40, 95, 98, 99 + 55])
    c["k"][at.cuda(), :, 0] = -float("inf")
    got = call(c, (20, 12), 2)
    want, _ = plain(c, (20, 12), 2, pair_buckets(c, 0.4, 4))
    tol = bounds(c, len(c["q"]))
    for n in ("out", "dk", "dv", "dbias"):
        assert bool(torch.isfinite(got[n]).all()) and bool(torch.isfinite(want[n]).all()), n
        assert float((got[n].detach().cpu().double() - want[n]).abs().max()) <= tol[n], n
    assert float(got["dk"][at].abs().max()) == 0 and float(got["dv"][at].abs().max()) == 0



@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [20, 64, 96])
@pytest.mark.parametrize("window,sinks,lens_q", [((30, 0), 3, None), ((-1, 0), 0, None), ((12, 9), 70, None), ((25, 0), 2, [5, 3])])
def test_buckets_of_minus_infinity(dt, dim, window, sinks, lens_q):
    """A table that cuts off distances by -inf: a row may see such keys alone (the first of a causal cloud sees
    itself). Its output is 0, and it takes no part in a gradient."""
    c = make(43, [150, 40], 2, 1, dim, DT[dt], lens_q=lens_q, buckets=8)
    c["bias"][0, 0] = c["bias"][1, 0] = -float("inf")   # not itself
    c["bias"][0, 4:] = c["bias"][1, 1:] = -float("inf")  # not far ones; the second head sees nothing at all
    got = call(c, window, sinks)
    want, _ = plain(c, window, sinks, pair_buckets(c, 0.4, 4))
    tol = bounds(c, len(c["q"]))
    for n in want:
        assert bool(torch.isfinite(got[n]).all()), n
        assert float((got[n].detach().cpu().double() - want[n]).abs().max()) <= tol[n], n
    assert float(got["out"][:, 1].abs().max()) == 0 and float(got["dq"][:, 1].abs().max()) == 0



@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_largest_windows_and_sinks_are_open_ones(dt):
    c = make(45, [200, 33], 2, 1, 32, DT[dt])
    for big in (sys.maxsize, 2 ** 62, 2 ** 70):
        for window, sinks, same in (((big, big), 0, (-1, -1)), ((big, 0), 0, (-1, 0)), ((10, big), 0, (10, -1)),
                                    ((10, 5), big, (-1, 5)), ((big, 5), big, (-1, 5))):
            got, want = call(c, window, sinks), call(c, same, 0)
            for n in want:
                assert torch.equal(got[n], want[n]), (n, window, sinks)



def test_a_tangent_is_refused_without_gradients_too():
    c = make(47, [40], 2, 2, 16, torch.float32)
    with torch.no_grad(), fwAD.dual_level():
        q = fwAD.make_dual(c["q"], torch.ones_like(c["q"]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            window_attention(q, c["k"], c["v"], c["ptr_q"], window=(4, 4))
        with pytest.raises((RuntimeError, NotImplementedError)):  # positions are constants: not of a tangent either
            window_attention(c["q"], c["k"], c["v"], c["ptr_q"], window=(4, 4), bias=torch.zeros(2, 4).cuda(),
                             pos_q=fwAD.make_dual(torch.rand(40, 3).cuda(), torch.ones(40, 3).cuda()))


def test_nothing_is_kept_without_gradients():
    c = make(49, [40], 2, 2, 16, torch.float32)
    q = c["q"].requires_grad_(True)
    with torch.no_grad():
        out = window_attention(q, c["k"], c["v"], c["ptr_q"], window=(4, 4))
    assert not out.requires_grad and out.grad_fn is None
    assert torch.equal(out, window_attention(q, c["k"], c["v"], c["ptr_q"], window=(4, 4)))



@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("sinks", [130, 500])
def test_many_sinks_of_many_clouds(dt, sinks):
    """More sinks than a tile of keys, than a chunk of queries, and than most clouds have rows."""
    verify(make(46, [1500, 3, 0, 140, 64, 700, 1], 2, 1, 32, DT[dt], buckets=8), (16, 16), sinks)



@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [20, 64, 96])
@pytest.mark.parametrize("mask", [-1e4, -1e9, "lowest"])
@pytest.mark.parametrize("lens_q", [None, [5, 3]])
def test_buckets_masked_by_large_negative_values(dt, dim, mask, lens_q):
    """A row whose keys are all masked by one finite value weighs them by what is left of their logits (by
    nothing, equally, where 32 bits hold no more than the mask), and so do its gradients."""
    c = make(44, [150, 40], 2, 1, dim, DT[dt], lens_q=lens_q, buckets=8)
    value = torch.finfo(DT[dt]).min if mask == "lowest" else mask
    c["bias"][0, :3] = c["bias"][1] = value
    window, sinks = (4, 2), 1
    got = call(c, window, sinks)
    want, _ = plain(c, window, sinks, pair_buckets(c, 0.4, 4), logits32=mask != -1e4)
    tol = bounds(c, len(c["q"]), extra=4 * 2.0 ** -23 * 1.5e4 if mask == -1e4 else 0.0)
    for n in want:
        assert bool(torch.isfinite(got[n]).all()), n
        assert float((got[n].detach().cpu().double() - want[n]).abs().max()) <= tol[n], n


@pytest.mark.parametrize("dim", [64, 96])
def test_the_status_word_stays_0(dim):
    c = make(50, [300], 2, 1, dim, torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = c["q"].requires_grad_(True)
    window_attention(q, c["k"], c["v"], c["ptr_q"], window=(40, 40), status=status).backward(c["dout"])
    assert int(status) == 0 and bool(torch.isfinite(q.grad).all())


@pytest.mark.parametrize("dim", [64, 96])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (2, 2)])
@pytest.mark.parametrize("lens", [[60], [190], [300, 40]])
@pytest.mark.parametrize("name", ["q", "k", "v", "dout"])
def test_second_passes_over_odd_numbers_of_tiles(dim, heads, kv, lens, name):
    """A second pass goes on where the first one left its rings of buffers, at any number of tiles (1, 3, 5 to a
    head here): no wait runs out, and rows that see nothing of it come out as they are."""
    c = make(51, lens, heads, kv, dim, torch.bfloat16, buckets=8)
    window = (200, 200)
    clean = call(c, window, 0)
    c[name][0] = float("nan")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    leaf = {n: c[n].detach().requires_grad_(True) for n in ("q", "k", "v", "bias")}
    out = window_attention(leaf["q"], leaf["k"], leaf["v"], c["ptr_q"], window=window, bias=leaf["bias"], pos_q=c["pos_q"],
                           radius=0.4, status=status)
    got = {"out": out, **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, [leaf[n] for n in "qkv"], c["dout"])))}
    assert int(status) == 0
    for n in got:
        # beyond what row 0 reaches, and in the other cloud
        far = min(2 * window[0] + 1 if n in ("dk", "dv", "dq") else window[0] + 1, lens[0])
        assert torch.equal(got[n][far:], clean[n][far:]), n


@pytest.mark.parametrize("dim,lens_q", [(32, None), (64, None), (96, None), (128, None), (20, None), (64, [12])])
def test_the_bias_gradient_sums_to_what_it_should(dim, lens_q):
    """With one bucket the gradient of the table is the sum of all dS, which is 0: what comes out is the error of delta
    = dO . O against sum_j P dP, the same that a gradient of few buckets is left with after most of it cancels. In 16
    bits of P and of O its parts are roundings of 2^-17 each, independent of one another: 8 standard deviations of
    their sum, and of dP's and the exponents' in f32 (2^-20). With P or O in 8 bits it is 5 times as far and more."""
    c = make(52, [128], 8, 8, dim, torch.bfloat16, lens_q=lens_q, buckets=1, bias_dt=torch.float32)
    got = call(c, (-1, -1), 0)["dbias"][:, 0].cpu().double()
    for h in range(8):
        q, k, v, do = (c[n][:, h].cpu().double() for n in ("q", "k", "v", "dout"))
        p = torch.softmax(q @ k.T / dim ** 0.5, 1)
        o = p @ v
        ds = p * (do @ v.T - (do * o).sum(1, keepdim=True))
        var = (do ** 2 * 2.0 ** -32 * ((p ** 2) @ (v ** 2) + o ** 2)).sum() + (ds ** 2).sum() * 2.0 ** -40
        assert abs(float(got[h])) <= 8 * float(var) ** 0.5, (h, float(got[h]), float(var) ** 0.5)
