"""Eviction by accumulated attention weight (``ops.evict``) against a plain selection on the CPU, and the
dense operators together: prompt, steps that accumulate weight, eviction, further steps."""

import math

import numpy as np
import pytest
import torch

from pqhsa_release_amd import _lib, ops
from tests.dense_util import DIM, SCALE, check_close, far_away
from tests.test_gpu_prompt import PromptProblem

gpu = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def rank_key(mass):
    """Order of the selection: by bit pattern, -0 equal to 0, a NaN without sign above +inf, one with below -inf."""
    u = mass.astype(np.float32).view(np.uint32).astype(np.int64)
    u = np.where(u == 0x80000000, 0, u)
    return np.where(u & 0x80000000, 0x80000000 - (u & 0x7fffffff) - 1, u + 0x80000000)


def plain(mass, n, keep, sink, recent):
    if n <= keep:
        return np.arange(n)
    low = min(sink, n)
    high = max(low, n - recent)
    middle = np.arange(low, high)
    order = np.lexsort((middle, -rank_key(mass[low:high])))
    best = middle[order[: keep - low - (n - high)]]
    return np.concatenate([np.arange(low), np.sort(best), np.arange(high, n)])


def caches(lens, heads, dtype, layout, block, cap, seed):
    """(source view, its K and V by [b, h, token], destination view, reader of the destination)."""
    g = torch.Generator().manual_seed(seed)
    B, n = len(lens), max(lens)
    K, V = (torch.randn(B, heads, n, DIM, generator=g).to(dtype) for _ in range(2))
    if layout == "dense":
        dk, dv = (torch.full((B, heads, cap, DIM), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        return ops.kv_contiguous(K.cuda(), V.cuda()), K, V, ops.kv_contiguous(dk, dv), lambda: (dk.cpu(), dv.cpu())

    def pages(tokens, start, total):
        per = -(-tokens // block)
        return torch.randperm(total, generator=g)[: B * per].reshape(B, per) + start, per

    # old and new blocks of one cache
    old_total, new_total = B * -(-n // block) + 1, B * -(-cap // block) + 1
    old, per = pages(n, 0, old_total)
    new, new_per = pages(cap, old_total, new_total)
    shape = (2, old_total + new_total, block, heads, DIM) if layout == "5d" else (old_total + new_total, heads, block, 2 * DIM)
    cache = torch.full(shape, 7.0, dtype=dtype)
    view = lambda c: (c[0].transpose(1, 2), c[1].transpose(1, 2)) if layout == "5d" else (c[..., :DIM], c[..., DIM:])  # noqa: E731
    kc, vc = view(cache)
    for b in range(B):
        for j in range(per):
            c = min(block, n - j * block)
            kc[old[b, j], :, :c], vc[old[b, j], :, :c] = K[b, :, j * block : j * block + c], V[b, :, j * block : j * block + c]
    dev = cache.cuda()
    src = ops.kv_paged(dev, old.to(torch.int32).cuda())
    dst = ops.kv_paged(dev, new.to(torch.int32).cuda())

    def read():
        out = []
        for c in view(dev.cpu()):
            out.append(torch.stack([c[new[b]].transpose(0, 1).reshape(heads, new_per * block, DIM)[:, :cap] for b in range(B)]))
        return out

    return src, K, V, dst, read


def check(lens, keep, sink, recent, *, heads=2, dtype=BF, layout="5d", block=16, masses="heavy", spare=3, seed=0):
    n, B = max(lens), len(lens)
    left = min(keep, n)
    src, K, V, dst, read = caches(lens, heads, dtype, layout, block, left + spare, seed)
    g = torch.Generator().manual_seed(seed + 1)
    mass = torch.exp(3 * torch.randn(B, heads, n + 2, generator=g) - 4)
    if masses == "ties":
        mass = torch.randint(0, 3, (B, heads, n + 2), generator=g).float()
    elif masses == "zero":
        mass = torch.zeros(B, heads, n + 2)
    elif masses == "odd":
        mass[torch.rand(mass.shape, generator=g) < 0.1] = math.inf
        mass[torch.rand(mass.shape, generator=g) < 0.1] = math.nan
        mass[torch.rand(mass.shape, generator=g) < 0.2] *= -1
        mass[torch.rand(mass.shape, generator=g) < 0.1] = -0.0
    out = torch.full((B, heads, left + spare), 7.0, device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept, new = ops.evict(src, dst, mass.cuda(), sl, keep=keep, sink=sink, recent=recent, n_max=n, mass_out=out)
    torch.cuda.synchronize()
    kept, out = kept.cpu().numpy(), out.cpu()
    dk, dv = read()
    assert new.tolist() == [min(x, keep) for x in lens]
    for b, x in enumerate(lens):
        for h in range(heads):
            want = plain(mass[b, h, :x].numpy(), x, keep, sink, recent)
            r = len(want)
            assert np.array_equal(kept[b, h, :r], want), (b, h)
            assert (kept[b, h, r:] == -1).all()
            assert np.array_equal(out[b, h, :r].numpy().view(np.uint32), mass[b, h, want].numpy().view(np.uint32))
            assert bool((out[b, h, r:] == 0).all())
            assert torch.equal(dk[b, h, :r], K[b, h, want]) and torch.equal(dv[b, h, :r], V[b, h, want])
            assert bool((dk[b, h, r:] == 7.0).all()) and bool((dv[b, h, r:] == 7.0).all()), "slots behind the kept keys were written"


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("layout,block", [("5d", 16), ("4d", 16), ("dense", 0), ("5d", 7), ("4d", 1)])
def test_layouts_and_types(dtype, layout, block):
    check([300, 40, 1, 129], 100, 4, 10, dtype=dtype, layout=layout, block=block, seed=3)


@gpu
@pytest.mark.parametrize("masses", ["heavy", "ties", "zero", "odd"])
@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 4, 60), (64, 64, 0), (65, 0, 0), (999, 3, 5), (1000, 3, 5), (5000, 3, 5)])
def test_selection(masses, keep, sink, recent):
    check([1000, 70, 0, 64], keep, sink, recent, masses=masses, heads=1, seed=keep)


@gpu
@pytest.mark.parametrize("n", [1, 2, 1023, 1024, 16383, 16384, 16385, 32768, 50001])
def test_long_and_odd_rows(n):
    check([n], max(1, n // 3), 0 if n < 10 else 4, 0 if n < 10 else 3, masses="ties", heads=1, seed=n)
    check([n], max(1, n // 2), 0 if n < 10 else 1, 0, heads=1, seed=n + 1)


@gpu
@pytest.mark.parametrize("masses", ["heavy", "ties", "zero", "odd"])
@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (17000, 16500, 300), (20000, 3, 16390), (34000, 40, 2)])
def test_streams_of_several_chunks(masses, keep, sink, recent):
    check([40000, 16385, 33000, 0, 9], keep, sink, recent, masses=masses, heads=1, layout="dense", seed=keep)


@gpu
def test_prompt_steps_eviction_and_further_steps_as_a_server_runs_them():
    """Prompt rows -> weights of the last rows -> two steps that add theirs -> eviction into new blocks -> a step on
    the shortened cache; every result against the 64-bit evaluation of what is left."""
    total, heads, groups, keep = 200, 2, 4, 96
    p = PromptProblem([total], [total], heads=heads, groups=groups, poison=False, seed=77, extra=0)
    kv = p.source()
    mass = torch.zeros(1, heads, total, device="cuda")
    q = p.q.cuda()
    n0 = total - 2
    first = PromptProblem([n0], [n0], heads=heads, groups=groups, poison=False, seed=1)
    first.K, first.V, first.q = p.K, p.V, p.q[:n0]
    out = torch.empty_like(q)
    sl = torch.tensor([n0], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n0], dtype=torch.int32, device="cuda")
    ops.prompt_attend(q[:n0], out[:n0], kv, groups, cu, sl, n_max=n0, rule=p.rule(), rows_max=n0, mass=mass, mass_rows=16)
    for step in range(2):
        sl = torch.tensor([n0 + step + 1], dtype=torch.int32, device="cuda")
        ops.dense_attend(q[n0 + step : n0 + step + 1], out[n0 + step : n0 + step + 1], kv, groups, sl, n_max=total,
                         rule=p.rule(), mass=mass, mass_in=mass)
    want, _, tol, _, weights, weight_tol = p.evaluate()
    check_close(out, want, tol, "out")
    add, t = p.mass(weights, weight_tol, 18)
    check_close(mass, add, t + 2.0 ** -20 * add, "mass")     # 18 rows' sums, and the log-sum-exp of the first 16
    dst_k, dst_v = (torch.zeros(1, heads, keep + 1, DIM, dtype=p.dtype, device="cuda") for _ in range(2))
    dst = ops.kv_contiguous(dst_k, dst_v)
    mass_out = torch.full((1, heads, keep + 1), 7.0, device="cuda")
    kept, new = ops.evict(kv, dst, mass, sl, keep=keep, sink=4, recent=32, n_max=total, mass_out=mass_out)
    m = mass.cpu().numpy()
    for h in range(heads):
        at = plain(m[0, h], total, keep, 4, 32)
        assert np.array_equal(kept[0, h].cpu().numpy(), at)
        assert torch.equal(dst_k[0, h, :keep].cpu(), p.K[0, h, at]) and torch.equal(dst_v[0, h, :keep].cpu(), p.V[0, h, at])
    # the next token's row behind the kept ones
    nxt = PromptProblem([keep + 1], [1], heads=heads, groups=groups, poison=False, seed=78, extra=0)
    dst_k[:, :, keep], dst_v[:, :, keep] = nxt.K[:, :, keep].cuda(), nxt.V[:, :, keep].cuda()
    nxt.K, nxt.V = dst_k.cpu(), dst_v.cpu()
    new += 1
    before = mass_out.clone()
    got = torch.empty(1, heads * groups, DIM, dtype=p.dtype, device="cuda")
    ops.dense_attend(nxt.q.cuda(), got, dst, groups, new, n_max=keep + 1, rule=nxt.rule(), mass=mass_out, mass_in=mass_out)
    nxt.weight_rounding = lambda: 0.0
    want, _, tol, _, weights, weight_tol = nxt.evaluate()
    check_close(got, want, tol, "out after the eviction")
    add, t = nxt.mass(weights, weight_tol)
    old = before.double().cpu()
    check_close(mass_out, old + add, t + (1 + groups) * 2.0 ** -24 * (old + add), "mass after the eviction")


@gpu
@pytest.mark.parametrize("layouts", [("4d", "dense"), ("dense", "5d")])
def test_from_one_layout_into_another(layouts):
    lens, keep = [130, 40, 1], 48
    src, K, V, _, _ = caches(lens, 2, BF, layouts[0], 16, keep, 11)
    _, _, _, dst, read = caches(lens, 2, BF, layouts[1], 16, keep, 11)
    mass = torch.rand(3, 2, 130, generator=torch.Generator().manual_seed(2))
    kept, new = ops.evict(src, dst, mass.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), keep=keep, sink=2, recent=5, n_max=130)
    assert new.tolist() == [48, 40, 1]
    for b, n in enumerate(lens):
        for h in range(2):
            want = plain(mass[b, h].numpy(), n, keep, 2, 5)
            assert np.array_equal(kept[b, h, : len(want)].cpu().numpy(), want) and bool((kept[b, h, len(want) :] == -1).all())
            k, v = (ops.paged_gather_range(dst, b, 0, len(want))[i][h].cpu() for i in range(2))
            assert torch.equal(k, K[b, h, torch.from_numpy(want)]) and torch.equal(v, V[b, h, torch.from_numpy(want)])


@gpu
def test_blocks_outside_either_cache():
    src, K, V, dst, read = caches([64], 1, BF, "5d", 16, 32, 5)
    src.keep[1][0, 1] = -1
    dst.keep[1][0, 1] = dst.blocks
    mass = torch.zeros(1, 1, 64, device="cuda")
    kept, _ = ops.evict(src, dst, mass, torch.tensor([64], dtype=torch.int32, device="cuda"), keep=32, sink=32, recent=0, n_max=64)
    torch.cuda.synchronize()
    assert kept.flatten().tolist() == list(range(32))
    cache = src.keep[0].cpu()
    block = int(dst.keep[1][0, 0])
    assert torch.equal(cache[0, block, :, 0], K[0, 0, :16]) and torch.equal(cache[1, block, :, 0], V[0, 0, :16])


@gpu
def test_rows_beyond_32_bit_offsets():
    src, K, V, dst, read = caches([500, 90], 8, BF, "5d", 16, 60, 6)
    mass = torch.rand(2, 8, 500, generator=torch.Generator().manual_seed(1)).cuda()
    sl = torch.tensor([500, 90], dtype=torch.int32, device="cuda")
    near, _ = ops.evict(src, dst, mass, sl, keep=60, sink=1, recent=2, n_max=500)
    far = far_away(src)
    first = far.blocks - src.blocks
    far_dst = ops.kv_paged(far.keep[0], dst.keep[1] + first)
    kept, _ = ops.evict(far, far_dst, mass, sl, keep=60, sink=1, recent=2, n_max=500)
    assert torch.equal(kept, near) and torch.equal(far.keep[0][:, first:], src.keep[0])


@gpu
def test_lengths_beyond_the_bound_and_a_replayed_graph():
    src, K, V, dst, read = caches([500], 2, BF, "4d", 16, 60, 6)
    mass = torch.rand(1, 2, 500, generator=torch.Generator().manual_seed(1)).cuda()
    sl = torch.tensor([900], dtype=torch.int32, device="cuda")
    kept, new = ops.evict(src, dst, mass, sl, keep=60, sink=1, recent=2, n_max=500)
    assert new.tolist() == [60]
    for h in range(2):
        assert np.array_equal(kept[0, h].cpu().numpy(), plain(mass[0, h].cpu().numpy(), 500, 60, 1, 2))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_new = ops.evict(src, dst, mass, sl, keep=60, sink=1, recent=2, n_max=500)
    for k in range(3):
        mass.copy_(torch.rand(1, 2, 500, generator=torch.Generator().manual_seed(k)))
        got.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        want, _ = ops.evict(src, dst, mass, sl, keep=60, sink=1, recent=2, n_max=500)
        assert torch.equal(got, want), k


@gpu
def test_refusals():
    src, K, V, dst, _ = caches([64, 30], 2, BF, "5d", 16, 32, 1)
    sl = torch.tensor([64, 30], dtype=torch.int32, device="cuda")
    mass = torch.zeros(2, 2, 64, device="cuda")

    def refused(match, kv=src, dst=dst, mass=mass, sl=sl, **kw):
        kw = {"keep": 32, "sink": 2, "recent": 2, "n_max": 64, **kw}
        with pytest.raises(ValueError, match=match):
            ops.evict(kv, dst, mass, sl, **kw)

    refused("keep", keep=3)
    refused("keep", keep=0, sink=0, recent=0)
    refused("keep", sink=-1)
    refused("n_max", n_max=65)
    refused("dst holds", keep=40)
    refused("apart", dst=src)
    refused("seq_lens", sl=sl.long())
    refused("mass must", mass=mass[:, :, :63])
    refused("mass must", mass=mass.double())
    refused("mass_out", mass_out=torch.zeros(2, 2, 31, device="cuda"))
    refused("share", mass_out=mass)
    other = ops.kv_contiguous(*(torch.zeros(2, 2, 40, DIM, dtype=HF, device="cuda") for _ in range(2)))
    refused("dtype", dst=other)
    same = torch.zeros(2, 2, 64, DIM, dtype=BF, device="cuda")
    dense = ops.kv_contiguous(same, torch.zeros_like(same))
    refused("apart", kv=dense, dst=ops.kv_contiguous(same[:, :, 8:], dense.keep[1][:, :, 8:]))


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: a call that were not refused must find no GPU")
def test_c_entry_refuses_bad_arguments_before_any_gpu_work():
    import ctypes

    lib = _lib.load()
    src, dst = _lib.KvView(), _lib.KvView()
    for k, v in enumerate((src, dst)):
        v.k_base = v.v_base = (1 + k) << 20
        v.dtype, v.stride_tok, v.stride_head, v.stride_seq = _lib.BF16, 128, 1280, 12800

    def call(B=1, H=1, n_max=10, stride=10, keep=5, sink=1, recent=1, mass=1 << 20, out=None, out_stride=0, ws=1 << 20, ws_bytes=1 << 20):
        return lib.pqhsa_evict(ctypes.byref(src), 0, ctypes.byref(dst), 0, B, H, mass, stride, 1 << 20, n_max, keep, sink, recent,
                               1 << 20, 1 << 20, out, out_stride, ws, ws_bytes, None)

    assert call(keep=1) == -1 and call(keep=0, sink=0, recent=0) == -1 and call(sink=-1) == -1
    assert call(keep=2**31 - 1, sink=2**31 - 1, recent=2**31 - 1) == -1
    assert call(stride=9) == -1 and call(n_max=-1) == -1 and call(H=0) == -1 and call(B=70000) == -1 and call(mass=None) == -1
    assert call(out=1 << 20, out_stride=4) == -1 and call(ws=None) == -1 and call(ws=16) == -1
    assert call(n_max=2**31 - 1, stride=1 << 31, ws_bytes=1 << 60) == -1 and b"large" in lib.pqhsa_last_error()
    assert call(n_max=1 << 20, stride=1 << 20, ws_bytes=256) == -3 and b"workspace" in lib.pqhsa_last_error()
    assert call(B=0) == 0
    dst.dtype = _lib.F16
    assert call() == -1
    dst.dtype, dst.k_base = _lib.BF16, src.k_base
    assert call() == -1 and b"apart" in lib.pqhsa_last_error()
