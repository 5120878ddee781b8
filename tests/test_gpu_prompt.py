"""Dense attention of packed prompt rows (``ops.prompt_attend``) against an evaluation in 64 bits."""

import math

import pytest
import torch

from pqhsa_release_amd import _lib, ops
from tests.dense_util import DIM, SCALE, HALF_STEP, DenseProblem, check_close, far_away

gpu = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


class PromptProblem(DenseProblem):
    def weight_rounding(self):
        # the 2-byte types round every weight once more, to half a step
        return 0.0 if self.dtype == FP else HALF_STEP[self.dtype]

    def weight_floor(self):
        # fp16 has no steps under 2^-24: a weight held as 2^(z2 - m + 13), m at most the maximum rounded up, is up to
        # half of that off, 2^-25 2^-13 2^1 of the largest (keys of other tiles lose less)
        return 2.0 ** -37 if self.dtype == HF else 0.0

    def cu_rows(self, device="cuda"):
        cu = [0]
        for r in self.rows:
            cu.append(cu[-1] + r)
        return torch.tensor(cu, dtype=torch.int32, device=device)


def run(p, *, mass=None, rows_max=None, with_lse=True, strided=False):
    kv, rule = p.source(), p.rule()
    total, heads = p.q.shape[0], p.H * p.G
    if strided:
        wide = torch.full((total, 3 * heads, DIM), math.nan, dtype=p.dtype, device="cuda")
        q = wide[:, heads : 2 * heads]
        q.copy_(p.q.cuda())
        out = torch.full((heads, total, DIM), 7.0, dtype=p.dtype, device="cuda").transpose(0, 1)
    else:
        q, out = p.q.cuda(), torch.full((total, heads, DIM), 7.0, dtype=p.dtype, device="cuda")
    lse = torch.full((total, heads), 7.0, device="cuda") if with_lse else None
    m = m_in = None
    if mass is not None:
        m_in = torch.rand(p.B, p.H, p.n_max + 1, generator=torch.Generator().manual_seed(6)).cuda()
        m = torch.full_like(m_in, 7.0)
    ops.prompt_attend(q, out, kv, p.G, p.cu_rows(), p.seq_lens(), n_max=p.n_max, rule=rule,
                      rows_max=max(p.rows) if rows_max is None else rows_max, lse=lse, mass=m, mass_in=m_in, decay=0.5,
                      mass_rows=mass or 0)
    torch.cuda.synchronize()
    return out, lse, m, m_in


def check(p, *, mass=None, **kw):
    out, lse, m, m_in = run(p, mass=mass, **kw)
    want, want_lse, tol, lse_tol, weights, weight_tol = p.evaluate()
    total = sum(p.rows)
    check_close(out[:total], want, tol, "out")
    assert bool((out[total:] == 7.0).all()), "rows behind the last sequence were written"
    if lse is not None:
        check_close(lse[:total], want_lse, lse_tol, "lse")
        assert bool((lse[total:] == 7.0).all())
    if mass is not None:
        add, t = p.mass(weights, weight_tol, mass)
        for b, n in enumerate(p.lens):
            old = 0.5 * m_in[b, :, :n].double().cpu()
            check_close(m[b, :, :n], old + add[b, :, :n], t[b, :, :n] + 2.0 ** -22 * (old + add[b, :, :n]), "mass")
            assert bool((m[b, :, n:] == 7.0).all())


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("layout,block", [("5d", 16), ("4d", 16), ("dense", 0), ("5d", 7), ("4d", 1), ("5d", 128)])
def test_layouts_types_and_ragged_prompts(dtype, layout, block):
    check(PromptProblem([150, 1, 70, 0, 64], [150, 1, 33, 0, 64], dtype=dtype, layout=layout, block=block, pad=3, seed=3), mass=0)


@gpu
@pytest.mark.parametrize("heads,groups", [(1, 1), (1, 16), (3, 7), (8, 4), (2, 5)])
def test_head_layouts(heads, groups):
    check(PromptProblem([190, 33], [190, 20], heads=heads, groups=groups, seed=11), mass=9, strided=True)


@gpu
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 500])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_one_whole_prompt_of_every_tail(dtype, length):
    check(PromptProblem([length], [length], heads=1, groups=3, dtype=dtype, seed=length, extra=0))


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("kw", [dict(softcap=3.0), dict(softcap=50.0, slopes=True), dict(slopes=True), dict(window=1),
                                dict(window=50), dict(window=50, prefix=4), dict(window=64, prefix=[0, 150, 3, 9]),
                                dict(prefix=[200, 7, 1, 0]), dict(docs=4), dict(docs=60),
                                dict(docs=3, window=40, prefix=30, softcap=10.0, slopes=True), dict(window=10000), dict(prefix=10000)])
def test_score_rules(dtype, kw):
    check(PromptProblem([300, 133, 2, 0], [300, 60, 2, 0], dtype=dtype, heads=2, groups=2, seed=21, pad=2, **kw), mass=0)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("kw", [dict(), dict(softcap=5.0, slopes=True), dict(window=50, prefix=4, docs=3)])
@pytest.mark.parametrize("scale", [-0.11, 0.0])
def test_scales_that_are_not_positive(dtype, kw, scale):
    check(PromptProblem([300, 133, 2, 0], [300, 60, 2, 0], dtype=dtype, heads=2, groups=2, seed=22, pad=2, scale=scale, **kw), mass=0)


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rows_max", [0, 5])
def test_few_rows_on_a_long_cache_split_and_joined(dtype, rows_max):
    check(PromptProblem([3000, 77], [5, 3], heads=2, groups=4, dtype=dtype, seed=5, pad=4), mass=2, rows_max=rows_max)


@gpu
@pytest.mark.parametrize("kw", [dict(docs=9), dict(window=300, prefix=20)])
def test_split_ranges_with_tiles_left_out(kw):
    check(PromptProblem([2500, 400], [64, 64], heads=1, groups=4, seed=7, **kw), mass=16)


@gpu
def test_rows_in_front_of_their_sequence_see_nothing():
    p = PromptProblem([5, 0, 40], [9, 3, 40], heads=2, groups=2, seed=8, prefix=3)
    check(p, mass=0)
    out, lse, _, _ = run(p)
    assert bool((out[:4] == 0).all()) and bool((lse[:4] == -math.inf).all()) and bool((out[9:12] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("prefix", [None, 3])
def test_a_window_near_2_31_with_rows_in_front_of_their_sequence(dtype, prefix):
    check(PromptProblem([5, 70], [9, 90], heads=2, groups=2, dtype=dtype, seed=8, window=2**31 - 1, prefix=prefix), mass=0)


@gpu
def test_a_long_prompt_and_large_scores():
    check(PromptProblem([1700], [1700], heads=1, groups=2, dtype=BF, seed=5, q_gain=6.0))


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_infinite_and_nan_values_reach_only_the_rows_that_see_them(dtype):
    """Position 90's value is NaN, 100's +inf in one dim, 101's -inf in another: rows before stay exact, rows
    after get NaN or the infinity, in every split."""
    p = PromptProblem([200], [200], heads=1, groups=1, dtype=dtype, poison=False, seed=13)
    want, want_lse, tol, lse_tol, _, _ = p.evaluate()
    p.V[0, 0, 90, 7] = math.nan
    p.V[0, 0, 100, 8] = math.inf
    p.V[0, 0, 101, 8] = -math.inf
    p.V[0, 0, 100, 9] = math.inf
    p.V[0, 0, 101, 10] = -math.inf
    out, lse, _, _ = run(p)
    check_close(lse, want_lse, lse_tol, "lse")
    clean = torch.ones(200, 1, DIM, dtype=torch.bool)
    clean[90:, 0, 7] = clean[100:, 0, 8] = clean[100:, 0, 9] = clean[101:, 0, 10] = False
    check_close(out[clean.cuda()], want[clean], tol[clean], "out")
    assert bool(out[90:, 0, 7].isnan().all())
    assert bool((out[100, 0, 8] == math.inf).all()) and bool(out[101:, 0, 8].isnan().all())
    assert bool((out[100:, 0, 9] == math.inf).all()) and bool((out[101:, 0, 10] == -math.inf).all())


def sinks(n, every, drop):
    """Levels of n keys: ``drop`` for one key in ``every``, 0 for the others."""
    return [drop if j % every == 0 else 0.0 for j in range(n)]


@gpu
@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("spread", [0.0, 0.7])
@pytest.mark.parametrize("drop", [10, 12, 14, 16, 18, 20, 24])
def test_light_keys_behind_sinks_without_a_value(drop, spread, dtype):
    """Keys whose weights are all far below the largest one make up the whole output, in values that
    keep it above fp16's subnormal numbers."""
    p = PromptProblem([4000, 90], [5, 9], heads=1, groups=2, dtype=dtype, seed=61)
    check(p.set_levels(sinks(4000, 100, drop), spread=spread, gain=min(2e4, math.exp(drop) / 100), silent=5.0), mass=2)


@gpu
@pytest.mark.parametrize("kw", [dict(), dict(docs=3), dict(softcap=40.0)])
def test_levels_of_keys_that_rise_and_fall_in_fp16(kw):
    g = torch.Generator().manual_seed(4)
    levels = (torch.randint(0, 4, (50,), generator=g) * -6.0).repeat_interleave(20)
    p = PromptProblem([1000, 700], [1000, 300], heads=2, groups=2, dtype=HF, seed=63, **kw)
    check(p.set_levels(levels, spread=0.5, gain=2e4, silent=-16.0), mass=0)


@gpu
def test_light_keys_in_the_large_workgroups_in_fp16():
    p = PromptProblem([901, 700, 512, 900, 650, 640, 577, 830], [512, 500, 512, 550, 520, 515, 490, 500], heads=2, groups=16,
                      dtype=HF, seed=44)
    check(p.set_levels(sinks(901, 150, 15.0), spread=0.5, gain=100.0, silent=5.0), mass=3)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_an_infinite_value_of_a_key_with_next_to_no_weight(dtype):
    """exp(-150) is no fp32 number, but it is more than nothing: every row that sees the key, in tiles that all rows
    see whole and others, is infinite there."""
    p = PromptProblem([500, 1500], [500, 3], heads=1, groups=2, dtype=dtype, poison=False, seed=15).set_levels([150.0] + [0.0] * 1499)
    p.V[0, 0, 57, 3] = p.V[0, 0, 7, 4] = math.inf
    p.V[1, 0, 1400, 5] = p.V[1, 0, 20, 6] = -math.inf
    p.V[1, 0, 21, 6] = math.inf
    out, _, _, _ = run(p)
    assert bool((out[57:500, :, 3] == math.inf).all()) and bool((out[7:500, :, 4] == math.inf).all())
    assert bool((out[500:, :, 5] == -math.inf).all()) and bool(out[500:, :, 6].isnan().all())
    out[57:500, :, 3] = out[7:500, :, 4] = out[500:, :, 5:7] = 0.0
    assert bool(out.isfinite().all())


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_infinite_values_in_the_large_workgroups(dtype):
    """Sequence 0's rows are at positions 389 to 900: one value only some of them see, one that all see, in whole tiles."""
    p = PromptProblem([901, 700, 512, 900, 650, 640, 577, 830], [512, 500, 512, 550, 520, 515, 490, 500], heads=2, groups=16,
                      dtype=dtype, poison=False, seed=45)
    want, _, tol, _, _, _ = p.evaluate()
    p.V[0, 1, 600, 4], p.V[0, 1, 100, 5], p.V[0, 1, 620, 6] = math.inf, -math.inf, math.nan
    out, _, _, _ = run(p)
    clean = torch.ones(want.shape, dtype=torch.bool)
    clean[600 - 389 : 512, 16:, 4] = clean[:512, 16:, 5] = clean[620 - 389 : 512, 16:, 6] = False
    check_close(out[clean.cuda()], want[clean], tol[clean], "out")
    assert bool((out[600 - 389 : 512, 16:, 4] == math.inf).all()) and bool((out[:512, 16:, 5] == -math.inf).all())
    assert bool(out[620 - 389 : 512, 16:, 6].isnan().all())


@gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("at", [0, 37, 700])
def test_a_key_that_stands_out_gives_its_value_unrounded(dtype, at):
    """All other weights together are under 1500 * exp(-30 + 5) = 2e-8: what is off beyond that (and beyond 2^-15, where
    fp16's base is cut) is a rounding of the one weight, which is avoidable."""
    p = PromptProblem([1500, 801], [700, 4], heads=2, groups=2, dtype=dtype, seed=71).set_levels([30.37 if j == at else 0.0 for j in range(1500)], spread=1.0)
    out, _, _, _ = run(p)
    want = p.V[:, :, at].repeat_interleave(2, 1)
    assert torch.equal(out.cpu(), torch.cat([want[:1].expand(700, -1, -1), want[1:].expand(4, -1, -1)]))


@gpu
def test_block_table_entries_outside_the_cache_mask_their_keys():
    kw = dict(heads=2, groups=2, block=16, poison=False, seed=9)
    p, q = PromptProblem([160], [160], **kw), PromptProblem([160], [160], **kw)
    kv = p.source()
    cache, table = kv.keep
    table[0, 2], table[0, 5] = -1, kv.blocks
    out = torch.empty(160, 4, DIM, dtype=p.dtype, device="cuda")
    ops.prompt_attend(p.q.cuda(), out, kv, 2, p.cu_rows(), p.seq_lens(), n_max=160, rule=p.rule())
    gone = torch.zeros(160, dtype=torch.bool)
    gone[32:48] = gone[80:96] = True
    see = q.visible(0) & ~gone
    q.visible = lambda b: see
    want, _, tol, _, _, _ = q.evaluate()
    check_close(out, want, tol, "out")


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_documents_that_alternate_between_keys_over_many_tiles(dtype):
    """Every tile of the walk is masked by its own keys' documents, which are read while later tiles' are on their way."""
    p = PromptProblem([1500, 900], [1500, 500], heads=1, groups=4, dtype=dtype, seed=41, docs=3)
    p.docs = torch.randint(0, 3, p.docs.shape, generator=torch.Generator().manual_seed(5)).to(torch.int32)
    check(p, mass=0)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("kw", [dict(), dict(docs=3), dict(window=300, prefix=20, softcap=30.0)])
def test_rows_enough_for_the_large_workgroups(dtype, kw):
    """131072 packed rows and more: eight waves a workgroup, four tiles of K and V in LDS."""
    p = PromptProblem([901, 700, 512, 900, 650, 640, 577, 830], [512, 500, 512, 550, 520, 515, 490, 500], heads=2, groups=16,
                      dtype=dtype, seed=43, **kw)
    if "docs" in kw:
        p.docs = torch.randint(0, 3, p.docs.shape, generator=torch.Generator().manual_seed(5)).to(torch.int32)
    check(p, mass=3)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("kw", [dict(slopes=True), dict(scale=-0.11), dict(scale=0.0, window=300)])
def test_biased_scores_and_other_scales_in_the_large_workgroups(dtype, kw):
    check(PromptProblem([901, 700, 512, 900, 650, 640, 577, 830], [512, 500, 512, 550, 520, 515, 490, 500], heads=2, groups=16,
                        dtype=dtype, seed=46, **kw), mass=3)


@gpu
def test_same_results_without_lse_and_from_a_replayed_graph():
    p = PromptProblem([260, 90], [260, 40], heads=2, groups=4, seed=31)
    kv, rule, q, sl, cu = p.source(), p.rule(), p.q.cuda(), p.seq_lens(), p.cu_rows()
    out, mass = torch.empty_like(q), torch.empty(2, 2, 260, device="cuda")

    def step():
        ops.prompt_attend(q, out, kv, 4, cu, sl, n_max=260, rule=rule, rows_max=260, mass=mass, mass_rows=8)

    step()
    torch.cuda.synchronize()
    eager, eager_mass = out.clone(), mass.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        out.fill_(math.nan)
        mass[:, :, :90] = math.nan
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(mass[0], eager_mass[0]) and torch.equal(mass[1, :, :90], eager_mass[1, :, :90])
        step()


@gpu
def test_no_keys_at_all_and_row_bounds_out_of_order():
    p = PromptProblem([40, 40], [30, 30], heads=2, groups=2, seed=8)
    kv, rule, q = p.source(), p.rule(), p.q.cuda()
    out, lse = torch.full_like(q, 7.0), torch.full((60, 4), 7.0, device="cuda")
    empty = torch.zeros(2, dtype=torch.int32, device="cuda")
    ops.prompt_attend(q, out, kv, 2, p.cu_rows(), empty, n_max=0, rule=rule, lse=lse)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    one = torch.full_like(q[:2], 7.0)
    ops.dense_attend(q[:2], one, kv, 2, empty, n_max=0, rule=rule)
    assert bool((one == 0).all())
    # bounds that do not ascend and run past the rows: rows of q only, nothing else is written
    wild = torch.tensor([50, -3, 1 << 30], dtype=torch.int32, device="cuda")
    out.fill_(7.0)
    ops.prompt_attend(q, out, kv, 2, wild, p.seq_lens(), n_max=40, rule=rule)
    assert bool(out.isfinite().all())


@gpu
def test_rows_beyond_32_bit_offsets():
    p = PromptProblem([300, 77], [90, 77], heads=8, groups=4, layout="5d", block=16, seed=17)
    near, q, sl, rule = p.source(), p.q.cuda(), p.seq_lens(), p.rule()
    far = far_away(near)
    outs, weights = [torch.empty_like(q) for _ in range(2)], [torch.zeros(2, 8, 300, device="cuda") for _ in range(2)]
    for kv, out, w in zip((near, far), outs, weights):
        ops.prompt_attend(q, out, kv, 4, p.cu_rows(), sl, n_max=300, rule=rule, mass=w, mass_rows=5)
    assert torch.equal(*outs) and torch.equal(*weights)


@gpu
def test_refusals():
    p = PromptProblem([64, 30], [64, 30], heads=2, groups=2, seed=1)
    kv, rule, q, sl, cu = p.source(), p.rule(), p.q.cuda(), p.seq_lens(), p.cu_rows()
    out = torch.empty_like(q)

    def refused(match=None, q=q, out=out, kv=kv, groups=2, cu=cu, sl=sl, **kw):
        kw = {"n_max": 64, "rule": rule, **kw}
        with pytest.raises(ValueError, match=match):
            ops.prompt_attend(q, out, kv, groups, cu, sl, **kw)

    refused("device", q=q.cpu())
    refused("dtype", q=q.float())
    refused("q must", groups=1)
    refused("groups", groups=17)
    refused("n_max", n_max=kv.capacity + 1)
    refused("cu_rows", cu=cu[:2])
    refused("cu_rows", cu=cu.long())
    refused("seq_lens", sl=sl[:1])
    refused("overlap", out=out[:1].expand(94, -1, -1))
    refused("overlap", out=out[:3])
    refused("overlap", out=q)
    refused("mass", mass=torch.zeros(2, 2, 63, device="cuda"))
    refused("mass_rows", mass=torch.zeros(2, 2, 64, device="cuda"), mass_rows=-1)
    refused("lse", lse=torch.zeros(2, 4, device="cuda"))
    refused("prefix", rule=ops.ScoreRule(scale=SCALE, prefix=torch.zeros(3, dtype=torch.int32, device="cuda")))


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: a call that were not refused must find no GPU")
def test_c_entry_refuses_bad_arguments_before_any_gpu_work():
    import ctypes

    lib = _lib.load()
    view, score, mass = _lib.KvView(), _lib.Score(), _lib.Mass()
    view.k_base = view.v_base = 1 << 20
    view.dtype, view.stride_tok, view.stride_head, view.stride_seq = _lib.BF16, 128, 1280, 12800
    score.scale = 1.0

    def call(q=1 << 20, dtype=_lib.BF16, stride=128, T=10, B=1, H=1, G=1, n_max=10, mass=None, ws=1 << 20, ws_bytes=1 << 20):
        return lib.pqhsa_prompt_attend_paged(q, dtype, 128, stride, 1 << 20, 128, 128, T, 1 << 20, ctypes.byref(view), 0, B, H, G,
                                             1 << 20, n_max, 0, ctypes.byref(score), None, mass, ws, ws_bytes, None)

    assert call(G=17) == -1 and b"16" in lib.pqhsa_last_error()
    assert call(q=None) == -1 and call(q=(1 << 20) + 8) == -1 and call(stride=4) == -1
    assert call(dtype=_lib.F32) == -1 and call(n_max=-1) == -1 and call(T=-1) == -1 and call(ws=(1 << 20) + 16) == -1
    assert call(n_max=2**31 - 1, ws_bytes=1 << 60) == -1 and b"large" in lib.pqhsa_last_error()
    assert call(n_max=1 << 20, ws_bytes=16) == -3 and b"workspace" in lib.pqhsa_last_error()
    assert call(T=1 << 30, H=4) == -1                              # more rows than one launch numbers
    assert call(B=70000, H=1) == -1
    mass.out, mass.stride, mass.decay, mass.rows = 1 << 20, 10, 1.0, -1
    assert call(mass=ctypes.byref(mass)) == -1
    view.paged, view.block_table, view.block_size, view.max_blocks, view.stride_block = 1, 1 << 20, 16, 1, 2048
    assert call() == -1
    assert call(B=0) == 0 and call(T=0) == 0
