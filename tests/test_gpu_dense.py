"""Dense attention of one new token per sequence (``ops.dense_attend``) against an evaluation in 64 bits."""

import math

import pytest
import torch

from pqhsa_release_amd import _lib, ops
from tests.dense_util import DIM, SCALE, DenseProblem, check_close, far_away

gpu = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def run(p, *, mass=False, decay=0.9, strided=False):
    kv, rule = p.source(), p.rule()
    B, heads = p.B, p.H * p.G
    if strided:     # rows inside a wider projection, output rows inside a wider buffer
        wide = torch.full((B, 3 * heads, DIM), math.nan, dtype=p.dtype, device="cuda")
        q = wide[:, heads : 2 * heads]
        q.copy_(p.q.cuda())
        out = torch.full((B, heads + 1, DIM), 7.0, dtype=p.dtype, device="cuda")[:, :heads]
    else:
        q, out = p.q.cuda(), torch.full((B, heads, DIM), math.nan, dtype=p.dtype, device="cuda")
    lse = torch.full((B, heads), math.nan, device="cuda")
    m = m_in = None
    if mass:
        m_in = torch.rand(B, p.H, p.n_max + 2, generator=torch.Generator().manual_seed(5)).cuda()
        m = torch.full_like(m_in, 7.0)
    ops.dense_attend(q, out, kv, p.G, p.seq_lens(), n_max=p.n_max, rule=rule, lse=lse, mass=m, mass_in=m_in, decay=decay)
    torch.cuda.synchronize()
    return out, lse, m, m_in


def check(p, *, mass=False, strided=False):
    out, lse, m, m_in = run(p, mass=mass, strided=strided)
    want, want_lse, tol, lse_tol, weights, weight_tol = p.evaluate()
    check_close(out, want, tol, "out")
    check_close(lse, want_lse, lse_tol, "lse")
    if strided:
        assert bool((out.as_strided((p.B, DIM), ((p.H * p.G + 1) * DIM, 1), p.H * p.G * DIM) == 7.0).all())
    if mass:
        add, t = p.mass(weights, weight_tol)
        for b, n in enumerate(p.lens):
            old = m_in[b, :, :n].double().cpu()
            # in fp32: the decay (0.9 is no fp32 number) and its product each half a step off, then G sums of at
            # most old + add, each half a step off: (2 + G) 2^-24 of old + add
            check_close(m[b, :, :n], 0.9 * old + add[b, :, :n], t[b, :, :n] + (2 + p.G) * 2.0 ** -24 * (old + add[b, :, :n]), "mass")
            assert bool((m[b, :, n:] == 7.0).all()), "entries behind the sequence were written"


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("layout,block", [("5d", 16), ("4d", 16), ("dense", 0), ("5d", 7), ("4d", 1), ("5d", 256)])
def test_layouts_types_and_ragged_lengths(dtype, layout, block):
    check(DenseProblem([300, 1, 129, 0, 64], [1] * 5, dtype=dtype, layout=layout, block=block, seed=3), mass=True)


@gpu
@pytest.mark.parametrize("heads,groups", [(1, 1), (1, 16), (3, 7), (8, 4), (2, 5)])
def test_head_layouts(heads, groups):
    check(DenseProblem([517, 33], [1, 1], heads=heads, groups=groups, seed=11), mass=True, strided=True)


@gpu
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 127, 128, 129, 255, 257, 1000, 5003])
def test_one_sequence_of_every_tail(length):
    check(DenseProblem([length], [1], heads=1, groups=3, seed=length, extra=0))


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("kw", [dict(softcap=3.0), dict(softcap=50.0, slopes=True), dict(slopes=True), dict(window=1),
                                dict(window=100), dict(window=100, prefix=4), dict(window=64, prefix=[0, 500, 3, 9]),
                                dict(docs=4), dict(docs=3, window=90, prefix=30, softcap=10.0, slopes=True),
                                dict(window=10000), dict(prefix=10000)])
def test_score_rules(dtype, kw):
    check(DenseProblem([700, 333, 2, 0], [1] * 4, dtype=dtype, seed=21, **kw), mass=True)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("kw", [dict(), dict(softcap=5.0, slopes=True), dict(window=90, prefix=4)])
@pytest.mark.parametrize("scale", [-0.11, 0.0])
def test_scales_that_are_not_positive(dtype, kw, scale):
    check(DenseProblem([700, 333, 2, 0], [1] * 4, dtype=dtype, seed=22, scale=scale, **kw), mass=True)


@gpu
def test_long_split_range_and_large_scores():
    check(DenseProblem([40000, 17], [1, 1], heads=1, groups=2, dtype=HF, seed=5, q_gain=6.0), mass=True)


@gpu
def test_prefilled_lengths_beyond_the_bound_are_cut_to_it():
    p = DenseProblem([200], [1], heads=1, groups=2, seed=8)
    out, lse, _, _ = run(p)
    kv, rule = p.source(), p.rule()
    longer = torch.tensor([500], dtype=torch.int32, device="cuda")
    again = torch.empty_like(out)
    ops.dense_attend(p.q.cuda(), again, kv, 2, longer, n_max=200, rule=rule)
    assert torch.equal(again, out)


@gpu
def test_block_table_entries_outside_the_cache_mask_their_keys():
    p = DenseProblem([160], [1], heads=2, groups=2, block=16, poison=False, seed=9)
    kv = p.source()
    cache, table = kv.keep
    table[0, 2], table[0, 5] = -1, kv.blocks
    out = torch.empty(1, 4, DIM, dtype=p.dtype, device="cuda")
    ops.dense_attend(p.q.cuda(), out, kv, 2, p.seq_lens(), n_max=160, rule=p.rule())
    gone = torch.zeros(160, dtype=torch.bool)
    gone[32:48] = gone[80:96] = True
    q = DenseProblem([160], [1], heads=2, groups=2, block=16, poison=False, seed=9)
    q.visible = lambda b: (~gone).reshape(1, -1)
    want, _, tol, _, _, _ = q.evaluate()
    check_close(out, want, tol, "out")


@gpu
def test_mass_in_place_over_steps_and_a_replayed_graph():
    p = DenseProblem([900, 250], [1, 1], heads=2, groups=4, seed=31)
    kv, rule, q, sl = p.source(), p.rule(), p.q.cuda(), p.seq_lens()
    out = torch.empty_like(q)
    mass = torch.zeros(2, 2, 900, device="cuda")
    call = ops.DenseAttendCall(q, out, kv, 4, sl, n_max=900, rule=rule, mass=mass, mass_in=mass, decay=0.5)
    seen = []
    for _ in range(3):
        call.run()
        seen.append(mass.clone())
    eager = out.clone()
    mass.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.run()
    mass.zero_()
    for k in range(3):
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(mass, seen[k]), k
        ops.dense_attend(q, torch.empty_like(q), kv, 4, sl, n_max=900, rule=rule)   # eager work in between


@gpu
def test_two_streams_with_a_call_each():
    p = DenseProblem([3001], [1], heads=4, groups=4, seed=41)
    kv, rule, q, sl = p.source(), p.rule(), p.q.cuda(), p.seq_lens()
    want = ops.dense_attend(q, torch.empty_like(q), kv, 4, sl, n_max=3001, rule=rule).clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(q) for _ in streams]
    calls = [ops.DenseAttendCall(q, o, kv, 4, sl, n_max=3001, rule=rule) for o in outs]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                c.run()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@gpu
def test_visible_nan_and_infinite_scores_reach_the_output_of_their_row_only():
    p = DenseProblem([100, 100], [1, 1], heads=1, groups=2, poison=False, seed=51)
    p.q[0, 1, 5] = math.nan
    out, lse, _, _ = run(p)
    assert bool(out[0, 1].isnan().all()) and bool(lse[0, 1].isnan())
    rest = torch.cat([out[0, :1], out[1]])
    assert bool(rest.isfinite().all())


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
    p = DenseProblem([4000, 90], [1, 1], heads=1, groups=2, dtype=dtype, seed=61)
    check(p.set_levels(sinks(4000, 100, drop), spread=spread, gain=min(2e4, math.exp(drop) / 100), silent=5.0), mass=True)


@gpu
def test_light_keys_behind_a_sink_in_streams_of_one_chunk():
    p = DenseProblem([1024] * 64, [1] * 64, heads=8, groups=1, dtype=HF, seed=62)
    check(p.set_levels(sinks(1024, 1024, 14.0), spread=0.5, silent=5.0))


@gpu
def test_levels_of_keys_that_rise_and_fall_in_fp16():
    g = torch.Generator().manual_seed(4)
    levels = (torch.randint(0, 4, (200,), generator=g) * -6.0).repeat_interleave(20)
    p = DenseProblem([4000, 1000], [1, 1], heads=2, groups=3, dtype=HF, seed=63)
    check(p.set_levels(levels, spread=0.5, gain=2e4, silent=-16.0), mass=True)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("length", [200, 3000])
def test_infinite_and_nan_values_reach_the_output_of_the_rows_that_see_them(dtype, length):
    """As the definition has it: a positive weight times infinity, whatever the weight; elements without one stay exact."""
    p = DenseProblem([length, 150], [1, 1], heads=2, groups=3, dtype=dtype, poison=False, seed=14)
    want, want_lse, tol, lse_tol, _, _ = p.evaluate()
    p.V[0, 0, 90, 7] = math.nan
    p.V[0, 0, 100, 8] = math.inf
    p.V[0, 0, 101, 8] = -math.inf
    p.V[0, 0, 100, 9] = p.V[0, 0, length - 1, 9] = math.inf
    p.V[0, 0, 101, 10] = -math.inf
    p.V[0, 0, length - 1, 127] = math.inf
    p.V[0, 0, length:] = math.inf                        # (behind the sequence: seen by nobody)
    out, lse, _, _ = run(p)
    check_close(lse, want_lse, lse_tol, "lse")
    clean = torch.ones(2, 6, DIM, dtype=torch.bool)
    clean[0, :3, 7:11] = clean[0, :3, 127] = False
    check_close(out[clean.cuda()], want[clean], tol[clean], "out")
    assert bool(out[0, :3, 7:9].isnan().all())
    assert bool((out[0, :3, 9] == math.inf).all()) and bool((out[0, :3, 10] == -math.inf).all()) and bool((out[0, :3, 127] == math.inf).all())


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_an_infinite_value_of_a_key_with_next_to_no_weight(dtype):
    """exp(-150) is no fp32 number, but it is more than nothing; in the sink's chunk, in another, in one wave's and another's keys."""
    p = DenseProblem([1500, 200], [1, 1], heads=1, groups=2, dtype=dtype, poison=False, seed=15).set_levels([150.0] + [0.0] * 1499)
    p.V[0, 0, 57, 3] = p.V[0, 0, 7, 4] = p.V[0, 0, 1400, 5] = math.inf
    p.V[1, 0, 33, 6] = -math.inf
    out, _, _, _ = run(p)
    assert bool((out[0, :, 3:6] == math.inf).all()) and bool((out[1, :, 6] == -math.inf).all())
    out[0, :, 3:6] = out[1, :, 6] = 0.0
    assert bool(out.isfinite().all())


@gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("at", [0, 37, 700])
def test_a_key_that_stands_out_gives_its_value_unrounded(dtype, at):
    """All other weights together are under 1500 * exp(-30 + 5) = 2e-8: what is off beyond that (and beyond 2^-15, where
    fp16's base is cut) is a rounding of the one weight, which is avoidable."""
    p = DenseProblem([1500, 801], [1, 1], heads=2, groups=2, dtype=dtype, seed=71).set_levels([30.37 if j == at else 0.0 for j in range(1500)], spread=1.0)
    out, _, _, _ = run(p)
    want = p.V[:, :, at].repeat_interleave(2, 1)
    assert torch.equal(out.cpu(), want)


@gpu
def test_rows_beyond_32_bit_offsets():
    p = DenseProblem([300, 77], [1, 1], heads=8, groups=4, layout="5d", block=16, seed=17)
    near, q, sl, rule = p.source(), p.q.cuda(), p.seq_lens(), p.rule()
    far = far_away(near)
    outs = [torch.empty_like(q) for _ in range(2)]
    for kv, out in zip((near, far), outs):
        ops.dense_attend(q, out, kv, 4, sl, n_max=300, rule=rule)
    assert torch.equal(*outs)


@gpu
def test_queries_and_outputs_side_by_side_in_one_buffer():
    p = DenseProblem([90, 200, 33], [1, 1, 1], heads=2, groups=3, seed=18)
    want, _, _, _ = run(p)
    buffer = torch.full((3, 14, DIM), math.nan, dtype=p.dtype, device="cuda")
    q, out = buffer[:, :6], buffer[:, 7:13]
    q.copy_(p.q.cuda())
    ops.dense_attend(q, out, p.source(), 3, p.seq_lens(), n_max=200, rule=p.rule())
    assert torch.equal(out, want) and torch.equal(q, p.q.cuda()) and bool(buffer[:, 6].isnan().all()) and bool(buffer[:, 13].isnan().all())


@gpu
def test_refusals():
    p = DenseProblem([64, 30], [1, 1], heads=2, groups=2, seed=1)
    kv, rule, q, sl = p.source(), p.rule(), p.q.cuda(), p.seq_lens()
    out = torch.empty_like(q)

    def refused(match=None, q=q, out=out, kv=kv, groups=2, sl=sl, **kw):
        kw = {"n_max": 64, "rule": rule, **kw}
        with pytest.raises(ValueError, match=match):
            ops.dense_attend(q, out, kv, groups, sl, **kw)

    refused("device", q=q.cpu())
    refused("dtype", q=q.float())
    refused("q must", groups=1)
    refused("groups", groups=17)
    refused("n_max", n_max=kv.capacity + 1)
    refused("n_max", n_max=-1)
    refused("seq_lens", sl=sl.long())
    refused("overlap", out=out[:, :1].expand(-1, 4, -1))
    refused("overlap", out=q)
    both = torch.zeros(2, 7, DIM, dtype=p.dtype, device="cuda")
    refused("overlap", q=both[:, :4], out=both[:, 3:])
    weights = torch.zeros(3, 2, 64, device="cuda")
    refused("apart", mass=weights[:2], mass_in=weights[1:])
    refused("aligned", q=torch.empty(2 * 4 * DIM + 1, dtype=p.dtype, device="cuda")[1:].view(2, 4, DIM))
    refused("mass", mass=torch.zeros(2, 2, 63, device="cuda"))
    refused("mass", mass=torch.zeros(2, 2, 64, device="cuda", dtype=torch.float64))
    refused("mass output", mass_in=torch.zeros(2, 2, 64, device="cuda"))
    refused("decay", mass=torch.zeros(2, 2, 64, device="cuda"), decay=math.inf)
    refused("lse", lse=torch.zeros(2, 3, device="cuda"))
    refused("prefix", rule=ops.ScoreRule(scale=SCALE, prefix=torch.zeros(3, dtype=torch.int32, device="cuda")))
    refused("slopes", rule=ops.ScoreRule(scale=SCALE, slopes=torch.zeros(3, device="cuda")))
    refused("docs", rule=ops.ScoreRule(scale=SCALE, docs=torch.zeros(2, 63, dtype=torch.int32, device="cuda")))


@gpu
def test_values_for_fewer_sequences_or_tokens_than_the_keys_are_refused():
    keys = torch.zeros(2, 2, 10, DIM, device="cuda")
    for values in (keys[:1], keys[:, :1], keys[:, :, :5]):       # (of the same strides)
        assert values.stride() == keys.stride()
        with pytest.raises(ValueError, match="shape"):
            ops.kv_contiguous(keys, values)


def test_rule_refusals_without_a_gpu():
    for kw in (dict(scale=math.nan), dict(scale=1.0, softcap=-1.0), dict(scale=1.0, softcap=math.inf), dict(scale=1.0, window=-1),
               dict(scale=1.0, prefix=-2), dict(scale=1.0, prefix=torch.zeros(2)), dict(scale=1.0, slopes=torch.zeros(2)),
               dict(scale=1.0, docs=torch.zeros(2, 2))):
        with pytest.raises(ValueError):
            ops.ScoreRule(**kw)


def test_numbers_of_more_than_32_bits_are_refused():
    for kw in (dict(window=2**32 + 5), dict(window=2**31), dict(prefix=2**32 + 3), dict(prefix=2**31)):
        with pytest.raises(ValueError, match="2\\^31"):
            ops.ScoreRule(scale=1.0, **kw)
    assert ops.ScoreRule(scale=1.0, window=2**31 - 1, prefix=2**31 - 1).struct.window == 2**31 - 1
    mass = torch.zeros(1, 1, 8)
    with pytest.raises(ValueError, match="mass_rows"):
        ops._mass_struct(mass, None, 1.0, 2**32 + 1, 1, 1, 8)
    for n_max in (2**31, 2**32 + 8):
        with pytest.raises(ValueError, match="n_max"):
            ops._check_bound(ops.KvSource(None, (), torch.float32, 1, 1, 2**33), n_max)


@gpu
def test_kept_keys_of_more_than_32_bits_are_refused():
    kv = ops.kv_contiguous(*torch.zeros(2, 1, 1, 8, DIM, device="cuda"))
    dst = ops.kv_contiguous(*torch.zeros(2, 1, 1, 8, DIM, device="cuda"))
    with pytest.raises(ValueError, match="keep"):
        ops.evict(kv, dst, torch.zeros(1, 1, 8, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"), keep=2**32 + 4,
                  sink=1, recent=1, n_max=8)


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: a call that were not refused must find no GPU")
def test_c_entry_refuses_bad_arguments_before_any_gpu_work():
    import ctypes

    lib = _lib.load()
    view, score, mass = _lib.KvView(), _lib.Score(), _lib.Mass()
    view.k_base = view.v_base = 1 << 20
    view.dtype, view.stride_tok, view.stride_head, view.stride_seq = _lib.BF16, 128, 1280, 12800
    score.scale = 1.0

    def call(q=1 << 20, dtype=_lib.BF16, stride=128, B=1, H=1, G=1, n_max=10, mass=None, ws=1 << 20, ws_bytes=1 << 20):
        return lib.pqhsa_dense_attend_paged(q, dtype, 0, stride, 1 << 20, 0, 128, ctypes.byref(view), 0, B, H, G, 1 << 20, n_max,
                                            ctypes.byref(score), None, mass, ws, ws_bytes, None)

    assert call(G=17) == -1 and b"16" in lib.pqhsa_last_error()
    assert call(q=None) == -1 and call(q=(1 << 20) + 8) == -1 and call(stride=4) == -1
    assert call(dtype=_lib.F32) == -1 and b"dtype" in lib.pqhsa_last_error()
    assert call(n_max=-1) == -1 and call(ws=(1 << 20) + 16) == -1
    assert call(n_max=2**31 - 1, ws_bytes=1 << 60) == -1 and b"large" in lib.pqhsa_last_error()
    assert call(n_max=1 << 20, ws_bytes=16) == -3 and b"workspace" in lib.pqhsa_last_error()
    mass.decay = 1.0
    assert call(mass=ctypes.byref(mass)) == -1
    mass.out, mass.stride = 1 << 20, 10
    assert call(B=70000, mass=ctypes.byref(mass), ws_bytes=1 << 60) == -1 and b"many" in lib.pqhsa_last_error()
    mass.out, mass.stride = 1 << 20, 9
    assert call(mass=ctypes.byref(mass)) == -1
    view.paged, view.block_table, view.block_size, view.max_blocks, view.stride_block = 1, 1 << 20, 16, 1, 2048
    assert call() == -1                      # a paged cache without blocks
    assert call(B=0) == 0
    for score.scale, score.softcap in ((math.nan, 0.0), (3e38, 0.0), (1.0, 1e-39), (1.0, 3e38)):
        assert call() == -1
