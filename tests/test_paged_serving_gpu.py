"""Serving from the paged cache as batches come: padding rows, sequences without rows, what the operators refuse."""

import pytest
import torch

import generative_recommenders_b200 as G
from generative_recommenders_b200 import hstu_attention, paged_stu
from oracle import paged_oracle as P

DEV = "cuda:0"


def offsets_of(counts, device=DEV):
    return torch.tensor([0] + list(counts)).cumsum(0).to(device)


@pytest.mark.parametrize("length_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("offset_type", [torch.int32, torch.int64])
def test_positions_of_new_rows(length_type, offset_type):
    for cached, new, rows in (([5, 0, 7], [2, 0, 4], 6), ([5, 0, 7], [2, 0, 4], 9), ([3], [0], 2), ([], [], 3), ([9], [1], 1)):
        pos = paged_stu._new_positions(torch.tensor(cached, dtype=length_type), offsets_of(new, "cpu").to(offset_type), rows)
        want = [c + i for c, n in zip(cached, new) for i in range(n)]
        assert pos.dtype == length_type and pos.shape == (rows,) and pos[:len(want)].tolist() == want


def layer_of(dtype, **options):
    torch.manual_seed(3)
    layer = G.RotarySTULayer(G.RotarySTULayerConfig(embedding_dim=96, num_heads=2, hidden_dim=64, attention_dim=64,
                                                    output_dropout_ratio=0.0, max_positions=400, **options))
    return layer.to(DEV).to(dtype).eval()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new,padding", [([3, 0, 1], 4), ([40, 20, 0], 130), ([0, 0, 0], 5)])
def test_padding_rows(new, padding, dtype):
    """Rows past the last offset are in no sequence: the others and the cache are what they are without them."""
    layer = layer_of(dtype)
    cached = torch.tensor([30, 0, 64], device=DEV)
    table = torch.arange(21, dtype=torch.int32, device=DEV).view(3, 7)
    rows = sum(new)
    x = torch.randn(rows + padding, 96, device=DEV).to(dtype)
    caches = [G.PagedKVCache(torch.zeros(21, 2, G.PagedKVCache.page_bytes(16, 64), dtype=torch.uint8, device=DEV), 16, 64)
              for _ in range(2)]
    outs = [layer.paged_forward(y, c, table, cached, offsets_of(new), 200) for y, c in zip((x[:rows], x), caches)]
    assert torch.equal(caches[0].pages, caches[1].pages)
    assert outs[1].shape == x.shape and torch.isfinite(outs[1]).all()
    if rows:
        # (where sums are cut depends on the number of rows)
        assert float((outs[1][:rows] - outs[0]).float().norm()) <= (1e-2 if dtype == torch.bfloat16 else 1e-4) * float(outs[0].float().norm())
    u = layer._uqvk(x)[0]
    alone = layer._output(torch.zeros(rows + padding, 2, 64, device=DEV, dtype=dtype), u, x)
    assert torch.equal(outs[1][rows:], alone[rows:])


@pytest.mark.gpu
def test_a_batch_of_no_sequences():
    layer = layer_of(torch.bfloat16)
    cache = layer.new_cache(2, 16)
    none = torch.zeros(0, dtype=torch.long, device=DEV)
    x = torch.randn(3, 96, device=DEV).bfloat16()
    out = layer.paged_forward(x, cache, torch.zeros(0, 0, dtype=torch.int32, device=DEV), none, torch.zeros(1, dtype=torch.long, device=DEV), 64)
    assert out.shape == x.shape and torch.isfinite(out).all()


@pytest.mark.gpu
def test_a_cache_of_no_heads_is_refused():
    with pytest.raises(RuntimeError, match="no heads"):
        G.PagedKVCache.allocate(4, 0, 64, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("field,value", [("page_size", 32), ("head_dim", 128), ("pages", torch.zeros(4, 2, 100, dtype=torch.uint8)),
                                         ("pages", torch.zeros(4, 2, 1088, dtype=torch.int8)), ("pages", torch.zeros(4, 1088, dtype=torch.uint8))])
def test_fields_that_do_not_fit_any_more(field, value):
    """A cache's fields can be replaced; every call looks at them before it hands them on."""
    cache = G.PagedKVCache.allocate(4, 2, 64, 16)
    setattr(cache, field, value.to(DEV) if isinstance(value, torch.Tensor) else value)
    d = cache.head_dim
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    one, x = torch.ones(1, dtype=torch.long, device=DEV), torch.zeros(1, 2, d, device=DEV)
    with pytest.raises((RuntimeError, TypeError)):
        G.append_paged_kv(cache, x, x, table, one, offsets_of([1]))
    with pytest.raises((RuntimeError, TypeError)):
        G.read_paged_kv(cache, table, offsets_of([1]), 1)
    with pytest.raises((RuntimeError, TypeError)):
        G.paged_mha(16, 1.0, x, cache, table, one, offsets_of([1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 12, 40])
def test_rows_before_the_first_offset_and_past_the_last(rows, dtype):
    """Rows of q that no sequence has are zeros, on either side."""
    cache = G.PagedKVCache(torch.full((4, 2, G.PagedKVCache.page_bytes(64, 64)), 0x3e, dtype=torch.uint8, device=DEV), 64, 64)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    lengths, off = torch.tensor([100, 77], device=DEV), 5 + offsets_of([rows, rows])
    q = torch.randn(5 + 2 * rows + 9, 4, 64, device=DEV).to(dtype)
    for act in ("silu", "softmax"):
        torch.full_like(q, float("nan"))   # (what the allocator hands out next)
        out = G.paged_mha(128, 0.1, q, cache, table, lengths, off, activation=act)
        same = G.paged_mha(128, 0.1, q[5:5 + 2 * rows], cache, table, lengths, off - 5, activation=act)
        assert float(out[:5].abs().sum()) == 0 and float(out[5 + 2 * rows:].abs().sum()) == 0
        assert torch.isfinite(same).all()
        assert float((out[5:5 + 2 * rows] - same).float().norm()) <= (2.0 ** -7 if dtype == torch.bfloat16 else 1e-5) * float(same.float().norm())
    none = G.paged_mha(128, 0.1, q, cache, table[:0], lengths[:0], torch.zeros(1, dtype=torch.long, device=DEV))
    assert float(none.abs().sum()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(64, 32), (128, 64), (128, 20), (256, 64), (96, 32), (64, 64)])
def test_positions_outside_the_tables_with_a_part_rotated(d, rotary, interleaved):
    """The whole row is NaN, also what is not rotated; with and without a norm, forward and backward."""
    cos, sin = G.rotary_tables(16, rotary, device=DEV)
    pos = torch.tensor([0, 15, 16, -1, 3], device=DEV)
    bad = torch.tensor([False, False, True, True, False])
    for weight in (None, torch.ones(d, device=DEV)):
        for dtype in (torch.float32, torch.bfloat16):
            x = torch.randn(5, 2, d, device=DEV).to(dtype).requires_grad_()
            y = G.qk_norm_rotary(x, None, pos, cos, sin, weight, interleaved=interleaved)[0]
            (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
            for t in (y.detach(), dx):
                nan = torch.isnan(t).flatten(1).cpu()
                assert torch.equal(nan.all(1), bad) and torch.equal(nan.any(1), bad)
            if d in G.paged_cache.HEAD_DIMS:
                cache = G.PagedKVCache.allocate(2, 2, d, 16)
                table = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV)
                k = x.detach()
                G.append_paged_kv(cache, k, k, table, torch.tensor([14], device=DEV), offsets_of([5]), cos, sin, interleaved, weight)
                both = G.read_paged_kv(cache, table, offsets_of([19]), 19)
                nan = torch.isnan(both[0][14:]).flatten(1).cpu()
                want = torch.tensor([False, False, True, True, True])
                assert torch.equal(nan.all(1), want) and torch.equal(nan.any(1), want) and torch.isfinite(both[1][14:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,k_heads", [(0, 0), (0, 3), (3, 0)])
def test_gradients_of_the_weights_of_no_heads(q_heads, k_heads):
    w = [torch.ones(64, device=DEV, requires_grad=True) for _ in range(2)]
    q, k = (torch.randn(5, h, 64, device=DEV, requires_grad=True) for h in (q_heads, k_heads))
    for _ in range(3):
        out = G.qk_norm_rotary(q, k, q_weight=w[0], k_weight=w[1])
        dy = tuple(torch.ones_like(t) for t in out)
        poison = [torch.full((64,), float("nan"), device=DEV) for _ in range(8)]   # (what the allocator hands out next)
        del poison
        dw = torch.autograd.grad(out, w, dy)
        for grad, heads in zip(dw, (q_heads, k_heads)):
            assert torch.isfinite(grad).all() and (float(grad.abs().sum()) == 0) == (heads == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [None, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("params", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_of_another_type_than_the_parameters(rows, params, autocast):
    """What ``STULayer`` takes and gives, in training and served."""
    layer = layer_of(params)
    plain = G.STULayer(G.STULayerConfig(embedding_dim=96, num_heads=2, hidden_dim=64, attention_dim=64, output_dropout_ratio=0.0))
    plain = plain.to(DEV).to(params).eval()
    x = torch.randn(50, 96, device=DEV).to(rows)
    off = offsets_of([20, 30])
    with torch.autocast("cuda", autocast or torch.bfloat16, enabled=autocast is not None):
        outs = []
        for m in (plain, layer):
            leaf = x.clone().requires_grad_()
            outs.append(m(leaf, off[1:] - off[:-1], off, 64, None))
            outs[-1].float().square().mean().backward()
            assert leaf.grad.dtype == rows and torch.isfinite(leaf.grad).all()
        cache = layer.new_cache(4, 64)
        served = layer.paged_forward(x, cache, torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2),
                                     torch.zeros(2, dtype=torch.long, device=DEV), off, 64)
    for p in layer.parameters():
        assert p.grad is not None and p.grad.dtype == params and torch.isfinite(p.grad).all()
    assert outs[0].dtype == outs[1].dtype == served.dtype
    # (the served rows go through 4 bits)
    assert float((served.float() - outs[1].float()).norm()) <= 0.25 * float(outs[1].float().norm())


def test_the_16_bit_cache_is_not_served_from():
    layer = G.RotarySTULayer(G.RotarySTULayerConfig(embedding_dim=8, num_heads=1, hidden_dim=64, attention_dim=64))
    with pytest.raises(NotImplementedError, match="paged_forward"):
        layer.cached_forward(torch.zeros(2, 8), None)
    with pytest.raises(NotImplementedError, match="paged_forward"):
        G.STUStack([layer]).cached_forward(torch.zeros(2, 8), None)


def test_only_causal_layers_are_served():
    layer = G.RotarySTULayer(G.RotarySTULayerConfig(embedding_dim=8, num_heads=1, hidden_dim=64, attention_dim=64, causal=False))
    with pytest.raises(AssertionError, match="causal"):
        layer.paged_forward(torch.zeros(2, 8), None, None, torch.zeros(1, dtype=torch.long), offsets_of([2], "cpu"), 8)


def test_every_operator_is_told_the_kernel(monkeypatch):
    layer = G.RotarySTULayer(G.RotarySTULayerConfig(embedding_dim=8, num_heads=1, hidden_dim=64, attention_dim=64, max_positions=9))
    layer._hammer_kernel = object()
    told = {}

    def fake(name, result):
        def op(*args, kernel=None, **kwargs):
            told[name] = kernel
            return result
        monkeypatch.setattr(paged_stu, name, op)

    x = torch.zeros(2, 1, 64)
    fake("hstu_compute_uqvk", (x, x, x, x))
    fake("qk_norm_rotary", (x, x))
    fake("append_paged_kv", None)
    fake("paged_mha", x)
    fake("hstu_mha", x)
    fake("hstu_compute_output", x)
    layer.paged_forward(torch.zeros(2, 8), None, None, torch.zeros(1, dtype=torch.long), offsets_of([2], "cpu"), 8)
    assert len(told) == 5 and all(kernel is layer._hammer_kernel for kernel in told.values())
    told.clear()
    layer(torch.zeros(2, 8), torch.tensor([2]), offsets_of([2], "cpu"), 8, None)
    assert len(told) == 4 and all(kernel is layer._hammer_kernel for kernel in told.values())


FEW = [([600], [1]), ([900, 300], [1, 1]), ([500, 200], [8, 5]), ([400, 30], [16, 12])]


@pytest.mark.gpu
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("lengths,new", FEW)
def test_weights_of_few_rows_keep_sixteen_bits(lengths, new, softmax):
    """The kernel for few rows rounds weights to the sum of two bfloat16 numbers.  float16 results, element by element: 2^-16 of
    every weight, 2^-16 of the sizes that a score is the sum of, half a unit of the result."""
    d, H = 128, 2
    g = torch.Generator().manual_seed(5)
    need = [-(-n // 64) for n in lengths]
    pool = torch.randint(0, 256, (sum(need), H, G.PagedKVCache.page_bytes(64, d)), generator=g).to(torch.uint8)
    codes = pool[..., :64 * d]
    codes.copy_(torch.where(codes & 15 == 0, codes | 8, codes))
    codes.copy_(torch.where(codes >> 4 == 0, codes | 128, codes))
    scales = (torch.rand(sum(need), H, 2 * 64 * d // 64, generator=g) * 0.3 + 0.2).bfloat16()
    pool[..., 64 * d:] = scales.view(torch.uint8)
    cache = G.PagedKVCache(pool.to(DEV), 64, d)
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(n) + sum(need[:b])
    q = torch.randn(sum(new), 4, d, generator=g).half().to(DEV)
    got = G.paged_mha(1, d ** -0.5, q, cache, table.to(DEV), torch.tensor(lengths, device=DEV), offsets_of(new),
                      activation="softmax" if softmax else "silu", attn_scale=0.02).double()
    at = 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        k, v = (x.to(DEV).repeat_interleave(2, 1).transpose(0, 1) for x in P.read_rows(cache, table[b], n)[:2])
        x = q[at:at + m].double().transpose(0, 1)
        s, off = x @ k.transpose(1, 2) * d ** -0.5, 2.0 ** -16 * (x.abs() @ k.abs().transpose(1, 2)) * d ** -0.5
        seen = torch.arange(n, device=DEV)[None] <= torch.arange(n - m, n, device=DEV)[:, None]
        none = torch.zeros((), dtype=torch.float64, device=DEV)
        if softmax:
            w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
            error, common = w * (2.0 ** -16 + off), (w * off).sum(-1, keepdim=True) + 2.0 ** -20
        else:
            w = torch.where(seen, s * torch.sigmoid(s) * 0.02, none)
            error, common = torch.where(seen, 2.0 ** -16 * w.abs() + 1.1 * 0.02 * off, none), 2.0 ** -20
        out = w @ v
        bound = error @ v.abs() + out.abs() * (common + 2.0 ** -11) + 2.0 ** -25
        at += m
        assert bool(((got[at - m:at].transpose(0, 1) - out).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new,width", [([1, 0, 1], 7), ([3, 1, 2], 100), ([40, 20, 7], 7), ([300, 20, 0], 100)])
def test_a_captured_step_is_the_step(new, width, monkeypatch):
    """``paged_forward`` in a CUDA graph, replayed with other rows, lengths, offsets and pages."""
    monkeypatch.setattr(hstu_attention, "_CHECK_STATUS", False)   # (which waits for every call)
    layer = layer_of(torch.bfloat16, max_attn_len=50)
    rows = sum(new) + 3
    caches = [G.PagedKVCache(torch.zeros(90, 2, G.PagedKVCache.page_bytes(16, 64), dtype=torch.uint8, device=DEV), 16, 64)
              for _ in range(2)]
    table = torch.full((3, width), -1, dtype=torch.int32, device=DEV)
    x = torch.zeros(rows, 96, device=DEV, dtype=torch.bfloat16)
    cached, off = torch.zeros(3, dtype=torch.long, device=DEV), torch.zeros(4, dtype=torch.long, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            layer.paged_forward(x, caches[0], table, cached, off, 200)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.paged_forward(x, caches[0], table, cached, off, 200)
    done = torch.zeros(3, dtype=torch.long)
    g = torch.Generator().manual_seed(1)
    pages = min(width, 30)
    table[:, :pages] = torch.randperm(90, generator=g)[:3 * pages].view(3, pages).to(torch.int32).to(DEV)
    for step in range(3):
        n = torch.tensor(new).roll(step)
        x.copy_(torch.randn(rows, 96, generator=g))
        cached.copy_(done)
        off.copy_(torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)]))
        graph.replay()
        want = layer.paged_forward(x, caches[1], table, cached, off, 200)
        # (rows without a page, or past the rotation's tables, are NaN in both)
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0))
        assert torch.equal(caches[0].pages, caches[1].pages)
        done += n


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 7])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scores_of_few_rows_are_sums_in_32_bits(d, new):
    """Rows that see one position: the result is SiLU of one score times V, in float16.  The score is a sum of terms of either
    sign; what it may be off by goes with the terms' sizes: sums of up to twice those (odd codes stand 64 above themselves)
    in four steps a group of 64, 2^-23 each, are 1.4e-6 of them; one rounding of the weight's 16 bits and of the result."""
    B, H = 300, 4
    g = torch.Generator().manual_seed(d + new)
    pool = torch.randint(0, 256, (B, H, G.PagedKVCache.page_bytes(16, d)), generator=g).to(torch.uint8)
    pool[..., 16 * d:] = (torch.rand(B, H, 2 * 16 * d // 64, generator=g) * 0.3 + 0.2).bfloat16().view(torch.uint8)
    cache = G.PagedKVCache(pool.to(DEV), 16, d)
    table = torch.arange(B, dtype=torch.int32)[:, None]
    q = torch.randn(B * new, H, d, generator=g).half().to(DEV)
    # candidates at the start of a sequence see themselves alone
    many = torch.full((B,), new, device=DEV)
    got = G.paged_mha(1, d ** -0.5, q, cache, table.to(DEV), many, offsets_of([new] * B), many, attn_scale=1.0).double()
    rows = [P.read_rows(cache, table[b], new)[:2] for b in range(B)]
    k, v = (torch.cat(x).to(DEV) for x in zip(*rows))
    s, sizes = (q.double() * k).sum(-1, keepdim=True) * d ** -0.5, (q.double() * k).abs().sum(-1, keepdim=True) * d ** -0.5
    w = s * torch.sigmoid(s)
    bound = (2.0 ** -16 * w.abs() + 1.1 * 1.4e-6 * sizes) * v.abs() + 2.0 ** -11 * (w * v).abs() + 2.0 ** -25
    assert float(((got - w * v).abs() / bound).max()) <= 1
