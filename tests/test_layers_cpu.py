"""The feed-forward operators on the CPU: the plain forms against independent
statements in 64 bits, gradients against differences, the 8-bit format's edges,
refusals, and the block in the language model under the sparse optimizer."""
import math

import pytest
import torch
import torch.nn.functional as F

from gtopkssgd_b200.models import FeedForward, create_net
from gtopkssgd_b200.ops import layers_oracle as oracle
from gtopkssgd_b200.ops.activation8 import Activation8
from gtopkssgd_b200.ops.feed_forward import FeedForwardKept, feed_forward, feed_forward_backward, feed_forward_block
from gtopkssgd_b200.ops.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
from gtopkssgd_b200.ops.linear import linear, linear_backward, linear_forward

LIBRARY = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}


def _leaf(*shape):
    return torch.randn(*shape, dtype=torch.float64, requires_grad=True)


@pytest.mark.parametrize("name", list(LIBRARY))
def test_activations_and_slopes(name):
    z = torch.linspace(-6, 6, 241, dtype=torch.float64, requires_grad=True)
    y = LIBRARY[name](z)
    slope, = torch.autograd.grad(y.sum(), z)
    assert torch.allclose(oracle.act(name, z), y, rtol=1e-12, atol=1e-14)
    assert torch.allclose(oracle.act_slope(name, z), slope, rtol=1e-12, atol=1e-14)


@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_of_large_values(name):
    z = torch.tensor([1e19, 2e19, 1e25, 3e38, 400.0])
    assert torch.equal(oracle.act_slope(name, z), torch.ones(5)) and torch.equal(oracle.act_slope(name, -z), torch.zeros(5))


def test_gradients_against_differences():
    torch.manual_seed(0)
    assert torch.autograd.gradcheck(lambda *a: layer_norm(*a), (_leaf(3, 2, 7), _leaf(7), _leaf(7)))
    assert torch.autograd.gradcheck(lambda x: layer_norm(x), (_leaf(4, 5),))
    for name in ("none", "gelu", "gelu_tanh", "silu"):
        assert torch.autograd.gradcheck(lambda x, w, b, r: linear(x, w, b, name, r), (_leaf(3, 2, 5), _leaf(4, 5), _leaf(4), _leaf(3, 2, 4)))
    assert torch.autograd.gradcheck(lambda *a: feed_forward_block(*a), (_leaf(3, 2, 5), _leaf(5), _leaf(5), _leaf(6, 5), _leaf(6), _leaf(5, 6), _leaf(5)))


def test_eight_bit_gradients_are_the_formula_at_the_kept_values():
    """With 8 bits the backward pass is the exact one at the values that the codes stand for."""
    torch.manual_seed(1)
    x, w, b = torch.randn(6, 70, dtype=torch.float64), torch.randn(33, 70, dtype=torch.float64), torch.randn(33, dtype=torch.float64)
    dy = torch.randn(6, 33, dtype=torch.float64)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    linear(*leaves, "gelu", bits=8).backward(dy)
    z8, x8 = Activation8.keep(x @ w.t() + b).restore(), Activation8.keep(x).restore()
    dz = dy * oracle.act_slope("gelu", z8)
    for got, want in zip(leaves, (dz @ w, dz.t() @ x8, dz.sum(0))):
        assert torch.allclose(got.grad, want, rtol=1e-10, atol=1e-12)


# -- the 8-bit format --------------------------------------------------------------
def test_codes_at_the_edges_of_the_format():
    block = torch.zeros(1, 32)

    def code(*values):
        x = block.clone()
        x[0, :len(values)] = torch.tensor(values)
        kept = Activation8.keep(x)
        return kept.q[0, :len(values)].tolist(), int(kept.e[0, 0]) - 127, kept.restore()[0, :len(values)].tolist()

    assert code(127.0, 1.0)[:2] == ([127, 1], 0)              # 127 * 2^0 is the largest that step 1 takes
    assert code(127.0 + 2 ** -17, 1.0)[:2] == ([64, 0], 1)    # the next f32 above takes step 2; 1 / 2 is a tie, to even
    assert code(254.0, 3.0)[:2] == ([127, 2], 1)              # 1.5 is a tie, to even
    assert code(-1.0, 0.5)[:2] == ([-64, 32], -6)
    assert code(0.0)[:2] == ([0], -127) and code(0.0)[2] == [0.0]
    tiny = 2.0 ** -149
    assert code(tiny)[0] == [0] and code(tiny)[2] == [0.0]     # steps end at 2^-127
    assert code(2.0 ** -126, 2.0 ** -127)[2] == [2.0 ** -126, 2.0 ** -127]
    big = torch.finfo(torch.float32).max
    q, e, back = code(big)
    assert q == [63] and e == 122 and back == [63 * 2.0 ** 122]   # 64 would stand for more than f32 holds
    half = torch.full((1, 32), 65504.0, dtype=torch.float16)
    assert torch.equal(Activation8.keep(half).restore(), half)    # 64 * 2^10 in f32
    for bad in (math.inf, -math.inf, math.nan):
        q, e, back = code(1.0, bad)
        assert e == 255 - 127 and all(math.isnan(v) for v in back)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (3, 32), (3, 33), (2, 100), (5, 1021)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_restored_values_are_within_half_a_step(rows, cols, dtype):
    torch.manual_seed(cols)
    x = (torch.randn(rows, cols) * torch.exp(torch.randn(rows, 1) * 3)).to(dtype)
    kept = Activation8.keep(x)
    assert kept.q.shape == (rows, cols) and kept.e.shape == (rows, -(-cols // 32)) and kept.restore().dtype == dtype
    step = torch.exp2(kept.e.double() - 127).repeat_interleave(32, 1)[:, :cols]
    assert torch.all((kept.restore().double() - x.double()).abs() <= step / 2)
    most = F.pad(x.double().abs(), (0, -cols % 32)).view(rows, -1, 32).amax(2)
    assert torch.all(most <= 127 * torch.exp2(kept.e.double() - 127))       # large enough
    assert torch.all(most > 127 * torch.exp2(kept.e.double() - 128))        # and the least such step
    again = Activation8.keep(kept.restore())                                # what is restored is kept exactly
    assert torch.equal(again.restore(), kept.restore())


def test_shapes_lengths_and_strides():
    x = torch.randn(5, 3, 24).transpose(0, 1)
    y, mean, rstd = layer_norm_forward(x)
    assert y.shape == x.shape and mean.shape == x.shape[:-1]
    assert torch.allclose(y, F.layer_norm(x, (24,)), atol=1e-5)
    assert layer_norm(torch.empty(0, 8)).shape == (0, 8)
    w = torch.randn(8, 24)
    y, z = linear_forward(x, w, activation="relu", keep=True)
    assert y.shape == (3, 5, 8) and z.shape == (15, 8)
    assert linear_forward(x, w)[1] is None and linear_forward(x, w, keep=True)[1] is None
    assert linear(torch.empty(0, 24), w).shape == (0, 8)
    dx, dw, db = linear_backward(torch.empty(0, 8), torch.empty(0, 24), w)
    assert dx.shape == (0, 24) and not dw.any() and not db.any()
    dx, dw, db = linear_backward(torch.randn(3, 5, 8), x, w, need=(False, True, False))
    assert dx is None and db is None and dw.shape == w.shape
    kept = Activation8.keep(x)
    assert kept.shape == x.shape and kept.restore().shape == x.shape


def _check_empty(device):
    for shape in ((0, 3), (5, 0), (2, 3, 0), (0, 3, 0), (3, 0, 4), (0,), (0, 0)):
        x = torch.zeros(shape, device=device)
        kept = Activation8.keep(x)
        assert kept.restore().shape == x.shape and kept.shape == x.shape
        dz, db = kept.backward(x, "gelu")
        assert dz.shape == x.shape and db.shape == shape[-1:] and not db.any()
    for shape in ((0, 8), (3, 0, 8), (0, 3, 8)):
        x = torch.zeros(shape, device=device, requires_grad=True)
        p = [torch.ones(n, device=device, requires_grad=True) for n in (8, 8, (5, 8), 5, (8, 5), 8)]
        for bits in (0, 8):
            y = linear(x, p[2], p[3], "gelu", bits=bits)
            z = feed_forward_block(x, *p, "gelu", 1e-5, bits)
            assert y.shape == (*shape[:-1], 5) and z.shape == shape
            (y.sum() + z.sum()).backward()
        assert x.grad.shape == shape and not any(t.grad.any() for t in p)
    w = torch.zeros(0, 8, device=device)
    y, z = linear_forward(torch.ones(3, 8, device=device), w, activation="gelu", keep=True, bits=8)
    assert y.shape == z.shape == (3, 0)
    dx, dw, db = linear_backward(y, torch.ones(3, 8, device=device), w, "gelu", z)
    assert dx.shape == (3, 8) and not dx.any() and dw.shape == (0, 8) and db.shape == (0,)


def test_empty_axes():
    _check_empty("cpu")


def test_refusals():
    x, w, b = torch.randn(4, 6), torch.randn(5, 6), torch.randn(5)
    with pytest.raises(TypeError):
        layer_norm(torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(2, 0))
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(5))
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(6, dtype=torch.bfloat16))
    y, mean, rstd = layer_norm_forward(x)
    with pytest.raises(ValueError):
        layer_norm_backward(y[:, :5], x, mean, rstd)
    with pytest.raises(ValueError):
        layer_norm_backward(y, x, mean[:3], rstd)
    with pytest.raises(ValueError):
        linear(x, torch.randn(5, 7))
    with pytest.raises(ValueError):
        linear(x, w, torch.randn(6))
    with pytest.raises(ValueError):
        linear(x, w, b, "swish")
    with pytest.raises(ValueError):
        linear(x, w, b, residual=torch.randn(5))          # a residual is not broadcast
    with pytest.raises(ValueError):
        linear(x, w.bfloat16())
    with pytest.raises(ValueError):
        linear(x, w, b, "gelu", bits=4)
    with pytest.raises(ValueError):
        linear(x, torch.randn(5, 0))
    with pytest.raises(ValueError):
        linear_backward(torch.randn(4, 5), x, w, "gelu", None)
    with pytest.raises(ValueError):
        linear_backward(torch.randn(4, 5), x, w, "gelu", torch.randn(4, 6))
    kept = Activation8.keep(x)
    with pytest.raises(ValueError):
        Activation8(kept.q.int(), kept.e, torch.float32)
    with pytest.raises(ValueError):
        Activation8(kept.q, kept.e[:, :0], torch.float32)
    with pytest.raises(ValueError):
        Activation8(kept.q, kept.e, torch.float32, (5, 6))
    with pytest.raises(TypeError):
        Activation8(kept.q, kept.e, torch.int32)
    with pytest.raises(ValueError):
        kept.backward(torch.randn(4, 5), "gelu")
    with pytest.raises(ValueError):
        kept.backward(torch.randn(4, 6), "elu")
    p = [torch.ones(6), torch.zeros(6), torch.randn(8, 6), torch.zeros(8), torch.randn(6, 8), torch.zeros(6)]
    with pytest.raises(ValueError):
        feed_forward(x, *p, activation="none")
    with pytest.raises(ValueError):
        feed_forward(x, *p[:4], torch.randn(8, 6), p[5])
    y, kept = feed_forward(x, *p)
    with pytest.raises(ValueError):
        feed_forward_backward(y[:3], kept, p[0], p[1], p[2], p[4])
    with pytest.raises(ValueError):
        feed_forward_backward(y, FeedForwardKept(kept.x, kept.mean, kept.rstd, kept.z[:, :7]), p[0], p[1], p[2], p[4])
    with pytest.raises(ValueError):
        FeedForward(8, 16, activation="none")


def test_refusals_of_a_block_s_statistics_and_of_scalars():
    x = torch.randn(4, 6)
    p = [torch.ones(6), torch.zeros(6), torch.randn(8, 6), torch.zeros(8), torch.randn(6, 8), torch.zeros(6)]
    with pytest.raises(ValueError):
        linear(torch.tensor(1.0), torch.randn(5, 6))
    for gone in (0, 1):
        with pytest.raises(ValueError):
            feed_forward(x, *(None if i == gone else t for i, t in enumerate(p)))
    y, kept = feed_forward(x, *p)
    with pytest.raises(ValueError):
        feed_forward_backward(y, kept, None, p[1], p[2], p[4])
    elsewhere = torch.empty(4, device="meta")
    with pytest.raises(ValueError):
        feed_forward_backward(y, kept._replace(mean=elsewhere), p[0], p[1], p[2], p[4])
    with pytest.raises(ValueError):
        feed_forward_backward(y, kept._replace(rstd=elsewhere), p[0], p[1], p[2], p[4])
    with pytest.raises(ValueError):
        layer_norm_backward(y, x, elsewhere, kept.rstd)


def test_block_forward_and_backward_parts_agree_with_autograd():
    torch.manual_seed(3)
    x = torch.randn(2, 5, 40, dtype=torch.float64)
    m = FeedForward(40, 72, activation="silu").double()
    leaf = x.clone().requires_grad_()
    dy = torch.randn_like(x)
    y = m(leaf)
    y.backward(dy)
    z = F.linear(F.layer_norm(x, (40,), m.norm_weight, m.norm_bias, 1e-5), m.w1, m.b1)
    assert torch.allclose(y, x + F.linear(F.silu(z), m.w2, m.b2), rtol=1e-10, atol=1e-12)
    p = [m.norm_weight, m.norm_bias, m.w1, m.b1, m.w2, m.b2]
    _, kept = feed_forward(x, *p, activation="silu")
    got = feed_forward_backward(dy, kept, *p[:3], m.w2, "silu")
    for a, b in zip(got, [leaf.grad] + [t.grad for t in p]):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)


def test_block_gives_the_gradients_that_are_wanted():
    x = torch.randn(4, 6)
    p = [torch.ones(6), torch.zeros(6), torch.randn(8, 6), torch.zeros(8), torch.randn(6, 8), torch.zeros(6)]
    y, kept = feed_forward(x, *p)
    full = feed_forward_backward(y, kept, *p[:3], p[4])
    for rows in (4, 0):
        some = FeedForwardKept(kept.x[:rows], kept.mean[:rows], kept.rstd[:rows], kept.z[:rows])
        for i in range(128):
            need = tuple(bool(i >> j & 1) for j in range(7))
            got = feed_forward_backward(y[:rows], some, *p[:3], p[4], need=need)
            assert all((a is None) != n and (a is None or a.shape == (rows, 6) or torch.equal(a, b) or not rows) for n, a, b in zip(need, got, full))
    with pytest.raises(ValueError):
        feed_forward_backward(y, kept, *p[:3], p[4], need=(True, True))


@pytest.mark.parametrize("bits", [0, 8])
def test_language_model_with_feed_forward_blocks_trains_sparsely(bits):
    from gtopkssgd_b200.parallel.compression import compressors
    from gtopkssgd_b200.parallel.distributed_optimizer import DistributedOptimizer
    torch.manual_seed(0)
    plain, _ = create_net(0, "lstm", vocab_size=50, batch_size=4, num_steps=5)
    assert not any("feed_forward" in n for n in plain.state_dict())
    from gtopkssgd_b200.models import lstm
    net = lstm(vocab_size=50, embedding_dim=36, num_steps=5, batch_size=4, ff_layers=2, ff_dim=72, ff_bits=bits)
    opt = DistributedOptimizer(torch.optim.SGD(net.parameters(), lr=0.1), net.named_parameters(), compression=compressors["gtopk"], is_sparse=True,
                               density=0.05)
    tokens = torch.randint(0, 50, (6, 4))
    losses = []
    for _ in range(60):
        opt.zero_grad()
        logits, _ = net(tokens[:-1], net.init_hidden())
        loss = F.cross_entropy(logits.view(-1, 50), tokens[1:].reshape(-1))
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    opt.stop()
    assert all(math.isfinite(v) for v in losses) and losses[-1] < 0.99 * losses[0]


# -- what autograd keeps ----------------------------------------------------------------
def _passes(bits, device="cpu", rows=6):
    """(linear, block) under autograd, on leaves of their own."""
    torch.manual_seed(2)
    x, w, b = (torch.randn(*s).to(device).requires_grad_() for s in ((rows, 40), (24, 40), (24,)))
    p = [torch.randn(*s).to(device).requires_grad_() for s in ((rows, 40), (40,), (40,), (24, 40), (24,), (40, 24), (40,))]
    return [(lambda: linear(x, w, b, "gelu", bits=bits), (x, w, b)), (lambda: feed_forward_block(*p, "gelu", 1e-5, bits), p)]


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("bits", [0, 8])
def test_what_is_kept_goes_through_autograd(which, bits):
    """Saved tensors: hooks see the 8-bit copies, may bring them back with other strides, and nothing of them outlives the
    backward pass, though the result does."""
    from torch.multiprocessing.reductions import StorageWeakRef
    run, leaves = _passes(bits)[which]
    want_y = run()
    want_y.sum().backward()
    want = [t.grad.clone() for t in leaves]
    kinds, codes = [], []
    keep = oracle.keep8

    def pack(t):
        kinds.append(t.dtype)
        return t.clone(memory_format=torch.contiguous_format)

    def watched(x):
        pair = keep(x)
        codes.extend(StorageWeakRef(t.untyped_storage()) for t in pair)
        return pair

    with pytest.MonkeyPatch.context() as patch:
        patch.setattr(oracle, "keep8", watched)
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = run()
        assert torch.equal(y, want_y)
        assert kinds.count(torch.int8) == kinds.count(torch.uint8) == (2 if bits else 0)
        assert len(codes) == (4 if bits else 0) and all(ref.expired() for ref in codes)   # the hook's copies are what is held
        for t in leaves:
            t.grad = None
        y.sum().backward()
        assert all(torch.equal(t.grad, g) for t, g in zip(leaves, want))
        codes.clear()   # without hooks: held by the graph until the backward pass, not by the result
        y = run()
    assert not any(ref.expired() for ref in codes)
    y.sum().backward()
    assert all(ref.expired() for ref in codes) and y.grad_fn is not None
    with pytest.raises(RuntimeError):
        y.sum().backward()


@pytest.mark.parametrize("which", [0, 1])
def test_nothing_is_kept_where_gradients_are_off(which, monkeypatch):
    from gtopkssgd_b200.ops import feed_forward as block_module
    from gtopkssgd_b200.ops import linear as linear_module
    run, leaves = _passes(8)[which]
    want = run().detach()
    copies, asked = [], []
    keep = oracle.keep8
    monkeypatch.setattr(oracle, "keep8", lambda x: copies.append(x) or keep(x))
    for module in (linear_module, block_module):
        whole = module._forward
        monkeypatch.setattr(module, "_forward", lambda x, w, b, act, r, kept, *rest, whole=whole: asked.append(kept) or whole(x, w, b, act, r, kept, *rest))
    with torch.no_grad():
        y = run()
    with torch.inference_mode():
        assert torch.equal(run(), want)
    assert torch.equal(y, want) and not y.requires_grad and not copies and asked and not any(asked)
    for t in leaves:
        t.requires_grad_(False)
    assert torch.equal(run(), want) and not copies and not any(asked)
    for t in leaves:
        t.requires_grad_()
    run().sum().backward()
    assert len(copies) == 2 and any(asked) and all(t.grad is not None for t in leaves)


@pytest.mark.parametrize("bits", [0, 8])
def test_a_frozen_weight_keeps_no_input(bits):
    x, w, b = torch.randn(6, 40), torch.randn(24, 40), torch.randn(24, requires_grad=True)
    for first in (False, True):
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(tuple(t.shape)) or t, lambda t: t):
            y = linear(x.requires_grad_(first), w, b, "gelu", bits=bits)
        assert (6, 40) not in saved and (6, 24) in saved
        y.sum().backward()
        assert (x.grad is not None) == first and b.grad is not None


# -- failures -----------------------------------------------------------------------
def test_a_product_whose_wait_ran_out_stops_the_training(monkeypatch):
    from gtopkssgd_b200 import settings
    from gtopkssgd_b200.ops import lib
    from gtopkssgd_b200.ops import linear as module
    from gtopkssgd_b200.parallel.compression import compressors
    from gtopkssgd_b200.parallel.distributed_optimizer import DistributedOptimizer
    net = torch.nn.Linear(8, 4)
    opt = DistributedOptimizer(torch.optim.SGD(net.parameters(), lr=0.1), net.named_parameters(), compression=compressors["gtopk"], is_sparse=True,
                               density=0.1)
    word = []
    monkeypatch.setattr(module, "status", lambda: word[0])
    opt.check_status()                                    # no product launched: the device is not asked
    monkeypatch.setattr(module, "_launched", True)
    word[:] = [0]
    opt.check_status()
    word[:] = [4]
    with pytest.raises(lib.GtopkNativeError, match="code location 4"):
        opt.check_status()
    with pytest.raises(lib.GtopkNativeError):
        module.check_status()
    word[:] = [0]
    opt.stop()
    # the limit is the framework's own, and launching says that there is something to ask for
    calls = []
    monkeypatch.setattr(lib, "calls", lambda: type("Calls", (), {"gtk_k8_gemm": staticmethod(lambda *a: calls.append(a) or 0)}))
    monkeypatch.setattr(settings, "WAIT_LIMIT_MS", 125.0)
    monkeypatch.setattr(module, "_launched", False)
    operand = module.Operand(16, 64, 1, 0, 0, None)
    module.product(64, 64, 64, operand, False, operand, False, torch.empty(64, 64), 0)
    assert module._launched and calls[0][-2] == 125_000_000
