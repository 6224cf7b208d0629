"""GraniteEngine with 4-bit experts (``experts="mx4"``) against the oracle of the same
weights: expert weights drawn from the values that both formats hold (e2m1 magnitudes times
a power of two a row), so that quantisation at load changes nothing and every step must meet
the fp8 engine's bound, 5e-2 of max |logit| (tests/test_gpu_granite.py)."""
import pytest
import torch

from oracle import hybrid_ref as H
from tests._hybrid_steps import check_steps, feed_of
from tilefoundry_amd.hybrid.granite import GraniteConfig, GraniteEngine, mx4_shared, \
    synthetic_weights

CFG = dict(layers=3, attention_layers=(1,), vocab=4096)


def _weights(cfg, seed, dev):
    w = synthetic_weights(cfg, seed=seed, device=dev)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    half = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=dev)
    grid = torch.cat((half, -half)).to(torch.float8_e4m3fn).view(torch.uint8)
    for name, scale in (("w_gate", "s_gate"), ("w_up", "s_up"), ("w_down", "s_down"),
                        ("w_shared_in", "w_shared_in_scale"),
                        ("w_shared_out", "w_shared_out_scale")):
        for i in range(cfg.layers):
            t = w[f"layer{i}.{name}"]
            t.copy_(grid[torch.randint(0, 16, t.shape, generator=g, device=dev)])
            s = w[f"layer{i}.{scale}"]
            s.copy_(2.0 ** torch.randint(-8, -6, s.shape, generator=g, device=dev))
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("rows,experts,top_k", [(1, 12, 4), (2, 12, 4), (8, 72, 10), (12, 12, 4),
                                                (12, 72, 10)])
def test_mx4_engine_matches_oracle_steps(gpu_device, rows, experts, top_k):
    """Steps whose experts run in two launches (up to 128 places) and, with 12 rows of 12
    places, by a list of tiles.

    Routing is followed for swaps within 16 ulps of the k-th router logit.  The fp8 engine's
    four cover sums of other orders at the oracle's own rounding points; here the experts'
    output is rounded once where the oracle rounds five times (each output, its product with
    the weight, the two sums, the multiplier), so most stream values may differ by a step,
    2 * 2^-8 of the value, and so may the normalised values rounded from them.  A router logit
    sums 4,096 such terms of random sign: with s its standard deviation over the experts, it
    moves by 4 * 2^-8 / sqrt(3) * s = 0.009 s (one deviation).  The 4th of 12 (10th of 72)
    logits lies near 0.43 s (1.1 s), whose ulp is 0.0017 to 0.0034 s (0.0078 s): one
    deviation of the gap between two logits is up to sqrt(2) * 5.3 = 7.5 ulps, 16 is two."""
    cfg = GraniteConfig(experts=experts, top_k=top_k, **CFG)
    w = _weights(cfg, 3, gpu_device)
    eng = GraniteEngine(cfg, w, rows=rows, device=gpu_device, max_steps=64, split_len=16,
                        record_routes=True, experts="mx4")
    g = torch.Generator().manual_seed(20 + rows)
    prompts = [torch.randint(0, cfg.vocab, (3 + b % 3,), generator=g).tolist()
               for b in range(rows)]
    new = 4
    tokens, _, logits = eng.generate(prompts, new, record_logits=True)
    steps = max(len(p) for p in prompts) - 1 + new
    feed = feed_of(eng, prompts, steps)
    assert all(tokens[b] == feed[b][len(p):len(p) + new] for b, p in enumerate(prompts))
    orc = H.GraniteOracle(cfg, {k: v.cpu() for k, v in w.items()}, rows)
    orc.route_slack = 16.0
    check_steps(orc, lambda t, tok, r: orc.step(tok, routes=r), logits, eng.route_history, feed,
                prompts, 5e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(2, 7), (3, 60)])
def test_mx4_prefill_is_the_walk(gpu_device, rows, n):
    """After a prompt in passes the next steps' logits are those after walking it, within
    the bound of two orders of the same sums through three layers."""
    cfg = GraniteConfig(experts=12, top_k=4, **CFG)
    w = _weights(cfg, 7, gpu_device)
    eng = GraniteEngine(cfg, w, rows=rows, device=gpu_device, max_steps=n + 16, split_len=16,
                        experts="mx4")
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for _ in range(rows)]
    _, _, logits = eng.generate(prompts, 1, record_logits=True)
    eng.prefill(prompts)
    assert eng._prefiller is not None and eng._prefiller.mx4
    eng.replay()
    eng.check_errors()
    want, got = logits[n - 1], eng.logits.cpu()
    assert ((got - want).abs().amax(1) <= 5e-2 * want.abs().amax(1)).all()


def test_mx4_engine_refuses():
    with pytest.raises(ValueError, match="experts must be"):
        GraniteEngine(GraniteConfig(), {}, rows=1, experts="int4")
    for bad in (dict(moe_inter=48, shared_inter=96), dict(shared_inter=1000),
                dict(experts=512), dict(top_k=63, experts=100)):
        with pytest.raises(ValueError, match="4-bit experts"):
            mx4_shared(GraniteConfig(**bad))
    assert mx4_shared(GraniteConfig()) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("M,tile", [(9, 0), (24, 16), (100, 64), (400, 128)])
def test_mx4_moe_of_a_step_and_of_passes(gpu_device, M, tile):
    """The engine's routing and experts added into a stream, in each way that a call may run,
    against 64 bits from the engine's own fp8 weights, with the shared MLP as one."""
    from tests import _mx4_ref as R
    from tests.test_gpu_mx4 import _check_experts

    cfg = GraniteConfig(experts=12, top_k=4, layers=2, attention_layers=(1,), vocab=4096)
    w = _weights(cfg, 11, gpu_device)
    eng = GraniteEngine(cfg, w, rows=1, device=gpu_device, max_steps=32, graph=False,
                        experts="mx4")
    E, n, k, H, I = cfg.experts, eng.shared, eng.picks, cfg.hidden, cfg.moe_inter
    assert (n, k) == (2, 6)
    assert eng._lib.tfd_mx4_experts_tile_rows(M, k, E + n, H, I) == tile

    def f64(name, scale):
        return w[f"layer0.{name}"].view(torch.float8_e4m3fn).double() * \
            w[f"layer0.{scale}"].double().unsqueeze(1)

    gate_s, up_s = f64("w_shared_in", "w_shared_in_scale").split(n * I)
    down_s = f64("w_shared_out", "w_shared_out_scale")
    values = [torch.cat((f64("w_gate", "s_gate").view(E, I, H), gate_s.view(n, I, H))),
              torch.cat((f64("w_up", "s_up").view(E, I, H), up_s.view(n, I, H))),
              torch.cat((f64("w_down", "s_down").view(E, H, I),
                         torch.stack(down_s.split(I, dim=1))))]
    g = torch.Generator(device=gpu_device).manual_seed(M)

    def draw(*shape):
        return torch.randn(*shape, generator=g, device=gpu_device)

    x, logits, stream = draw(M, H).bfloat16(), draw(M, E), draw(M, H).bfloat16()
    before, weights = stream.clone(), torch.empty(M, k, device=gpu_device)
    ids = torch.empty(M, k, dtype=torch.int32, device=gpu_device)
    need = eng._lib.tfd_mx4_experts_work_bytes(M, k, E + n, H, I)
    work = torch.empty(need, dtype=torch.uint8, device=gpu_device)
    eng.mx4_moe(eng.layers[0], M, x, logits, weights, ids, stream, work, need, eng._stream())
    eng.check_errors()
    want_w, want_i = R.route(logits, None, k=cfg.top_k, score="softmax", shared=n)
    assert torch.equal(ids.cpu(), want_i)
    assert ((weights.cpu().double() - want_w).abs() <= want_w * 2.0 ** -23).all()
    _check_experts(stream, x, ids, weights, values, mult=cfg.residual_multiplier, start=before)
