"""TD3 with regularised critics on the GPU: the networks against their definition in 64 bits, eager and captured updates, and the training command."""
import json

import pytest
import torch

import reg_critic
from plen_ml_walk_amd import td3 as T

pytestmark = pytest.mark.gpu
KINDS = [(0.1, True), (0.01, False), (0.0, True)]


@pytest.mark.parametrize("dropout,norm", KINDS)
@pytest.mark.parametrize("B", [1, 33, 300])
def test_critic_against_its_definition(dropout, norm, B):
    reg_critic.check_against_definition("cuda", dropout, norm, B)


def _agent(dropout, norm):
    torch.manual_seed(5)
    return T.TD3Agent(26, 18, 1.0, critic_dropout=dropout, critic_norm=norm, data_parallel=False)


def _batch(n, seed=9):
    g = torch.Generator().manual_seed(seed)
    b = (torch.randn(n, 26, generator=g), torch.rand(n, 18, generator=g) * 2 - 1, torch.randn(n, 26, generator=g), torch.randn(n, 1, generator=g), torch.ones(n, 1))
    return tuple(t.cuda() for t in b), torch.randn(n, 18, generator=g).cuda()


@pytest.mark.parametrize("dropout,norm", KINDS + [(0.0, False)])
@pytest.mark.parametrize("B", [100, 257, 4096, 9000])
def test_captured_backward_equals_eager_at_every_replay(dropout, norm, B):
    """The critic's forward and backward captured once: each replay draws the masks of the calls counter as it stands and leaves the eager gradients (the same
    kernels on the same values; the library's products may sum in another order: 258 and B terms, 3 products deep, 2^-24 each, as in reg_critic)."""
    agent = _agent(dropout, norm)
    reseed = lambda k: agent.regularised and agent.seed_masks(11, 5 * k)  # noqa: E731
    batch, noise = _batch(B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            T.td3_critic_backward(agent, batch, noise)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = T.td3_critic_backward(agent, batch, noise)
    calls, seen = 1 if dropout > 0 else 0, []
    for k in range(4):
        reseed(k)
        loss = T.td3_critic_backward(agent, batch, noise)
        want = agent._critic_grads.flat.clone()
        reseed(k)
        agent._critic_grads.flat.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = agent._critic_grads.flat
        assert float((got - want).abs().max()) <= 1.1e-3 * float(want.abs().max()), k
        assert abs(float(loss) - float(captured)) <= 1e-5 * float(loss)              # a mean of B positive values, sums of at most 4096 + 64 terms in a tree
        assert not dropout or agent.critic.rng[1] == agent.critic_target.rng[1] == 5 * k + calls
        seen.append(want)
    assert (dropout > 0) != torch.equal(seen[0], seen[1])            # other masks, other gradients


@pytest.mark.parametrize("dropout,norm", KINDS)
@pytest.mark.parametrize("graphs,updates", [(0, 1), (1, 1), (1, 4)])
def test_trainers_run_regularised_critics(dropout, norm, graphs, updates):
    from plen_ml_walk_amd.train_vec import GraphedVecTD3Trainer, VecTD3Trainer
    from plen_ml_walk_amd.vec_env import PlenVecEnv
    n = 256
    env, agent, replay = PlenVecEnv(n, dtype=torch.float32), _agent(dropout, norm), T.ReplayBuffer(20000)
    before = [p.detach().clone() for p in agent.critic.parameters()]
    kw = dict(start_timesteps=512, batch_size=256, updates_per_step=updates, seed=0)
    tr = GraphedVecTD3Trainer(env, agent, replay, fused=False, **kw) if graphs else VecTD3Trainer(env, agent, replay, **kw)
    for _ in range(12):
        tr.step()
    torch.cuda.synchronize()
    its = 11 * updates
    assert tr.grad_steps == its and torch.isfinite(agent.last_critic_loss)
    assert all(torch.isfinite(p).all() and not torch.equal(p, q) for p, q in zip(agent.critic.parameters(), before))
    if dropout > 0:           # one pass over the critic per iteration and one more with every second; the target's one per iteration
        assert agent.critic.rng[1] == its + its // 2 and agent.critic_target.rng[1] == its
    env.close()


def test_fused_update_refuses_regularised_critics():
    from plen_ml_walk_amd.td3_fused import FusedTD3, PlenTd3Error
    with pytest.raises(PlenTd3Error, match="critic_dropout"):
        FusedTD3(_agent(0.1, True))


def test_training_command(tmp_path, capsys):
    from plen_ml_walk_amd import train_vec
    common = ["--envs", "256", "--steps", "6", "--warmup", "4", "--batch", "256", "--start-timesteps", "512", "--replay", "20000", "--critic-dropout", "0.01", "--critic-norm"]
    train_vec.main(common + ["--updates-per-step", "2", "--save", str(tmp_path / "run")])
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert line["critic_dropout"] == 0.01 and line["critic_norm"] and line["hip_graphs"] and line["critic_loss"] == line["critic_loss"]
    train_vec.main(common + ["--graphs", "0", "--resume", str(tmp_path / "run")])
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert not line["hip_graphs"] and line["critic_loss"] == line["critic_loss"]


@pytest.mark.parametrize("dropout,norm", [(0.1, True), (0.0, False)])
@pytest.mark.parametrize("B", [100, 9000])
def test_captured_policy_backward_equals_eager_at_every_replay(dropout, norm, B):
    agent = _agent(dropout, norm)
    reseed = lambda k: agent.regularised and agent.seed_masks(11, 5 * k)  # noqa: E731
    batch, _ = _batch(B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            T.td3_actor_backward(agent, batch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = T.td3_actor_backward(agent, batch)
    for k in range(4):
        reseed(k)
        loss = T.td3_actor_backward(agent, batch)
        want = agent._actor_grads.flat.clone()
        reseed(k)
        agent._actor_grads.flat.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert float((agent._actor_grads.flat - want).abs().max()) <= 1.1e-3 * float(want.abs().max()), k
        assert abs(float(loss) - float(captured)) <= 1e-4


@pytest.mark.parametrize("B,k,n", [(257, 26, 256), (4096, 256, 256), (4096, 256, 1), (9000, 44, 300)])
def test_captured_layers_keep_their_hooks_and_their_gradients(B, k, n):
    """One linear layer with a forward hook, forward and backward in a graph: the hook's work is part of it, and at every replay the gradients of weight and bias are their sums over the rows to the
    roundings of the kernel's order: a quarter of one of 8 chunks of rows added one after the other, then the quarters and the chunks; the product rounds once."""
    g = torch.Generator().manual_seed(B + n)
    layer = torch.nn.Linear(k, n).cuda()
    x, dy = torch.randn(B, k, generator=g).cuda(), torch.randn(B, n, generator=g).cuda()
    calls = []
    layer.register_forward_hook(lambda m, i, o: calls.append(m) or 2 * o)
    step = lambda: torch.autograd.grad(T._layer(layer, x), (layer.weight, layer.bias), dy)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    calls.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw, db = step()
    assert len(calls) == 1
    depth = -(-B // 8) // 4 + 16 + 4 + 8 + 2
    for replay in range(3):
        x.normal_(), dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        x64, d64 = x.cpu().double(), 2 * dy.cpu().double()
        for got, want, size in ((dw, d64.t() @ x64, d64.abs().t() @ x64.abs()), (db, d64.sum(0), d64.abs().sum(0))):
            assert bool(((got.cpu().double() - want).abs() <= depth * 2.0 ** -24 * size).all()), replay
        assert torch.isfinite(torch.randn(1 << 20, device="cuda").sum())              # the program's own work between replays
