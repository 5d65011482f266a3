"""TD3 with regularised critics on the CPU: the networks against their definition, the agent around them, and the data-parallel step over gloo."""
import json
import os
import subprocess
import sys

import pytest
import torch

import reg_critic
from test_distributed_cpu import ROOT, _free_port
from plen_ml_walk_amd import td3 as T

KINDS = [(0.1, True), (0.01, False), (0.0, True)]


@pytest.mark.parametrize("dropout,norm", KINDS)
@pytest.mark.parametrize("B", [1, 33])
def test_critic_against_its_definition(dropout, norm, B):
    reg_critic.check_against_definition("cpu", dropout, norm, B)


def _agent(dropout=0.1, norm=True, **kw):
    torch.manual_seed(5)
    return T.TD3Agent(26, 18, 1.0, device="cpu", critic_dropout=dropout, critic_norm=norm, **kw)


def _buffer(n=64):
    g = torch.Generator().manual_seed(9)
    buf = T.ReplayBuffer(200, device="cpu")
    buf.add_batch(torch.randn(n, 26, generator=g), torch.rand(n, 18, generator=g) * 2 - 1, torch.randn(n, 26, generator=g), torch.randn(n, generator=g), torch.zeros(n))
    return buf


def test_plain_agents_are_as_they_were():
    agent = T.TD3Agent(26, 18, 1.0, device="cpu")
    assert type(agent.critic) is T.Critic and not agent.regularised
    assert list(agent.critic.state_dict()) == ["fc%d.%s" % (k, w) for k in range(1, 7) for w in ("weight", "bias")]
    only_dropout = _agent(0.1, False)
    assert list(only_dropout.critic.state_dict()) == list(agent.critic.state_dict())          # dropout has no parameters: checkpoints go both ways
    only_dropout.critic.load_state_dict(agent.critic.state_dict())


@pytest.mark.parametrize("dropout,norm", KINDS)
def test_flat_buffers_hold_every_parameter_once(dropout, norm):
    agent = _agent(dropout, norm)
    for net, flat in ((agent.critic, agent._critic_flat.flat), (agent.critic_target, agent._critic_target_flat.flat)):
        assert flat.numel() == sum(p.numel() for p in net.parameters())
        lo, hi = flat.data_ptr(), flat.data_ptr() + 4 * flat.numel()
        spans = sorted((p.data_ptr(), p.data_ptr() + 4 * p.numel()) for p in net.parameters())
        assert spans[0][0] == lo and spans[-1][1] == hi and all(a[1] == b[0] for a, b in zip(spans, spans[1:]))
        assert torch.equal(agent._critic_flat.views["W14"], torch.cat((agent.critic.fc1.weight, agent.critic.fc4.weight)))
    assert sum(p.grad.numel() for p in agent.critic.parameters()) == agent._critic_grads.flat.numel()


@pytest.mark.parametrize("dropout,norm", KINDS)
def test_training_moves_every_parameter_and_draws_new_masks(dropout, norm):
    agent, buf = _agent(dropout, norm), _buffer()
    assert agent.critic.rng.tolist() != agent.critic_target.rng.tolist() and agent._fused_for(buf) is None
    before = [p.detach().clone() for p in agent.critic.parameters()]
    for _ in range(4):
        agent.train(buf, 32)
    assert all(not torch.equal(a, b) for a, b in zip(before, agent.critic.parameters())) and torch.isfinite(agent.last_critic_loss)
    drawn = 1 if dropout > 0 else 0
    assert agent.critic.rng[1] == 6 * drawn and agent.critic_target.rng[1] == 4 * drawn        # four critic passes and two policy passes; four targets


def test_refusals():
    for bad in (-0.1, 1.0, float("nan"), 7):
        with pytest.raises(ValueError, match="dropout"):
            T.TD3Agent(26, 18, 1.0, device="cpu", critic_dropout=bad)
    agent = _agent()
    plain = T.TD3Agent(26, 18, 1.0, device="cpu")
    with pytest.raises(RuntimeError, match="norm1"):
        agent.critic.load_state_dict(plain.critic.state_dict())
    from plen_ml_walk_amd import td3_fused
    agent.device = torch.device("cuda", 0)                # (the check lies before anything touches a device)
    with pytest.raises(td3_fused.PlenTd3Error, match="critic_dropout"):
        td3_fused.FusedTD3(agent)


def test_train_vec_refuses_what_it_cannot_run(capsys):
    from plen_ml_walk_amd import train_vec
    for argv, text in ((["--critic-norm", "--schedule", "pipelined"], "--schedule sync"), (["--critic-dropout", "1.5"], "[0, 1)"), (["--critic-dropout", "nan"], "[0, 1)")):
        with pytest.raises(SystemExit):
            train_vec.main(argv)
        assert text in capsys.readouterr().err


def test_checkpoint_goes_on_with_masks_not_drawn_before(tmp_path):
    from plen_ml_walk_amd.train_vec import resume_training, save_training
    agent, buf = _agent(), _buffer()
    for _ in range(5):
        agent.train(buf, 16)

    class Counters(object):
        env_steps, grad_steps = 50, 5
    save_training(agent, Counters, str(tmp_path / "run"))
    other = _agent()
    resume_training(other, buf, str(tmp_path / "run"))
    for a, b in ((agent.critic, other.critic), (agent.critic_target, other.critic_target)):
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
        assert b.rng[0] == a.rng[0] and b.rng[1] == 10 >= a.rng[1]
    other.train(buf, 16)
    assert torch.isfinite(other.last_critic_loss)


@pytest.mark.parametrize("dropout,norm", KINDS + [(0.0, False)])
def test_the_evaluation_command_loads_every_kind_of_checkpoint(tmp_path, dropout, norm):
    from plen_ml_walk_amd.walk_eval import load_policy
    agent = _agent(dropout, norm)
    agent.save(str(tmp_path / "run"))
    policy, state = load_policy(str(tmp_path / "run"), device="cpu"), torch.randn(5, 26)
    assert torch.equal(policy.select_action_batch(state), agent.select_action_batch(state))


def test_two_ranks_share_gradients_and_draw_their_own_masks(tmp_path):
    out = str(tmp_path / "reg")
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1", "--master-port", str(_free_port()),
           os.path.join(ROOT, "tests", "dist_reg_worker.py"), out]
    subprocess.run(cmd, check=True, timeout=180, env=dict(os.environ, OMP_NUM_THREADS="1"), cwd=ROOT)
    a, b = (json.load(open("%s.rank%d.json" % (out, r))) for r in range(2))
    assert a["same_across_ranks"] and b["same_across_ranks"] and a["moved"] > 1e-5
    seeds = a["seeds"] + b["seeds"]
    assert len(set(seeds)) == 4
    assert a["mean_gradient_off"] <= 1e-6 * a["gradient"] + 1e-9          # the bucket is the mean of the two ranks' own gradients: two roundings of 2^-24


@pytest.mark.parametrize("regularised", [False, True])
def test_hooks_and_replaced_forwards_run_while_capturing(monkeypatch, regularised):
    """A captured step calls the linear modules as an eager one does (here: the forward passes with the capture's switch on; gradients on the device in the GPU tests)."""
    agent = _agent() if regularised else T.TD3Agent(26, 18, 1.0, device="cpu")
    agent.critic.eval()
    state, action, seen = torch.randn(300, 26), torch.rand(300, 18), []
    modules = [agent.actor.fc1, agent.actor.fc3, agent.critic.fc2, agent.critic.fc6]
    handles = [m.register_forward_hook(lambda m, i, o: seen.append(m) or 2 * o) for m in modules]
    handles.append(agent.actor.fc2.register_forward_pre_hook(lambda m, i: seen.append(m)))
    agent.critic.fc5.forward = lambda x: seen.append(agent.critic.fc5) or torch.nn.functional.linear(x, agent.critic.fc5.weight + 1, agent.critic.fc5.bias)
    run = lambda: (agent.actor(state),) + tuple(agent.critic(state, action)) + (agent.critic.Q1(state, action),)  # noqa: E731
    want, eager = run(), list(seen)
    assert all(m in eager for m in modules + [agent.actor.fc2, agent.critic.fc5])
    seen.clear()
    monkeypatch.setattr(T, "_capturing", lambda x: True)
    got = run()
    assert seen == eager
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for h in handles:
        h.remove()
    assert "forward" not in vars(agent.actor.fc1)
    bare = torch.nn.Linear(26, 5, bias=False)                   # a layer without a bias
    (g,) = torch.autograd.grad(T._layer(bare, state).sum(), bare.weight)
    assert torch.equal(g, torch.autograd.grad(bare(state).sum(), bare.weight)[0])


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_critics_do_not_get_other_masks(reentrant):
    """Activation checkpointing runs the forward pass again inside the backward pass, when the mask stream has moved on: other masks, and wrong gradients.  It is an error; without dropout it works."""
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator().manual_seed(1)
    state, action = torch.randn(20, 26, generator=g), torch.rand(20, 18, generator=g).requires_grad_()
    for run in (lambda c: checkpoint(lambda s, a: sum(c(s, a)), state, action, use_reentrant=reentrant), lambda c: checkpoint(c.Q1, state, action, use_reentrant=reentrant)):
        critic = _agent(0.3, True).critic
        with pytest.raises(RuntimeError, match="mask"):
            run(critic).sum().backward()
        plain = _agent(0.0, True).critic
        critic.eval()
        for p in list(critic.parameters()) + list(plain.parameters()):
            p.grad = None
        run(plain).sum().backward()
        run(critic).sum().backward()
        for p, q in zip(critic.parameters(), plain.parameters()):
            assert (p.grad is None) == (q.grad is None) and (p.grad is None or torch.equal(p.grad, q.grad))


def test_dropout_that_its_steps_round_away_is_refused():
    """The masks hold p in steps of 2^-16: what would drop nothing, or everything, is no regularisation."""
    for bad in (1e-6, 2.0 ** -17, 1 - 2.0 ** -17, 1 - 1e-7, 0.9999999):
        with pytest.raises(ValueError, match="dropout"):
            T.TD3Agent(26, 18, 1.0, device="cpu", critic_dropout=bad)
        with pytest.raises(ValueError, match="dropout"):
            T.RegularisedCritic(26, 18, bad, True)
    for good in (2.0 ** -16, 1 - 2.0 ** -16, 0.0):
        assert T.RegularisedCritic(26, 18, good, True).dropout == good


def test_train_vec_refuses_dropout_that_its_steps_round_away(capsys):
    from plen_ml_walk_amd import train_vec
    for bad in ("1e-6", "0.999999"):
        with pytest.raises(SystemExit):
            train_vec.main(["--critic-dropout", bad])
        assert "2^-16" in capsys.readouterr().err
