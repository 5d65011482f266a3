"""Worker for tests/test_regularised_td3_cpu.py: TD3 with regularised critics on two ranks over gloo."""
import json
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from plen_ml_walk_amd import td3 as T          # noqa: E402


def main():
    dist.init_process_group("gloo")
    rank, world = dist.get_rank(), dist.get_world_size()
    torch.manual_seed(40 + rank)                # different initialisations: the constructor broadcasts rank 0's, the norms' among them
    agent = T.TD3Agent(26, 18, 1.0, device="cpu", critic_dropout=0.1, critic_norm=True)
    everything = lambda: torch.cat([p.detach().reshape(-1) for p in list(agent.actor.parameters()) + list(agent.critic.parameters())])  # noqa: E731
    start = everything().clone()
    buf = T.ReplayBuffer(100, device="cpu")
    buf.add_batch(torch.randn(40, 26), torch.rand(40, 18) * 2 - 1, torch.randn(40, 26), torch.randn(40), torch.zeros(40))
    T.td3_critic_backward(agent, buf.sample(32))
    own = agent._critic_grads.flat.clone()
    agent._critic_grads.all_reduce_mean()
    all_own = [torch.zeros_like(own) for _ in range(world)]
    dist.all_gather(all_own, own)
    off = (agent._critic_grads.flat.double() - sum(g.double() for g in all_own) / world).abs().max()
    for _ in range(4):
        agent.train(buf, 32)
    flat = everything()
    gathered = [torch.zeros_like(flat) for _ in range(world)]
    dist.all_gather(gathered, flat)
    res = {"same_across_ranks": all(torch.equal(gathered[0], g) for g in gathered), "moved": float((flat - start).abs().max()), "mean_gradient_off": float(off),
           "gradient": float(own.abs().max()), "seeds": [int(agent.critic.rng[0]), int(agent.critic_target.rng[0])]}
    with open("%s.rank%d.json" % (sys.argv[1], rank), "w") as f:
        json.dump(res, f)
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
