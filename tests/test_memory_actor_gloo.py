"""The sharded learner with a memory actor and clipped gradients on CPU: two gloo ranks, stub envs.  A rank stores and samples
windows of its own envs only; every rank clips the same averaged gradients, so the weights stay bit-identical."""
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from rlfluidcontrol_amd import td3
from rlfluidcontrol_amd.train import run_episode
from rlfluidcontrol_amd.vec_env import ShardedVecEnv
from tests.test_train_sharded_gloo import StubBackend

WORLD, E, T, LIMIT = 2, 6, 9, 1e-3


def _worker(rank, port, q):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    torch.set_num_threads(2)
    dist.init_process_group("gloo", rank=rank, world_size=WORLD)
    try:
        torch.manual_seed(0)
        vec = ShardedVecEnv(StubBackend(rank, E, T + 1), E)
        learner = td3.BatchedLearner(WORLD * E, device="cpu", seed=3, shard=(rank, WORLD), actor="memory", window=4, max_grad_norm=LIMIT)
        learner.agent.bs = 32
        run_episode(vec, learner, plan=(T + 1, T))
        agent, norms = learner.agent, []
        clip = agent._clip_grads

        def clipped(params):  # (looked at here: the actor's loss adds to the critics' gradients after their own step)
            clip(params)
            norms.append(float(torch.stack([p.grad.double().square().sum() for p in params]).sum().sqrt()))

        agent._clip_grads = clipped
        learner.train(3)
        nets = (agent.main_actor, agent.main_critic_1, agent.main_critic_2, agent.target_actor)
        flat = torch.cat([p.detach().reshape(-1) for net in nets for p in net.parameters()])
        both = [torch.zeros_like(flat) for _ in range(WORLD)]
        dist.all_gather(both, flat)
        q.put((rank, bool(torch.equal(both[0], both[1])), bool(torch.isfinite(flat).all()), norms, agent.replay_buffer.rows, agent.replay_buffer.size))
    finally:
        dist.destroy_process_group()


def test_two_ranks_keep_the_same_weights():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, port, q)) for r in range(WORLD)]
    for p in procs:
        p.start()
    res = sorted(q.get(timeout=120) for _ in range(WORLD))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for rank, same, finite, norms, rows, size in res:
        assert len(norms) == 5  # three updates of the critics, the actor with the first and the third
        assert norms == res[0][3]
        assert same and finite and rows == E and size == E * (T - 1)
        # scaled to the limit, less the 1e-6 of the formula beside a norm of more than the limit
        # (each of the three float32 roundings of a scaled element is at most half a step: the factor, the product, the stored value)
        for norm in norms:
            assert norm <= LIMIT * (1 + 3 * 2 ** -24) and norm >= LIMIT * (1 - 1e-3 - 3 * 2 ** -24)
