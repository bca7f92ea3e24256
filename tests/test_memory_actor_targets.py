"""The targets that a memory actor learns from are those of the policy that acts, on the CPU."""
import torch

from rlfluidcontrol_amd import td3


def agent_with_an_episode(steps=12, rows=3, window=8):
    ag = td3.Agent(2, 2, seed=5, num_envs=rows, replay_capacity=1000, actor="memory", window=window)
    ag.criticreg_noise_size = 0.0
    with torch.no_grad():  # a target of its own, as after some updates
        for p in ag.target_actor.parameters():
            p.add_(0.1 * torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())))
    g = torch.Generator().manual_seed(6)
    states = torch.randn(steps + 1, rows, 2, generator=g)
    for t in range(steps):
        ag.replay_buffer.store(states[t], torch.rand(rows, 2, generator=g) * 2 - 1, torch.randn(rows, generator=g), states[t + 1], torch.zeros(rows), pos=t)
    return ag, states


def test_target_actions_are_those_of_the_acting_policy():
    ag, states = agent_with_an_episode()
    b = ag.replay_buffer.sample_windows(200, 8, generator=ag.gen)
    seen = []
    critic = ag.target_critic_1
    ag.target_critic_1 = lambda sa: (seen.append(sa[..., 2:]), critic(sa))[1]
    ag.window_losses(b)
    memory = ag.target_actor.new_memory(3)
    acts = torch.stack([ag.target_actor.step(states[t], memory) for t in range(13)])  # [time, env, action] from the episode's start
    starts = 0
    for k in range(200):
        for env in range(3):
            if torch.equal(b["obs1"][k, 0], states[0, env]):  # a window at the episode's start: both have read the same states
                n = int(b["lengths"][k])
                assert n == 8
                # 32 bits on both sides: sums over 256 values, nine positions
                assert torch.allclose(seen[0][k, :n], acts[1:n + 1, env], atol=2e-5, rtol=0)
                starts += 1
    assert starts


def test_a_target_has_read_what_the_actor_has_in_the_same_state():
    ag, _ = agent_with_an_episode()
    ag.target_actor.load_state_dict(ag.main_actor.state_dict())
    b = ag.replay_buffer.sample_windows(50, 8, generator=ag.gen)
    with torch.no_grad():
        now, then = ag.main_actor(b["obs1"], b["lengths"]), ag._window_target_actions(b)
    for k in range(50):
        n = int(b["lengths"][k])
        assert torch.allclose(then[k, :n - 1], now[k, 1:n], atol=2e-5, rtol=0)
