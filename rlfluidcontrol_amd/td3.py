"""TD3 learner next to the batched envs -- counterpart of the reference's
TF-1.x agent (`server/agent_TD3.py`, `server/utils.py`, `server/server.py:61-65,148-170`).

Same algorithm and constants; re-designed for the batched setting: every buffer is a device tensor,
a whole batch of envs is filtered / recorded / acted on per call, and nothing crosses to the host
inside the agent-step loop.  PyTorch is the plumbing here (autograd + Adam on 0.2 M parameters);
the hot path is the HIP environment.

Reference constants (agent_TD3.py:12-27): lr 1e-4 (Adam, TF defaults), gamma 0.99, tau 0.005,
batch 512, buffer 1e6, policy delay 2, exploration sigma 0.1, target smoothing sigma 0.2 clipped to
0.5, actor 2->256->256->2 (ReLU, ReLU, tanh), twin critics (2+2)->256->256->1, Glorot-uniform
kernels and zero biases (tf.layers.dense defaults).

Beside the reference's actor there is one with memory (`actor="memory"`): the agent sees two force coefficients of a wake, and
what it saw before tells more about the flow.  It reads the episode through a short causal convolution and a selective state
space scan (rlfluidcontrol_amd.ops) and is trained on windows of the replay; `max_grad_norm` clips either kind's gradients by
their global norm.
"""
import math

import torch
import torch.nn as nn

from . import ops

REWARD_ACTION_COST = math.pi * (1 / 8) * 0.0097 * (3.66 ** 3)  # server.py:64 (= 0.186756...)


def reward_func(next_state, action):
    """server.py:61-65: r = -Cd(next) - pi/8 * 0.0097 * 3.66^3 * sum |a|^3.
    next_state [...,2] = (Cl, Cd); action [...,A]."""
    return -next_state[..., 1] - REWARD_ACTION_COST * (action.abs() ** 3).sum(-1)


class KalmanFilter:
    """utils.py:3-23: scalar-gain filter applied to every observation component, one independent
    copy per env (the reference keeps one for its single env)."""

    def __init__(self, Q=0.25, R=11.0):
        self.Q, self.R = Q, R
        self.posteri = None
        self.posteri_error = 1.0

    def reset(self, mask=None):
        if mask is None or self.posteri is None:
            self.posteri = None
            self.posteri_error = 1.0
        else:  # per-env reset
            self.posteri = torch.where(mask[:, None], torch.zeros_like(self.posteri), self.posteri)
            self.posteri_error = torch.where(mask[:, None], torch.ones_like(self.posteri_error), self.posteri_error)

    def estimate(self, measurement=None):
        if measurement is not None:
            if self.posteri is None:
                self.posteri = torch.zeros_like(measurement)
                self.posteri_error = torch.ones_like(measurement)
            priori = self.posteri
            priori_error = self.posteri_error + self.Q
            K = priori_error / (priori_error + self.R)
            self.posteri = priori + K * (measurement - priori)
            self.posteri_error = (1 - K) * priori_error
        return self.posteri


class NoneFilter:
    """utils.py:26-37"""

    def __init__(self):
        self.posteri = None

    def reset(self, mask=None):
        if mask is None:
            self.posteri = None

    def estimate(self, measurement=None):
        if measurement is not None:
            self.posteri = measurement
        return self.posteri


class ProcessNoise:
    """Ornstein-Uhlenbeck exploration noise (utils.py:69-86): theta 1, sigma sqrt(2), ten Euler
    sub-steps of dt 0.01 per call.  `normal(shape)` supplies the N(0,1) draws (tests feed numpy's
    legacy stream to reproduce the reference's numbers)."""

    def __init__(self, dim, batch=1, device="cpu", dtype=torch.float64, normal=None, generator=None):
        self.x = torch.zeros(batch, dim, device=device, dtype=dtype)
        self.t, self.n = 0.1, 10
        self.dt = self.t / self.n
        self.theta, self.sigma = 1.0, math.sqrt(2.0)
        self._normal = normal
        self._gen = generator

    def _draw(self):
        if self._normal is not None:
            return torch.as_tensor(self._normal(tuple(self.x.shape)), dtype=self.x.dtype, device=self.x.device)
        return torch.randn(self.x.shape, device=self.x.device, dtype=self.x.dtype, generator=self._gen)

    def next(self):
        for _ in range(self.n):
            self.x = self.x - self.theta * self.x * self.dt + self.sigma * self._draw() * math.sqrt(self.dt)
        return self.x


class ReplayBuffer:
    """FIFO ring (utils.py:40-66) held on the device; `store` takes one transition or a batch."""

    def __init__(self, obs_dim, act_dim, size, device="cpu"):
        f = dict(dtype=torch.float32, device=device)
        self.obs1_buf = torch.zeros(size, obs_dim, **f)
        self.obs2_buf = torch.zeros(size, obs_dim, **f)
        self.acts_buf = torch.zeros(size, act_dim, **f)
        self.rews_buf = torch.zeros(size, 1, **f)
        self.done_buf = torch.zeros(size, 1, **f)
        self.ptr, self.size, self.max_size = 0, 0, size
        self.device = device

    def store(self, obs, act, rew, next_obs, done, pos=0):
        """`pos`: the transitions' place in their episode (WindowReplayBuffer keeps it)"""
        obs = torch.as_tensor(obs, dtype=torch.float32, device=self.device).reshape(-1, self.obs1_buf.shape[1])
        B = obs.shape[0]
        act = torch.as_tensor(act, dtype=torch.float32, device=self.device).reshape(B, -1)
        next_obs = torch.as_tensor(next_obs, dtype=torch.float32, device=self.device).reshape(B, -1)
        rew = torch.as_tensor(rew, dtype=torch.float32, device=self.device).reshape(-1).expand(B)
        done = torch.as_tensor(done, dtype=torch.float32, device=self.device).reshape(-1).expand(B)
        if B > self.max_size:  # only the newest max_size transitions survive, as with one-by-one stores
            raise ValueError("batch larger than the buffer")
        idx = (self.ptr + torch.arange(B, device=self.device)) % self.max_size
        self.obs1_buf[idx] = obs
        self.obs2_buf[idx] = next_obs
        self.acts_buf[idx] = act
        self.rews_buf[idx, 0] = rew
        self.done_buf[idx, 0] = done
        self.ptr = (self.ptr + B) % self.max_size
        self.size = min(self.size + B, self.max_size)

    def sample_batch(self, batch_size=32, generator=None):
        idxs = torch.randint(0, self.size, (batch_size,), device=self.device, generator=generator)
        return dict(obs1=self.obs1_buf[idxs], obs2=self.obs2_buf[idxs], acts=self.acts_buf[idxs],
                    rews=self.rews_buf[idxs], done=self.done_buf[idxs])

    def state_dict(self):
        n = self.size
        return dict(obs1=self.obs1_buf[:n].cpu(), obs2=self.obs2_buf[:n].cpu(), acts=self.acts_buf[:n].cpu(),
                    rews=self.rews_buf[:n].cpu(), done=self.done_buf[:n].cpu(), ptr=self.ptr, size=self.size,
                    max_size=self.max_size)

    def check_state_dict(self, sd):
        """raises if the checkpointed buffer cannot be restored into this one (nothing is modified)"""
        n = int(sd["size"])
        if n > self.max_size or n < 0:
            raise ValueError("replay buffer checkpoint holds %d transitions, this buffer %d at most" % (n, self.max_size))
        for key, buf in (("obs1", self.obs1_buf), ("obs2", self.obs2_buf), ("acts", self.acts_buf), ("rews", self.rews_buf),
                         ("done", self.done_buf)):
            if tuple(sd[key].shape) != (n,) + tuple(buf.shape[1:]):
                raise ValueError("replay buffer checkpoint: %s has shape %s, expected %s"
                                 % (key, tuple(sd[key].shape), (n,) + tuple(buf.shape[1:])))

    def load_state_dict(self, sd):
        """The reference restores by replacing the buffer object wholesale (server.py:192-198), so any pickled buffer
        restores there; here any checkpoint whose CONTENT fits is accepted, whatever capacity it was saved from: the
        saved transitions are the oldest-to-newest prefix and the write pointer follows them."""
        self.check_state_dict(sd)
        n = int(sd["size"])
        same = int(sd.get("max_size", self.max_size)) == self.max_size
        if same:
            order = torch.arange(n)
        else:  # a full buffer of another capacity is a ring: unroll it so that index 0 is the oldest transition
            old_max, ptr = int(sd.get("max_size", n)), int(sd["ptr"])
            order = (torch.arange(n) + (ptr if n == old_max else 0)) % max(n, 1)
        for name, key in (("obs1_buf", "obs1"), ("obs2_buf", "obs2"), ("acts_buf", "acts"), ("rews_buf", "rews"),
                          ("done_buf", "done")):
            getattr(self, name)[:n] = sd[key][order].to(self.device)
        self.size = n
        self.ptr = int(sd["ptr"]) % self.max_size if same else n % self.max_size


class WindowReplayBuffer(ReplayBuffer):
    """A replay ring for an actor with memory: every store holds one transition of each of `rows` envs, so that an env's next
    transition lies `rows` places on, and windows of consecutive transitions of one env and episode can be drawn."""

    def __init__(self, obs_dim, act_dim, size, rows, device="cpu"):
        super().__init__(obs_dim, act_dim, max(size // rows, 1) * rows, device=device)
        self.rows = rows
        self.pos_buf = torch.zeros(self.max_size, dtype=torch.int64, device=device)

    def store(self, obs, act, rew, next_obs, done, pos=0):
        at = self.ptr
        obs = torch.as_tensor(obs, dtype=torch.float32, device=self.device).reshape(-1, self.obs1_buf.shape[1])
        if obs.shape[0] != self.rows:
            raise ValueError("a store holds one transition of each of %d envs, not %d" % (self.rows, obs.shape[0]))
        super().store(obs, act, rew, next_obs, done)
        self.pos_buf[at:at + self.rows] = pos

    def sample_windows(self, batch_size, length, generator=None):
        """`batch_size` windows [batch, length, ...] that start at any stored transition and end with the episode, the newest
        transition or after `length`; `lengths` (int32) says where"""
        start = torch.randint(0, self.size, (batch_size,), device=self.device, generator=generator)
        newest = self.ptr - 1 - start
        newest = newest % self.max_size if self.size == self.max_size else newest
        k = torch.arange(length, device=self.device)
        at = (start[:, None] + k * self.rows) % self.max_size
        inside = (k <= torch.div(newest, self.rows, rounding_mode="floor")[:, None]) & (self.pos_buf[at] == self.pos_buf[start][:, None] + k)
        lengths = inside.long().cumprod(1).sum(1).to(torch.int32)
        return dict(obs1=self.obs1_buf[at], obs2=self.obs2_buf[at], acts=self.acts_buf[at], rews=self.rews_buf[at], done=self.done_buf[at], lengths=lengths)

    def state_dict(self):
        return dict(super().state_dict(), pos=self.pos_buf[:self.size].cpu(), rows=self.rows)

    def check_state_dict(self, sd):
        super().check_state_dict(sd)
        if int(sd.get("rows", 0)) != self.rows or tuple(sd["pos"].shape) != (int(sd["size"]),):
            raise ValueError("replay buffer checkpoint: transitions of %s envs side by side, expected %d" % (sd.get("rows"), self.rows))

    def load_state_dict(self, sd):
        super().load_state_dict(sd)
        n, old_max = self.size, int(sd["max_size"])
        order = torch.arange(n)
        if old_max != self.max_size and n == old_max:  # unrolled as the transitions are
            order = (order + int(sd["ptr"])) % max(n, 1)
        self.pos_buf[:n] = sd["pos"][order].to(self.device)


def _mlp(sizes, last):
    layers = []
    for i in range(len(sizes) - 1):
        lin = nn.Linear(sizes[i], sizes[i + 1])
        nn.init.xavier_uniform_(lin.weight)  # tf.layers.dense: glorot_uniform kernel, zero bias
        nn.init.zeros_(lin.bias)
        layers.append(lin)
        if i < len(sizes) - 2:
            layers.append(nn.ReLU())
    if last is not None:
        layers.append(last)
    return nn.Sequential(*layers)


class MemoryActor(nn.Module):
    """States of an episode -> actions, each from all states up to its own:

        (u, z) = W_in s     u = silu(causal convolution of u)     (d, B, C) = W_x u     y = scan(u, W_dt d, B, C) silu(z)
        a = tanh(MLP(y))

    `forward` takes whole windows [batch, length, state_dim] (with `lengths` of its own for each row), `step` one state of every
    env and the memory it advances, which is of a fixed size whatever has been read."""

    def __init__(self, state_dim, action_dim, width=256, state=16, taps=4):
        super().__init__()
        self.width, self.state, self.taps, self.rank = width, state, taps, max(1, width // 16)
        self.proj_in = nn.Linear(state_dim, 2 * width)
        self.conv_weight = nn.Parameter((2 * torch.rand(width, taps) - 1) / math.sqrt(taps))
        self.conv_bias = nn.Parameter(torch.zeros(width))
        self.proj_x = nn.Linear(width, self.rank + 2 * state, bias=False)
        self.proj_dt = nn.Linear(self.rank, width, bias=False)
        # decay rates 1 .. state for every channel; step sizes from 0.001 to 0.1 (dt_bias: the inverse of softplus at them)
        self.log_rate = nn.Parameter(torch.log(torch.arange(1, state + 1, dtype=torch.float32)).repeat(width, 1))
        dt = torch.exp(torch.rand(width) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.skip = nn.Parameter(torch.ones(width))
        self.head = _mlp([width, 256, action_dim], nn.Tanh())
        for lin in (self.proj_in, self.proj_x, self.proj_dt):
            nn.init.xavier_uniform_(lin.weight)
        nn.init.zeros_(self.proj_in.bias)

    def _split(self, u):
        d, B, C = self.proj_x(u).split([self.rank, self.state, self.state], -1)
        return self.proj_dt(d), B, C

    def forward(self, states, lengths=None):
        u, z = self.proj_in(states).chunk(2, -1)
        u = ops.causal_conv(u, self.conv_weight, self.conv_bias, silu=True, lengths=lengths)
        dt, B, C = self._split(u)
        y = ops.selective_scan(u, dt, -self.log_rate.exp(), B, C, D=self.skip, z=z, dt_bias=self.dt_bias, softplus=True, lengths=lengths)
        return self.head(y)

    def new_memory(self, rows):
        dev = self.skip.device
        return (torch.zeros(rows, self.taps - 1, self.width, device=dev), torch.zeros(rows, self.width, self.state, device=dev))

    @torch.no_grad()
    def step(self, states, memory):
        u, z = self.proj_in(states).chunk(2, -1)
        u = ops.causal_conv_step(u, memory[0], self.conv_weight, self.conv_bias, silu=True)
        dt, B, C = self._split(u)
        y = ops.selective_scan_step(u, dt, -self.log_rate.exp(), B, C, memory[1], D=self.skip, z=z, dt_bias=self.dt_bias, softplus=True)
        return self.head(y)


class Agent:
    """agent_TD3.py:10-184.  `get_action`, `train_iter`, `record`, `reset_agent`, `reset_episode`
    keep the reference's names and meaning; states/actions may carry any batch size."""

    # Transitions per env and episode of the reference's case (clientCFD.pde: 16-step windows from t = 1 to t = 50 at
    # dt = 0.0075: 408 requests, 407 transitions): what a rank's replay ring has to hold per env to cover one whole
    # episode -- the DEFAULT; a trainer on another time stepping passes steps_per_episode (train.py: the request count of
    # its episode_plan).
    STEPS_PER_EPISODE = 410

    def __init__(self, state_dim, action_dim, explore_noise="Gaussian", device="cpu", seed=None, num_envs=1, world=1,
                 replay_capacity=None, replay_episodes=3, steps_per_episode=None, actor="mlp", window=64, max_grad_norm=None):
        """actor: "mlp" (the reference's) or "memory" (MemoryActor: it acts on all states since reset_episode, one call of
        get_action after the other, and learns from windows of `window` transitions, as many as make up the batch size; a
        window starts with an empty memory).  max_grad_norm: the gradients of each update are clipped to this global norm."""
        if actor not in ("mlp", "memory"):
            raise ValueError("actor must be 'mlp' or 'memory', it is %r" % (actor,))
        if window < 1:
            raise ValueError("window must be 1 or more, it is %r" % (window,))
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise ValueError("max_grad_norm must be 0 or more, it is %r" % (max_grad_norm,))
        self.actor, self.window, self.max_grad_norm = actor, int(window), max_grad_norm
        self._memory = None
        self.world = world  # > 1: sharded learner (gradients averaged over the ranks, see _sync_grads)
        self.num_envs = num_envs
        self.n_grad_allreduce = 0
        self.lr, self.gamma, self.tau = 1e-4, 0.99, 0.005
        self.bs, self.bfs, self.d = 512, 1000000, 2
        self.explore_noise = explore_noise
        self.explore_noise_size = 0.1
        self.criticreg_noise_size, self.criticreg_noise_clip = 0.2, 0.5
        self.state_dim, self.action_dim = state_dim, action_dim
        self.device = torch.device(device)
        self.gen = torch.Generator(device=self.device)
        if seed is not None:
            self.gen.manual_seed(seed)
            torch.manual_seed(seed)
        self.process_noise_generator = ProcessNoise(action_dim, batch=num_envs, device=self.device, dtype=torch.float32,
                                                    generator=self.gen)
        if world > 1 and self.bs % world:
            raise ValueError("sharded learner: the batch size %d must be a multiple of the world size %d" % (self.bs, world))
        self._build()
        if world > 1:
            self._sync_from_rank0(seed)
        # Replay capacity PER RANK (a rank stores the transitions of its own envs only, time-major): the reference's
        # 1 M (agent_TD3.py:27) spans ~2400 single-env episodes; a batched rank writes num_envs transitions per agent
        # step, so the ring must hold whole episodes of ALL its envs or training never sees the early part of an
        # episode (1024 envs x 410 steps = 420 k per episode: a 1 M / world share would keep the last ~120 agent steps
        # only).  max(1 M, replay_episodes x num_envs x STEPS_PER_EPISODE) transitions of 32 bytes each.
        # (job-wide that is world x this -- against the reference's single 1 M FIFO: a sampling deviation of the batched
        # trainer, recorded as `replay_capacity` in train.py's episode log)
        local_envs = max(1, int(num_envs) // max(int(world), 1))  # (num_envs counts the envs of ALL ranks)
        self.steps_per_episode = int(steps_per_episode) if steps_per_episode else self.STEPS_PER_EPISODE
        self.replay_capacity = int(replay_capacity) if replay_capacity else max(
            self.bfs, int(replay_episodes) * local_envs * self.steps_per_episode)
        self._rows = local_envs
        self.replay_buffer = self._new_buffer()
        self.step_count = self.total_step_count = self.episode_count = self.train_count = 0

    def _new_buffer(self):
        if self.actor == "memory":
            return WindowReplayBuffer(self.state_dim, self.action_dim, self.replay_capacity, self._rows, device=self.device)
        return ReplayBuffer(self.state_dim, self.action_dim, self.replay_capacity, device=self.device)

    def _nets(self):
        return (self.main_actor, self.target_actor, self.main_critic_1, self.main_critic_2, self.target_critic_1,
                self.target_critic_2)

    def _sync_from_rank0(self, seed):
        """sharded learner: every rank must start from the same weights and the same generator state (the ranks average
        gradients onto THEIR weights and draw the same exploration / target noise).  With a process group up, rank 0's
        are broadcast -- seeded or not; without one, only an explicit seed can guarantee it."""
        import torch.distributed as dist
        if not (dist.is_available() and dist.is_initialized()):
            if seed is None:
                raise ValueError("Agent(world > 1) needs a seed or an initialised torch.distributed process group: "
                                 "ranks that start from different weights never converge to one model")
            return
        for net in self._nets():
            for p in net.parameters():
                dist.broadcast(p.data, 0)
        st = self.gen.get_state().to(self.device)
        dist.broadcast(st, 0)
        self.gen.set_state(st.cpu())

    def _build(self):
        s, a, dev = self.state_dim, self.action_dim, self.device
        self._memory = None
        new_actor = (lambda: MemoryActor(s, a)) if self.actor == "memory" else (lambda: _mlp([s, 256, 256, a], nn.Tanh()))
        self.main_actor = new_actor().to(dev)
        self.target_actor = new_actor().to(dev)
        self.main_critic_1 = _mlp([s + a, 256, 256, 1], None).to(dev)
        self.main_critic_2 = _mlp([s + a, 256, 256, 1], None).to(dev)
        self.target_critic_1 = _mlp([s + a, 256, 256, 1], None).to(dev)
        self.target_critic_2 = _mlp([s + a, 256, 256, 1], None).to(dev)
        self._pairs = [(self.target_critic_1, self.main_critic_1), (self.target_critic_2, self.main_critic_2),
                       (self.target_actor, self.main_actor)]
        for t, m in self._pairs:  # T_init
            t.load_state_dict(m.state_dict())
            for p in t.parameters():
                p.requires_grad_(False)
        critic_params = list(self.main_critic_1.parameters()) + list(self.main_critic_2.parameters())
        self._critic_params = critic_params
        self.Q_opt = torch.optim.Adam(critic_params, lr=self.lr, eps=1e-8)
        self.P_opt = torch.optim.Adam(self.main_actor.parameters(), lr=self.lr, eps=1e-8)

    # -- acting --
    @torch.no_grad()
    def get_action(self, state_data, stochastic=True):
        state = torch.as_tensor(state_data, dtype=torch.float32, device=self.device).reshape(-1, self.state_dim)
        if self.actor == "memory":
            if self._memory is None or self._memory[0].shape[0] != state.shape[0]:
                self._memory = self.main_actor.new_memory(state.shape[0])
            action = self.main_actor.step(state, self._memory)
        else:
            action = self.main_actor(state)
        if stochastic:
            if self.explore_noise == "Gaussian":
                noise = self.explore_noise_size * torch.randn(action.shape, device=self.device, generator=self.gen)
            elif self.explore_noise == "Process":
                if self.process_noise_generator.x.shape[0] != action.shape[0]:
                    self.process_noise_generator = ProcessNoise(self.action_dim, batch=action.shape[0], device=self.device,
                                                                dtype=torch.float32, generator=self.gen)
                noise = self.explore_noise_size * self.process_noise_generator.next()
            else:
                raise NotImplementedError
            action = torch.clamp(action + noise, -1, 1)
        return action

    # -- learning --
    def losses(self, batch):
        """(Q_loss, target y) of agent_TD3.py:36-48 for a batch dict."""
        with torch.no_grad():
            nxt = self.target_actor(batch["obs2"])
            noise = torch.clamp(self.criticreg_noise_size * torch.randn(nxt.shape, device=self.device, generator=self.gen),
                                -self.criticreg_noise_clip, self.criticreg_noise_clip)
            nxt = torch.clamp(nxt + noise, -1, 1)
            sa2 = torch.cat([batch["obs2"], nxt], 1)
            q_min = torch.minimum(self.target_critic_1(sa2), self.target_critic_2(sa2))
            y = batch["rews"] + self.gamma * (1 - batch["done"]) * q_min
        sa1 = torch.cat([batch["obs1"], batch["acts"]], 1)
        q_loss = ((self.main_critic_1(sa1) - y) ** 2).mean() + ((self.main_critic_2(sa1) - y) ** 2).mean()
        return q_loss, y

    def _window_target_actions(self, batch):
        """The target actor's actions in the next states of windows.  It reads a window's first state too, so that it has seen in
        state k + 1 what an actor that starts with the window has seen there (obs2[k] is obs1[k + 1])."""
        seen = torch.cat([batch["obs1"][:, :1], batch["obs2"]], 1)
        return self.target_actor(seen, batch["lengths"] + 1)[:, 1:]

    def window_losses(self, batch):
        """losses() over windows [batch, length, ...]; the mean runs over what lies within the windows"""
        lengths = batch["lengths"]
        keep = (torch.arange(batch["obs1"].shape[1], device=self.device) < lengths[:, None])[..., None]
        with torch.no_grad():
            nxt = self._window_target_actions(batch)
            noise = torch.clamp(self.criticreg_noise_size * torch.randn(nxt.shape, device=self.device, generator=self.gen),
                                -self.criticreg_noise_clip, self.criticreg_noise_clip)
            sa2 = torch.cat([batch["obs2"], torch.clamp(nxt + noise, -1, 1)], -1)
            q_min = torch.minimum(self.target_critic_1(sa2), self.target_critic_2(sa2))
            y = batch["rews"] + self.gamma * (1 - batch["done"]) * q_min
        sa1 = torch.cat([batch["obs1"], batch["acts"]], -1)
        off = (self.main_critic_1(sa1) - y) ** 2 + (self.main_critic_2(sa1) - y) ** 2
        return torch.where(keep, off, 0.0).sum() / keep.sum(), y

    def window_policy_loss(self, batch):
        lengths = batch["lengths"]
        keep = (torch.arange(batch["obs1"].shape[1], device=self.device) < lengths[:, None])[..., None]
        q = self.main_critic_1(torch.cat([batch["obs1"], self.main_actor(batch["obs1"], lengths)], -1))
        return -torch.where(keep, q, 0.0).sum() / keep.sum()

    def _clip_grads(self, params):
        """after _sync_grads: every rank clips the same averaged gradients by the same norm"""
        if self.max_grad_norm is not None:
            ops.clip_grad_norm([p.grad for p in params], self.max_grad_norm)

    def _sync_grads(self, params):
        """sharded learner: every rank holds the transitions of its own envs and a 1/world share of the batch; the
        gradients are averaged over the ranks (one all-reduce of the flattened gradients), so every rank applies the
        same update to the same weights"""
        if self.world <= 1:
            return
        import torch.distributed as dist
        params = [p for p in params if p.grad is not None]
        flat = torch.cat([p.grad.reshape(-1) for p in params])
        dist.all_reduce(flat)
        flat /= self.world
        o = 0
        for p in params:
            n = p.grad.numel()
            p.grad.copy_(flat[o:o + n].view_as(p.grad))
            o += n
        self.n_grad_allreduce += 1

    def train_iter(self):
        bs = self.bs // max(self.world, 1)  # this rank's share of the batch (bs is a multiple of world: __init__)
        if bs > self.replay_buffer.size:
            return
        if self.actor == "memory":
            batch = self.replay_buffer.sample_windows(max(1, bs // self.window), self.window, generator=self.gen)
            q_loss, _ = self.window_losses(batch)
        else:
            batch = self.replay_buffer.sample_batch(bs, generator=self.gen)
            q_loss, _ = self.losses(batch)
        self.Q_opt.zero_grad(set_to_none=True)
        q_loss.backward()
        self._sync_grads(self._critic_params)
        self._clip_grads(self._critic_params)
        self.Q_opt.step()
        if self.total_step_count % self.d == 0:
            if self.actor == "memory":
                p_loss = self.window_policy_loss(batch)
            else:
                p_loss = -self.main_critic_1(torch.cat([batch["obs1"], self.main_actor(batch["obs1"])], 1)).mean()
            self.P_opt.zero_grad(set_to_none=True)
            p_loss.backward()
            self._sync_grads(list(self.main_actor.parameters()))
            self._clip_grads(list(self.main_actor.parameters()))
            self.P_opt.step()
            with torch.no_grad():  # T_op
                for t, m in self._pairs:
                    for pt, pm in zip(t.parameters(), m.parameters()):
                        pt.mul_(1 - self.tau).add_(pm, alpha=self.tau)
        self.train_count += 1
        self.total_step_count += 1

    def record(self, this_state, this_action, this_reward, this_done, next_state):
        self.replay_buffer.store(obs=this_state, act=this_action, rew=this_reward, next_obs=next_state, done=this_done, pos=self.step_count)
        self.step_count += 1

    def reset_agent(self):
        self.replay_buffer = self._new_buffer()
        self.step_count = self.total_step_count = self.train_count = self.episode_count = 0
        self._build()
        if self.world > 1:
            self._sync_from_rank0(0)  # a fresh model on every rank: rank 0's where a process group is up

    def reset_episode(self):
        self._memory = None
        self.step_count = 0
        self.train_count = 0
        self.episode_count += 1

    # -- checkpoint (server.py:181-198 saves a TF checkpoint + the pickled buffer) --
    def state_dict(self):
        nets = {n: getattr(self, n).state_dict() for n in ("main_actor", "target_actor", "main_critic_1", "main_critic_2",
                                                           "target_critic_1", "target_critic_2")}
        return dict(nets=nets, Q_opt=self.Q_opt.state_dict(), P_opt=self.P_opt.state_dict(),
                    replay=self.replay_buffer.state_dict(), episode_count=self.episode_count,
                    total_step_count=self.total_step_count, actor=self.actor)

    def load_state_dict(self, sd):
        if sd.get("actor", "mlp") != self.actor:  # validate everything before the first mutation
            raise ValueError("checkpoint of a %r actor, this agent has a %r one" % (sd.get("actor", "mlp"), self.actor))
        self.replay_buffer.check_state_dict(sd["replay"])
        for n in sd["nets"]:
            if not hasattr(self, n):
                raise ValueError("checkpoint has an unknown network %r" % n)
        self._memory = None
        for n, s in sd["nets"].items():
            getattr(self, n).load_state_dict(s)
        self.Q_opt.load_state_dict(sd["Q_opt"])
        self.P_opt.load_state_dict(sd["P_opt"])
        self.replay_buffer.load_state_dict(sd["replay"])
        self.episode_count = sd["episode_count"]
        # total_step_count is NOT restored: in the reference it is a plain Python attribute outside the TF
        # checkpoint and the pickled buffer (server.py:192-198, agent_TD3.py:167-173), so a restored agent
        # restarts its policy-delay phase from 0; the saved value is kept in the file for information only


def assemble_transitions(state_record, action_record, action_dim):
    """server.py:157-165: consecutive recorded (filtered) states and actions of ONE episode become
    transitions (s_i, a_i[:action_dim], r_i, s_{i+1}, done = 0), i = 0 .. len-2.
    state_record [T, ..., 2], action_record [T, ..., A] (any batch dims in the middle)."""
    s = torch.as_tensor(state_record)
    a = torch.as_tensor(action_record)
    s1, s2, act = s[:-1], s[1:], a[:-1]
    r = reward_func(s2, act)
    return s1, act[..., :action_dim], r, s2, torch.zeros_like(r)


class BatchedLearner:
    """The reference's episode protocol (clientCFD.pde:35-85 + server.py) for E envs stepping together:
    act on the filtered obs of every env each agent step, keep the episode's records on the device,
    and at the end of the episode turn them into transitions and run `train_steps` TD3 iterations."""

    def __init__(self, num_envs, device="cpu", filter="None", explore_noise="Gaussian", one_action=False, seed=None,
                 shard=None, steps_per_episode=None, actor="mlp", window=64, max_grad_norm=None):
        """num_envs = ALL envs this learner acts for (every rank evaluates the same actor on the gathered obs).
        shard = (rank, world): the learner is sharded -- this rank stores the transitions of ITS envs only (the block
        [rank*E, (rank+1)*E) of the env axis) and trains on a 1/world share of every batch with averaged gradients.
        actor, window, max_grad_norm: see Agent."""
        self.E = num_envs
        self.rank, self.world = shard if shard is not None else (0, 1)
        self.one_action = one_action
        self.action_dim = 1 if one_action else 2
        self.agent = Agent(2, self.action_dim, explore_noise=explore_noise, device=device, seed=seed, num_envs=num_envs,
                           world=self.world, steps_per_episode=steps_per_episode, actor=actor, window=window, max_grad_norm=max_grad_norm)
        self.filter = KalmanFilter() if filter == "Kalman" else NoneFilter()
        self.state_record, self.action_record = [], []

    def start_episode(self):
        self.state_record, self.action_record = [], []
        self.agent.reset_episode()
        self.filter.reset()

    def request_action(self, obs, stochastic=True):
        """obs [E,2] = (Cl, Cd) -> action [E,2] in [-1,1]"""
        filtered = self.filter.estimate(obs)
        action = self.agent.get_action(filtered, stochastic=stochastic)
        if self.one_action:
            action = torch.cat([action, -action], 1)
        self.state_record.append(filtered.clone())
        self.action_record.append(action.clone())
        return action

    def train(self, steps):
        if len(self.state_record) >= 2:
            s1, act, r, s2, done = assemble_transitions(torch.stack(self.state_record), torch.stack(self.action_record),
                                                        self.action_dim)
            if self.world > 1:  # this rank keeps its own envs' transitions
                per = self.E // self.world
                sl = slice(self.rank * per, (self.rank + 1) * per)
                s1, act, r, s2, done = s1[:, sl], act[:, sl], r[:, sl], s2[:, sl], done[:, sl]
            # time-major records -> one store per agent step keeps the reference's FIFO order per env
            for t in range(s1.shape[0]):
                self.agent.replay_buffer.store(s1[t], act[t], r[t], s2[t], done[t], pos=t)
        for _ in range(steps):
            self.agent.train_iter()
