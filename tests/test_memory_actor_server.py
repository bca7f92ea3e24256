"""The server of the reference's protocol with the memory actor inside, on the CPU."""
import pytest

from rlfluidcontrol_amd import learner_server, td3


def test_the_command_sets_the_window(monkeypatch):
    made = []

    class Server(learner_server.LearnerServer):
        def start_server(self):
            made.append(self)
            self.server.server_close()

    monkeypatch.setattr(learner_server, "LearnerServer", Server)
    for argv, window in ((["--window", "8"], 8), ([], 64)):
        learner_server.main(["--actor", "memory", "--max-grad-norm", "0.5", "--port", "0", "--device", "cpu"] + argv)
        agent = made.pop().agent
        assert agent.window == window and agent.max_grad_norm == 0.5 and isinstance(agent.main_actor, td3.MemoryActor)
    with pytest.raises(ValueError, match="window"):
        learner_server.LearnerServer(port=0, actor="memory", window=0)


def test_an_episode_through_the_server(tmp_path):
    s = learner_server.LearnerServer(port=0, actor="memory", window=4, max_grad_norm=1.0, seed=1, save_dir=str(tmp_path / "m"), data_dir=str(tmp_path / "d"))
    try:
        s.agent.bs = 4
        s._start_episode("")
        first = [s._request_deterministic_action("0.1_1.2") for _ in range(6)]
        assert len(set(first)) > 1  # the same observation at another time: the memory has moved on
        assert s._train(2) and s.agent.total_step_count == 2 and s._save()
        s._start_episode("")
        later = s._request_deterministic_action("0.1_1.2")
        assert s._init(s.agent.episode_count - 1)
        s._start_episode("")
        assert s._request_deterministic_action("0.1_1.2") == later  # the restored weights, from an empty memory
    finally:
        s.server.server_close()
