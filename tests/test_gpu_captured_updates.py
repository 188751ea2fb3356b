"""Captured updates: what a graph holds, and that its replays are the eager step whatever runs between them."""
import collections
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def _nodes(graph):
    """counts of the graph's nodes by kind (the runtime that torch has loaded)"""
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    raw, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert hip.hipGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    kinds = collections.Counter()
    for node in nodes:
        kind = ctypes.c_int()
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        kinds[{0: "kernel", 1: "memcpy", 2: "memset"}.get(kind.value, kind.value)] += 1
    return kinds


@pytest.fixture
def kept_graphs(monkeypatch):
    """torch.cuda.CUDAGraph that keeps its nodes"""
    plain = torch.cuda.CUDAGraph
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: plain(keep_graph=True))


def _learner(name, minibatch, trunk, bits, fused, graph):
    from marl_amd import agents
    from marl_amd.policy import Agent
    from marl_amd.rollout_buffer import Buffer
    from marl_amd.spaces import Box, Discrete

    class Env:
        single_observation_space = Box(-1, 1, (101,))

    E, A = 16, 2
    T = minibatch * 2 // (E * A)
    torch.manual_seed(3)
    net = Agent(Box(-1, 1, (101,)), Discrete(7), A, E, build_centralised=name == "CMAPPO").cuda()
    if trunk != "float32":
        net.use_mxfp4_trunk(straight_through=trunk == "straight")
    if bits == 8:
        net.use_activation_checkpoints()
    buf = Buffer(101, A, E, max_size=T, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, E * A, 101, device="cuda", generator=g)
    buf.obs_buff.copy_((x.abs() > 0.9).float() * (x * 1.3).round())
    buf.actions_buff.copy_(torch.randint(0, 7, (T, E * A), device="cuda", generator=g).float())
    buf.rewards_buff.copy_(torch.randn(T, E * A, device="cuda", generator=g))
    buf.logprobs_buff.fill_(-1.9459)
    opt = torch.optim.Adam(net.parameters(), lr=1e-3, fused=True)
    learner = getattr(agents, name)(Env, opt, net, buf, (101,), 7, batch_size=T * E * A, num_mini_batches=2, num_agents=A, ppo_epoch=1,
                                    graph_update="on" if graph else "off", fused_loss=fused)
    return learner, net, x[0].contiguous()


@pytest.mark.parametrize("name", ["MAPPO", "CMAPPO"])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("trunk,bits", [("float32", 32), ("mxfp4", 32), ("float32", 8), ("mxfp4", 8), ("straight", 32), ("straight", 8)])
@pytest.mark.parametrize("minibatch", [512, 2048, 65536])
def test_no_memory_set_nodes(kept_graphs, name, fused, trunk, bits, minibatch):
    learner, _, obs = _learner(name, minibatch, trunk, bits, fused, True)
    for _ in range(2):
        learner.update(obs)
    kinds = _nodes(learner._g["graph"])
    assert kinds["kernel"] > 10 and kinds["memset"] == 0, kinds


def test_a_captured_mean_of_many_targets(kept_graphs):
    learner, _, obs = _learner("CMAPPO", 131072, "float32", 8, True, True)
    for _ in range(2):
        learner.update(obs)
    assert _nodes(learner._g["graph"])["memset"] == 0
    learner, _, obs = _learner("CMAPPO", 131072, "float32", 8, False, True)
    for _ in range(2):
        learner.update(obs)
    assert learner._g is None  # the autograd loss has means over more values than one block takes


@pytest.mark.parametrize("flags", [[], ["--sampler", "torch"], ["--algorithm", "cmappo"], ["--algorithm", "cmappo", "--sampler", "torch"],
                                   ["--env-shards", "2"], ["--trunk-precision", "mxfp4"], ["--trunk-precision", "mxfp4", "--algorithm", "cmappo"],
                                   ["--fused-loss", "off"], ["--adam", "foreach"]])
def test_no_memory_set_nodes_in_training(tmp_path, monkeypatch, flags):
    """every graph that the command captures, rollouts and updates"""
    from marl_amd import train

    plain, made = torch.cuda.CUDAGraph, []
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: (made.append(plain(keep_graph=True)), made[-1])[1])
    E, A, T = 64, 2, 64
    train.main(["--num-agents", str(A), "--num-envs", str(E), "--layout", "overcooked_cramped_room_v0", "--num-steps", str(T), "--num-minibatches", "4",
                "--total-steps", str(E * A * T * 3), "--ppo-epoch", "1", "--max-steps", "50", "--data-path", str(tmp_path), "--seed", "3",
                "--graph-rollout", "on", "--graph-update", "on"] + flags)
    assert len(made) >= 2
    for graph in made:
        kinds = _nodes(graph)
        assert kinds["kernel"] > 0 and kinds["memset"] == 0, kinds


@pytest.mark.parametrize("trunk,bits", [("float32", 32), ("mxfp4", 32), ("mxfp4", 8), ("straight", 32), ("straight", 8)])
def test_replays_between_eager_work_are_the_eager_steps(trunk, bits):
    got = []
    for graph in (False, True):
        learner, net, obs = _learner("MAPPO", 2048, trunk, bits, True, graph)
        torch.manual_seed(11)
        for k in range(12):
            learner.update(obs)
            if k % 3 == 0:
                torch.cuda.synchronize()
            with torch.no_grad():  # the program's own work, library sums among it
                for n in (1, 7, 40):
                    net.get_value(obs[:n])
                    torch.full((4096 * n, 256), float(k), device="cuda").sum(0)
        got.append([p.detach().clone() for p in net.parameters()])
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (32, 512), (257, 255), (2048, 512), (2048, 1), (65536, 7), (5, 1031), (100003, 33), (9, 4099), (70000, 256)])
def test_column_sums(rows, cols, dtype):
    """Off 64 bits by the roundings of a thread's own rows, never more than the rows, of the workgroup's sum and of the result,
    half a step each.  Independent roundings grow as the root of their number, of which a thread has at most 17 here: over all
    columns they stay below five half steps of the sums of magnitudes."""
    from marl_amd import _lib, act8
    from marl_amd.mxfp4 import _TYPES, _p

    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    want, size = x.double().sum(0), x.double().abs().sum(0)
    for view in (x, x.t().contiguous().t(), torch.cat([x, x], 1)[:, :cols]):
        got = act8.column_sums(view)
        assert got.dtype == torch.float32 and torch.equal(got, act8.column_sums(x))
    assert ((got.double() - want).abs() <= (rows + 2) * 2.0 ** -24 * size).all()
    assert (got.double() - want).norm() <= 5 * 2.0 ** -24 * size.norm()
    L = _lib.lib()
    need = L.marl_column_sums_workspace_bytes(rows, cols)
    out, work = torch.full((cols + 128,), 7.0, device="cuda"), torch.full((need + 64,), 9, dtype=torch.uint8, device="cuda")
    _lib.check(L.marl_column_sums(_p(x), _TYPES[dtype], rows, cols, _p(out[64:]), _p(work), torch.cuda.current_stream().cuda_stream), "marl_column_sums")
    assert torch.equal(out[64:-64], got) and (out[:64] == 7).all() and (out[-64:] == 7).all() and (work[need:] == 9).all()


def test_column_sums_of_infinities_nans_and_nothing():
    from marl_amd import act8

    x = torch.ones(3000, 70, device="cuda")
    x[5, 3], x[2999, 4], x[7, 69], x[8, 69] = float("nan"), float("inf"), float("inf"), -float("inf")
    got = act8.column_sums(x)
    assert torch.isnan(got[[3, 69]]).all() and got[4] == float("inf")
    keep = [c for c in range(70) if c not in (3, 4, 69)]
    assert (got[keep] == 3000).all()
    assert not act8.column_sums(x[:0]).any() and act8.column_sums(x[:0]).shape == (70,)
    for bad in (x.cpu(), x.double(), x[0], x[:, :0]):
        with pytest.raises(ValueError):
            act8.column_sums(bad)


def test_column_sums_beyond_32_bits():
    from marl_amd import act8

    rows = (1 << 32) // 512 + 5
    x = torch.zeros(rows, 512, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.arange(512, device="cuda").bfloat16()
    assert torch.equal(act8.column_sums(x), 3 * torch.arange(512, device="cuda").bfloat16().float())


def test_column_sums_on_streams_and_from_a_graph():
    from marl_amd import act8

    x = torch.randn(70000, 256, device="cuda")
    want = act8.column_sums(x)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for stream in streams * 3:
        with torch.cuda.stream(stream):
            got.append(act8.column_sums(x))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        out = act8.column_sums(x)
    for k in range(4):
        x.normal_()
        want = act8.column_sums(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
