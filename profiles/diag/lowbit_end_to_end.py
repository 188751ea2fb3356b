#!/usr/bin/env python3
"""A rollout step (policy, sampling, env) at 65,536 two-agent kitchens with the trunk in float32 and in 4 bits, the policy's part of
it for few kitchens, and forward and backward of an update's minibatch with float32 and with 8-bit activations (time, and the peak of allocated memory)."""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
from marl_amd.env import make_env, make_vector_env  # noqa: E402
from marl_amd.policy import Agent  # noqa: E402


# "straight": the backward pass that reads the rounded operands, as `train` takes it
TRUNKS = (("float32", 32), ("float32", 8), ("mxfp4", 8), ("mxfp4 straight", 32), ("mxfp4 straight", 8))


def us(f, n):
    for _ in range(5):
        f()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(n):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / n * 1e6


def main():
    dev, E = torch.device("cuda:0"), 65536
    vec = make_vector_env(E, make_env(2, "overcooked_cramped_room_v0", "global_obs"), device=dev)
    torch.manual_seed(0)
    net = Agent(vec.single_observation_space, vec.single_action_space, 2, 1, build_centralised=False).to(dev).use_fused_sampling(1)
    N = 2 * E
    obs = vec.reset()[0]["n_agent_overcooked_features"]
    logp, value, rewards = (torch.empty(N, device=dev) for _ in range(3))
    actions = torch.empty(N, dtype=torch.int64, device=dev)
    term, trunc = (torch.empty(N, dtype=torch.bool, device=dev) for _ in range(2))

    def step():
        net.rollout_step(obs, logp, value, actions)
        vec.step_into(actions, obs, rewards, term, trunc)

    for precision in ("float32", "mxfp4"):
        if precision == "mxfp4":
            net.use_mxfp4_trunk()
        net.refresh_rollout_heads()
        t = us(step, 50)
        print(f"rollout step, {precision}: {t:.1f} us, {N / t * 1e6:.3g} agent-steps/s", flush=True)
    for M in (2048, 131072, 1048576):
        x = obs.repeat(-(-M // N), 1)[:M].contiguous()
        g = torch.randn(M, 8, device=dev) / M
        for trunk, bits in TRUNKS:
            net._keep_in_8_bits, net._coarse, net._straight = bits == 8, None if trunk == "float32" else {}, trunk == "mxfp4 straight"

            def update():
                net.zero_grad(set_to_none=True)
                logits, v = net.logits_and_value(x)
                torch.autograd.backward([logits, v], [g[:, :7], g[:, 7:]])

            torch.cuda.empty_cache()
            torch.cuda.reset_peak_memory_stats()
            t = us(update, 10)
            print(f"forward and backward of {M} samples, {trunk} trunk, {bits}-bit activations: {t:.0f} us, peak {torch.cuda.max_memory_allocated() / 1e9:.2f} GB", flush=True)
    for rows in (32, 512, 4096):  # the policy's part of a step, replayed from a graph of 32 as small rollouts are
        for precision in ("float32", "mxfp4"):
            net._coarse = None
            if precision == "mxfp4":
                net.use_mxfp4_trunk()
            net.refresh_rollout_heads()
            policy = lambda: net.rollout_step(obs[:rows], logp[:rows], value[:rows], actions[:rows])  # noqa: E731
            us(policy, 3)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                for _ in range(32):
                    policy()
            print(f"policy of {rows} rows in a graph, {precision}: {us(graph.replay, 20) / 32:.1f} us", flush=True)
    for M in (512, 2048, 16384, 65536):  # as updates of up to 65,536 samples run
        x = obs[:M].contiguous()
        g = torch.randn(M, 8, device=dev) / M
        for trunk, bits in TRUNKS:
            net._keep_in_8_bits, net._coarse, net._straight = bits == 8, None if trunk == "float32" else {}, trunk == "mxfp4 straight"

            def captured():
                net.zero_grad(set_to_none=False)
                logits, v = net.logits_and_value(x)
                torch.autograd.backward([logits, v], [g[:, :7], g[:, 7:]])

            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(3):
                    captured()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                captured()
            print(f"forward and backward of {M} samples in a graph, {trunk} trunk, {bits}-bit activations: {us(graph.replay, 50):.0f} us", flush=True)
            del graph


if __name__ == "__main__":
    main()
