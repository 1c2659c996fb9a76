"""What an asynchronous worker's push and pull move on the GPU, and that the
copies leave the host's cores to the parameter server's threads."""

import json
import os
import socket
import subprocess
import sys
import time

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_push_and_pull_leave_the_cores_alone():
    from rocps.cluster import ClusterSpec, ControlClient, Server, \
        shutdown_cluster
    from rocps.engine.async_engine import AsyncWorkerEngine
    from rocps.train.optimizer import GradientDescentOptimizer
    ports = []
    for _ in range(3):
        with socket.socket() as s:
            s.bind(("127.0.0.1", 0))
            ports.append(s.getsockname()[1])
    spec = {"ps": [f"127.0.0.1:{p}" for p in ports[:2]],
            "worker": [f"127.0.0.1:{ports[2]}"]}
    cluster = ClusterSpec(spec)
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", HIP_VISIBLE_DEVICES="",
               ROCPS_BIND_HOST="127.0.0.1")
    shards = [subprocess.Popen(
        [sys.executable, "-m", "rocps.cli.ps_server", "--cluster-json",
         json.dumps(spec), "--task-index", str(i)], env=env, cwd=ROOT)
        for i in range(2)]
    try:
        Server(cluster, "worker", 0)
        control = ControlClient(cluster.master_address)
        model = torch.nn.Sequential(*(torch.nn.Linear(
            2048, 2048, bias=False) for _ in range(4))).cuda().bfloat16()
        gen = torch.Generator("cuda").manual_seed(1)
        start = []
        for p in model.parameters():
            p.data.random_(-8, 9, generator=gen)
            start.append(p.detach().clone())
        engine = AsyncWorkerEngine(model, cluster, control, 0,
                                   torch.device("cuda:0"))
        engine.initialize(GradientDescentOptimizer(1.0))
        # whole numbers: every update is exact in bfloat16
        for step in range(3):
            engine.zero_grad()
            for p in model.parameters():
                p.grad.random_(-8, 9, generator=gen)
            want = [p.detach() - p.grad for p in model.parameters()]
            engine.push_and_pull()
            for p, q in zip(model.parameters(), want):
                assert torch.equal(p, q), step
        assert not torch.equal(start[0], next(model.parameters()))

        # CPU seconds a second: 1 for a thread that copies; torch's threads
        # would make it the number of cores
        def cores(f):
            f()
            torch.cuda.synchronize()
            wall, cpu = time.time(), time.process_time()
            for _ in range(50):
                f()
            torch.cuda.synchronize()
            return (time.process_time() - cpu) / (time.time() - wall)

        assert cores(engine.pull) < 4
    finally:
        shutdown_cluster(cluster)
        for p in shards:
            try:
                p.wait(20)
            except subprocess.TimeoutExpired:
                p.kill()
    assert [p.returncode for p in shards] == [0, 0]
