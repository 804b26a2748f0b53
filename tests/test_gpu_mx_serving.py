"""The engine over 4-bit microscaled weights: what it keeps, and the ways to it."""
import http.client
import json

import numpy as np
import pytest
import torch

from test_gpu_mx_engine import Forward
from voxelengine import cuda as cu
from voxelengine import engine as ve

pytestmark = pytest.mark.gpu
SPEC = dict(vocab=1000, hidden=192, inter=336, layers=2, heads=3, kv_heads=1, max_pos=512)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    return ve.synth_model(str(tmp_path_factory.mktemp("mx") / "m"), seed=11, **SPEC)


def test_gate_and_up_begin_on_tiles(model, tmp_path):
    """336 gate rows take the place of 384, so that no step sorts scales and no size of gate and up
    is refused after the weights are there: what is kept equals that of a model with 384."""
    whole = ve.synth_model(str(tmp_path / "w"), seed=11, **{**SPEC, "inter": 384})
    with ve.Engine(model, max_len=64, weights=ve.WEIGHTS_MXFP4) as a, ve.Engine(whole, max_len=64, weights=ve.WEIGHTS_MXFP4) as b:
        assert a.info.inter == 336 and b.info.inter == 384
        assert a.info.weight_bytes == b.info.weight_bytes


def test_one_rank_of_tensor_parallelism(model):
    """A communicator of one rank holds the whole model: the same tokens, and all memory comes back."""
    prompt = [int(t) for t in ve.prompt(2, SPEC["vocab"], 7)]
    with ve.Engine(model, max_len=64, weights=ve.WEIGHTS_MXFP4) as eng:
        want = eng.generate([prompt], 6)[0][0]
    with cu.Ctx(0) as ctx:
        comm = cu.Comm(ctx, 1, 0, cu.comm_unique_id())
        free = []
        for _ in range(5):
            with ve.Engine(model, max_len=64, max_batch=8192, weights=ve.WEIGHTS_MXFP4, comm=comm) as eng:
                assert [int(t) for t in eng.generate([prompt], 6)[0][0]] == [int(t) for t in want]
            ctx.sync()
            free.append(torch.cuda.mem_get_info()[0])
        comm.close()
    assert free[1:] == free[:-1], free  # 8192 rows of 192 values are 6 MB


def test_server_over_microscaled_weights(model):
    """POST /generate gives the microscaled engine's tokens, which are not the stored weights'."""
    prompt = [int(t) for t in ve.prompt(3, SPEC["vocab"], 9)]
    with ve.Engine(model, max_len=64, weights=ve.WEIGHTS_MXFP4) as eng:
        want = [int(t) for t in eng.generate([prompt], 12)[0][0]]
    with ve.Server(model, devices=[0], max_len=64, weights=ve.WEIGHTS_MXFP4) as s:
        c = http.client.HTTPConnection("127.0.0.1", s.port, timeout=60)
        c.request("POST", "/generate", json.dumps({"tokens": prompt, "max_tokens": 12}))
        r = c.getresponse()
        got = json.loads(r.read())
        c.close()
    assert r.status == 200 and got["tokens"] == want


def test_after_work_of_another_stream(model):
    """Memory that another stream (here torch's) writes and reads: ordered on the device, in both
    directions, through the stream that opure_stream gives."""
    n, cols = 4096, 4096
    with cu.Ctx(0) as ctx:
        own = torch.cuda.ExternalStream(cu.lib().opure_stream(ctx.h))
        side = torch.cuda.Stream()
        q = ctx.mx_matrix(n, cols, cu.MX_FP8)
        x, y = torch.zeros(n, cols, device="cuda"), torch.zeros(n, cols, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for k in range(5):
                big = torch.full((n, cols), float(k), device="cuda")
                for _ in range(20):
                    big = big * 1.0
                x.copy_(big)              # not there yet when the next lines run
                own.wait_stream(side)
                ctx.mx_quantize(x.data_ptr(), cu.F32, cols, q)
                ctx.mx_dequantize(q, y.data_ptr(), cu.F32, cols)
                side.wait_stream(own)
                got = y.clone()
                y.zero_()
                assert bool((got == float(k)).all())
        torch.cuda.synchronize()


def test_logits_are_those_of_the_definition(model):
    """Against the 64-bit forward. What differs: an 8-bit operand whose value lies within fp32's error of
    a rounding boundary is a step off (16,000 operands for 9 positions, a chance of 2^-15 each: under
    0.5 expected, each 2^-3.5 of one of 192 inputs, 0.6% of a layer's share), and a few fp16 keys and
    values likewise (6e-5 each). So most prompts agree to 1e-3 of the logits' spread, all to 2e-2."""
    forward, errors = Forward(model), []
    with ve.Engine(model, max_len=64, weights=ve.WEIGHTS_MXFP4) as eng:
        for seed in range(11):
            prompt = [int(t) for t in ve.prompt(50 + seed, SPEC["vocab"], 9)]
            want = forward.logits(prompt)[-1]
            errors.append(np.sqrt(np.mean((eng.forward_logits(prompt) - want) ** 2)) / want.std())
    assert np.median(errors) <= 1e-3 and max(errors) <= 2e-2, errors
