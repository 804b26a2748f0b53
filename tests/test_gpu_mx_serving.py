"""The engine over 4-bit microscaled weights: what it keeps, and the ways to it."""
import pytest
import torch

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
