"""The 8-bit forward on feature shards: CPU ranks (gloo, world size 2), plain torch in place of the operators."""
import os
import sys
from pathlib import Path

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = Path(__file__).resolve().parents[1]


def _worker(rank, world, port, q):
    sys.path.insert(0, str(ROOT))
    import crosslayer_transcoder_b200.model as M
    from crosslayer_transcoder_b200 import parallel
    from tests import fp8_stand_in

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        fp8_stand_in.install()
        L, D, F = 3, 8, 16
        for decoder_cls, nl in ((M.CrosslayerDecoder, M.JumpReLU(0.03, 1.0, L, F)), (M.Decoder, M.ReLU()), (M.Decoder, M.PerLayerTopK(k=2))):
            torch.manual_seed(5)
            module = M.CrossLayerTranscoderModule(model=M.CrossLayerTranscoder(nl, M.Encoder(D, F, L), decoder_cls(D, F, L)))
            with torch.no_grad():
                module.model.decoder.b.normal_()
            x = torch.randn(6, L, D)
            module.model.eight_bit = True
            whole = module(x)                            # an unsharded module takes the switch
            assert whole[2].shape == (6, L, D)
            parallel.shard_module(module, rank, world)
            parallel.attach(module, fused=False)
            for call in (module, module.model):
                for grads in (True, False):
                    with torch.set_grad_enabled(grads):
                        try:
                            out = call(x)
                        except NotImplementedError as e:
                            assert "feature shards" in str(e)
                        else:
                            raise AssertionError(f"off by {float((out[2] - whole[2]).detach().abs().max())} and nothing raised")
            module.model.eight_bit = False
            assert module(x)[0].shape == (6, L, F // world)
        q.put((rank, "ok"))
    except Exception:  # pragma: no cover
        import traceback

        q.put((rank, traceback.format_exc()))
    finally:
        dist.destroy_process_group()


def test_eight_bit_is_refused_on_feature_shards():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, 29619, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = [q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(timeout=30)
    assert all(v == "ok" for _, v in res), res
