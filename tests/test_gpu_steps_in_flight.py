"""Device-resident decode steps issued one after the other while the stream is still busy: each step keeps its own
positions and sequences, whatever the host prepares meanwhile."""
import numpy as np
import pytest

from bitnetrs_b200 import KV_BF16, KV_F32, KV_I4, KV_I8, BitNetModel, ModelConfig, synth

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kv", [KV_F32, KV_BF16, KV_I8, KV_I4])
def test_steps_in_flight_keep_their_positions(cuda_backend, kv):
    cfg = ModelConfig(777, 512, 2, 4, 1, 640, 600, 10000.0, 1e-5)
    m = BitNetModel(synth.random_model(cfg, seed=5), cuda_backend, max_batch_tokens=64)
    dev = torch.device("cuda", cuda_backend.device_id)
    lens, steps = [40, 7, 100], 4
    stream = torch.cuda.Stream(dev)
    got, caches = [], []
    for busy in (False, True):
        cache = m.new_kv_cache(num_pages=80, max_seqs=len(lens), kv_dtype=kv)
        caches.append(cache)  # kept: the second has pages of its own
        for s, n in enumerate(lens):
            cache.fill_random(s, n, 21)
            cache.reserve(s, n + steps)
        tok = torch.tensor([5, 6, 7], dtype=torch.int32, device=dev)
        seqs = np.arange(len(lens), dtype=np.uint32)
        m.decode_step_device(cache, seqs, tok.data_ptr(), tok.data_ptr(), 0, stream.cuda_stream)  # the graph is captured
        torch.cuda.synchronize()
        if busy:
            with torch.cuda.stream(stream):
                torch.cuda._sleep(400_000_000)  # some 0.2 s, behind which the steps queue up
        for _ in range(steps - 1):
            m.decode_step_device(cache, seqs, tok.data_ptr(), tok.data_ptr(), 0, stream.cuda_stream)
            if not busy:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        m.check()
        got.append([tok.cpu().numpy()] + [x for s, n in enumerate(lens) for x in cache.read(s, n + steps)])
    for a, b in zip(*got):
        np.testing.assert_array_equal(a, b)
