"""Calls that run at the same time, each with a workspace and outputs of its own: attention (single tokens, prompts) and beam
selection on several streams and from several captured graphs give the bits that they give alone."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_serve import Batch, dev

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::RuntimeWarning")]


class Attention:
    def __init__(self, b2, seed, lengths, n_kv, group, dim):
        self.b2, self.b = b2, Batch(b2, rng(330, seed), lengths, n_kv, group, dim, 32)
        b = self.b
        self.args = [dev(b.q), dev(b.table), dev(b.q_start), dev(b.kv)]
        self.y = torch.empty(b.rows, b.n_head, dim, device="cuda")
        self.need = b2.kv4_attn_workspace(0, b.p.h, b.rows, b.n_head, len(b.kv), max(b.new), max(b.kv))
        self.room = torch.empty(self.need, dtype=torch.uint8, device="cuda")

    def run(self, stream):
        b, (q, table, q_start, kv) = self.b, self.args
        self.b2.kv4_attn(0, b.p.h, q.data_ptr(), self.y.data_ptr(), b.rows, b.n_head, table.data_ptr(), b.stride, q_start.data_ptr(),
                         kv.data_ptr(), len(b.kv), max(b.new), max(b.kv), b.scale, self.room.data_ptr(), self.need, stream=stream)

    def out(self):
        return self.y.cpu().numpy()


class Select:
    def __init__(self, b2, seed, n_req, beams, vocab, n_out):
        r = rng(331, seed)
        self.b2, self.shape = b2, (n_req, beams, n_out)
        self.x, self.vocab = dev(r.normal(0, 2, (n_req * beams, vocab)).astype(np.float32)), vocab
        self.scores = dev(-r.uniform(0, 9, n_req * beams).astype(np.float32))
        self.o = [torch.empty(n_req * n_out, device="cuda"), *(torch.empty(n_req * n_out, dtype=torch.int32, device="cuda") for _ in range(2))]
        self.need = b2.beam_select_workspace(0, n_req, beams, vocab, n_out)
        self.room = torch.empty(self.need, dtype=torch.uint8, device="cuda")

    def run(self, stream):
        n_req, beams, n_out = self.shape
        self.b2.beam_select(0, self.x.data_ptr(), self.vocab, self.scores.data_ptr(), n_req, beams, n_out, *(t.data_ptr() for t in self.o),
                            self.room.data_ptr(), self.need, stream=stream)

    def out(self):
        return np.stack([t.cpu().numpy().view(np.uint32) for t in self.o])


def jobs(b2):
    return [Attention(b2, 0, [(1, 3000), (1, 40)], 2, 4, 128), Attention(b2, 1, [(3, 900)] * 5, 2, 3, 64),
            Attention(b2, 2, [(150, 150), (1, 700), (90, 200)], 2, 16, 64), Select(b2, 3, 8, 4, 30000, 8), Select(b2, 4, 300, 1, 20000, 16)]


@pytest.mark.parametrize("graphs", [False, True])
def test_calls_at_the_same_time_give_what_they_give_alone(b2, graphs):
    all_ = jobs(b2)
    alone = []
    for j in all_:
        j.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        alone.append(j.out())
    streams = [torch.cuda.Stream() for _ in all_]
    held = []
    for j, s in zip(all_, streams):
        if graphs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                j.run(torch.cuda.current_stream().cuda_stream)
            held.append(g)
    for _ in range(20):
        for i, (j, s) in enumerate(zip(all_, streams)):
            if graphs:
                with torch.cuda.stream(s):
                    held[i].replay()
            else:
                j.run(s.cuda_stream)
    torch.cuda.synchronize()
    for j, want in zip(all_, alone):
        assert np.array_equal(j.out(), want)
