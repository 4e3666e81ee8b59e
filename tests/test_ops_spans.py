"""Document spans: documents over many chunks of a row's tokens, in one launch and in two (rows of over 8 chunks), whose time follows the tokens."""
import pytest
import torch

from gqa_kernels import document_spans

pytestmark = pytest.mark.gpu
CHUNK = 4096  # tokens a workgroup


def spans_of(ids):
    S = ids.shape[1]
    change = torch.ones_like(ids, dtype=torch.bool)
    change[:, 1:] = ids[:, 1:] != ids[:, :-1]
    at = torch.arange(S, device=ids.device).expand_as(ids)
    start = torch.where(change, at, torch.zeros_like(at)).cummax(1).values
    nxt = torch.full_like(at, S)
    nxt[:, :-1] = torch.where(change[:, 1:], at[:, 1:], torch.full_like(at[:, 1:], S))
    end = nxt.flip(1).cummin(1).values.flip(1)
    return tuple(torch.where(ids < 0, torch.zeros_like(x), x).int() for x in (start, end))


def ids_of(lengths, S):
    ids = torch.repeat_interleave(torch.tensor([i for _, i in lengths]), torch.tensor([n for n, _ in lengths]))
    return torch.cat([ids, torch.full((max(0, S - len(ids)),), -1)])[:S].to(torch.int32).cuda()


@pytest.mark.parametrize("S", [CHUNK - 1, CHUNK, CHUNK + 1, 2 * CHUNK, 3 * CHUNK + 5, 8 * CHUNK, 8 * CHUNK + 1, 9 * CHUNK, 20 * CHUNK])
def test_documents_that_start_and_end_at_the_chunks_borders(S):
    c = CHUNK
    rows = [ids_of([(n, i) for i, n in enumerate(lengths)], S) for lengths in (
        [S], [c, S], [c - 1, 1, c, 1, S], [c + 1, c - 1, S], [1, S], [S - 1, 1], [2 * c, c, c, S], [3 * c - 1, c + 2, S], [7] * 3000 + [S])]
    rows.append(ids_of([(c, -1), (5, 0), (2 * c, -3), (2 * c, -4), (S, 2)], S))  # padding over the borders
    rows.append(ids_of([(3, 1), (3 * c, 0), (c, -1), (S, 0)], S))
    ids = torch.stack(rows)
    got, want = document_spans(ids), spans_of(ids)
    assert torch.equal(got.starts, want[0]) and torch.equal(got.ends, want[1])
    wide = torch.zeros(len(rows), S + 3, dtype=torch.int32, device="cuda")
    wide[:, 1:S + 1] = ids
    got = document_spans(wide[:, 1:S + 1])
    assert torch.equal(got.starts, want[0]) and torch.equal(got.ends, want[1])


def test_a_document_over_more_chunks_than_threads():
    S = 2500 * CHUNK + 17
    ids = torch.stack([ids_of([(n, i) for i, n in enumerate(ls)], S) for ls in ([S], [100, 1300 * CHUNK, 1100 * CHUNK, S], [5000] * 10 + [S])])
    got, want = document_spans(ids), spans_of(ids)
    assert torch.equal(got.starts, want[0]) and torch.equal(got.ends, want[1])


@pytest.mark.parametrize("S", [5 * CHUNK + 3, 12 * CHUNK + 3])
def test_captured(S):
    ids = ids_of([(3 * CHUNK + 1, 0), (100, 1), (S, 2)], S).repeat(2, 1)
    document_spans(ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = document_spans(ids)
    for n in (1, CHUNK, 2 * CHUNK + 9, S - 1):
        ids.copy_(ids_of([(n, 0), (S, 1)], S).repeat(2, 1))
        got.starts.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = spans_of(ids)
        assert torch.equal(got.starts, want[0]) and torch.equal(got.ends, want[1])


def test_one_document_of_millions_of_tokens_takes_no_longer_than_many():
    S = 1 << 22
    rows = {"one": torch.zeros(1, S, dtype=torch.int32, device="cuda"), "many": (torch.arange(S, device="cuda") // 300).int()[None].contiguous()}
    times = {}
    for name, ids in rows.items():
        document_spans(ids)
        torch.cuda.synchronize()
        best = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            document_spans(ids)
            b.record()
            torch.cuda.synchronize()
            best.append(a.elapsed_time(b))
        times[name] = min(best)
    assert times["one"] < 8 * times["many"], times  # (a walk from every chunk to the document's ends: hundreds of times)
