"""The kept fold of the router's running statistics: graphs and streams that read it, and what changes it meanwhile."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def layer(tokens=96, seed=0):
    from omni_moe_b200.modules import OmniMoE, OmniMoEConfig
    torch.manual_seed(seed)
    m = OmniMoE(OmniMoEConfig(256, 512, "silu", 1024, 8)).bfloat16().cuda().eval()
    return m, torch.randn(1, tokens, 256, device="cuda").bfloat16()


def move(m, to):
    """Statistics under which other experts are selected."""
    with torch.no_grad():
        for j, bn in enumerate((m.router_norm_x, m.router_norm_y)):
            bn.running_mean.copy_(torch.linspace(-to, to * (j + 1), bn.running_mean.numel()))
            bn.running_var.copy_(torch.linspace(0.5, 2.0, bn.running_var.numel()))


def fresh(m, x):
    """What a module gives that has never seen other statistics."""
    other, _ = layer()
    other.load_state_dict(m.state_dict())
    with torch.no_grad():
        return other.eval()(x)


def junk():
    """Fills memory that was given back with NaN."""
    return [torch.full((64,), float("nan"), device="cuda") for _ in range(256)]


def test_graph_follows_statistics():
    m, x = layer()
    g = m.graphed(96)
    assert torch.equal(g(x), fresh(m, x))
    for to in (0.5, 2.0):
        move(m, to)
        full = junk()
        assert torch.equal(g(x), fresh(m, x))
        del full
    outs = [g(x).clone()]
    with torch.no_grad():
        m.train()
        m(x)                       # a training forward: statistics that move behind torch's version counters
        m.eval()
        full = junk()
        assert torch.equal(m(x), fresh(m, x))
    outs.append(g(x).clone())
    assert torch.equal(outs[1], fresh(m, x)) and not torch.equal(*outs)
    del full


def test_two_graphs_and_eager_calls_share_the_fold():
    m, x = layer(48)
    a, b = m.graphed(48), m.graphed(48)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for to in (0.0, 0.5, 2.0):
        move(m, to)
        want = fresh(m, x)
        torch.cuda.synchronize()
        for _ in range(10):
            for g, s in zip((a, b), streams):
                with torch.cuda.stream(s):
                    g(x)
            with torch.no_grad():
                y, z = m(x), m.decode(x)
        torch.cuda.synchronize()
        assert torch.equal(a.y.view_as(want), want) and torch.equal(b.y.view_as(want), want) and torch.equal(y, want)
        assert float((z.double() - want.double()).norm() / want.double().norm()) < 2 ** -7  # both round activation and output


@pytest.mark.parametrize("call", ["forward", "decode"])
def test_other_streams_wait_for_the_fold(call):
    m, x = layer(40)
    run = m.forward if call == "forward" else m.decode
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        want = {0.5: None, 2.0: None, 1.0: None}
        for to in want:
            move(m, to)
            other, _ = layer()
            other.load_state_dict(m.state_dict())
            want[to] = (other.eval().forward if call == "forward" else other.decode)(x)
        for to in want:
            move(m, to)
            torch.cuda.synchronize()
            with torch.cuda.stream(a):
                torch.cuda._sleep(20_000_000)   # some 10 ms before the fold is computed
                first = run(x)
            with torch.cuda.stream(b):
                second = run(x)
            torch.cuda.synchronize()
            assert torch.equal(first, want[to]) and torch.equal(second, want[to])


@pytest.mark.parametrize("call", ["forward", "decode"])
def test_a_change_waits_for_calls_on_other_streams(call):
    m, x = layer(40)
    run = m.forward if call == "forward" else m.decode
    with torch.no_grad():
        move(m, 0.5)
        want = run(x).clone()       # made on this stream
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(x)
            torch.cuda._sleep(20_000_000)
            late = run(x)           # in flight while the statistics change
        move(m, 2.0)
        changed = run(x)
        full = junk()
        torch.cuda.synchronize()
        assert torch.equal(late, want) and not torch.equal(changed, want)
        del full


def test_one_stream_does_not_wait():
    """A change replaces a pair that one stream alone has read: the call is enqueued behind a long kernel, not held up by it."""
    m, x = layer(40)
    with torch.no_grad():
        for call in (m.forward, m.decode):
            call(x)
        torch.cuda.synchronize()
        move(m, 2.0)
        done = torch.cuda.Event()
        torch.cuda._sleep(200_000_000)      # some 100 ms
        done.record()
        m.decode(x), m(x)
        assert not done.query()
        torch.cuda.synchronize()


@pytest.mark.parametrize("how", ["graphed", "raw"])
def test_statistics_that_a_captured_training_step_moves(how):
    """Replays move the running statistics without any Python code: eval calls between them see each step's."""
    m, x = layer()
    m.train()
    if how == "graphed":
        g = m.graphed(96)
        step = lambda: g(x)
    else:
        # a step through the differentiable form, as a training program captures it
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.autograd.grad(m(x).float().square().mean(), m.gate_proj.weight)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            torch.autograd.grad(m(x).float().square().mean(), m.gate_proj.weight)
        step = graph.replay
    m.eval()
    outs = []
    with torch.no_grad():
        for _ in range(3):
            step()
            want = fresh(m, x)
            assert torch.equal(m(x), want)
            few = fresh(m, x[:, :7]), m.decode(x[:, :7])
            assert float((few[1].double() - few[0].double()).norm() / few[0].double().norm()) < 2 ** -7
            other, _ = layer()
            other.load_state_dict(m.state_dict())
            assert torch.equal(few[1], other.eval().decode(x[:, :7]))
            outs.append(want)
    assert not torch.equal(outs[0], outs[2])


def test_eval_graph_beside_a_training_graph():
    m, x = layer()
    trained, tested = m.train().graphed(96), m.eval().graphed(96)
    with torch.no_grad():
        for _ in range(2):
            trained(x)
            assert torch.equal(tested(x), fresh(m, x))
