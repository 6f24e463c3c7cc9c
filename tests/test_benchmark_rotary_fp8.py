"""The benchmark commands' rotary and 8-bit cache options, on the CPU and the GPU."""
import json

import pytest
import torch

from kotflash_amd import benchmark_decode, benchmark_decoder_block as bdb
from kotflash_amd.rotary import Rotary


@pytest.mark.parametrize("interleaved", [False, True])
def test_block_turns_queries_and_keys(interleaved):
    torch.manual_seed(0)
    rot = Rotary(16, interleaved=interleaved, device="cpu")
    block = bdb.DecoderBlock(4, 2, 16, attention_dtype=torch.float32, rotary=rot)
    x = torch.randn(2, 24, 64)
    a, b = block(x, "sdpa_expanded_kv"), block(x, "sdpa_native_gqa")
    assert torch.allclose(a, b, atol=1e-5, rtol=1e-5)
    block.rotary = None
    assert not torch.allclose(a, block(x, "sdpa_expanded_kv"), atol=1e-3)


@pytest.mark.parametrize("argv, message", [
    (["--rotary", "yes"], "invalid choice"), (["--rotary", "half", "--head-dim", "33"], "even --head-dim"),
])
def test_block_arguments(argv, message, capsys):
    with pytest.raises(SystemExit):
        bdb.parse_args(argv)
    assert message in capsys.readouterr().err


@pytest.mark.parametrize("argv", [["--kv-fp8"], ["--kv-fp8", "--page-size", "24"]])
def test_decode_arguments(argv, capsys):
    with pytest.raises(SystemExit):
        benchmark_decode.parse_args(["--device", "cpu"] + argv)
    assert "--kv-fp8 needs --page-size" in capsys.readouterr().err


def test_decode_report_on_cpu(capsys):
    benchmark_decode.main(["--device", "cpu", "--batch", "1", "--q-heads", "4", "--kv-heads", "2", "--head-dim", "16",
                           "--kv-seq", "1024", "--warmup", "1", "--iterations", "1", "--repeats", "3",
                           "--page-size", "32", "--kv-fp8"])
    report = json.loads(capsys.readouterr().out)
    assert {"paged_auto", "paged_fp8_auto"} <= set(report["results"])
    for metric in ("attention_only", "append_plus_attention"):
        assert report["correctness"]["paged_fp8_auto"][metric]["within_tolerance"]


@pytest.mark.gpu
def test_decode_report_on_gpu(capsys):
    benchmark_decode.main(["--kv-seq", "2048", "--warmup", "2", "--iterations", "3", "--repeats", "3",
                           "--page-size", "16", "--kv-fp8"])
    report = json.loads(capsys.readouterr().out)
    assert report["backend_failures"] == {}
    assert report["results"]["paged_fp8_auto"]["append_plus_attention"]["gpu_median_ms"] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", ["half", "interleaved"])
def test_block_report_on_gpu(rotary, capsys):
    bdb.main(["--batch", "1", "--seq", "256", "--q-heads", "4", "--kv-heads", "2", "--head-dim", "64",
              "--warmup", "1", "--iterations", "3", "--rotary", rotary])
    report = json.loads(capsys.readouterr().out)
    assert "hip_forward" not in report, report.get("hip_forward")
    assert report["rotary"] == rotary
    for name in bdb.BACKENDS:
        assert report[name]["loss_finite"] and report[name]["parameters_finite_after_update"], name


@pytest.mark.gpu
def test_block_gradients_on_gpu():
    """Parameter gradients of the HIP block against the fp32 SDPA block. Ten
    fp16 roundings lie on a gradient's way (q, k, v, turned q and k, P, dP, dO
    and the two input gradients), each 2^-11 relative: 5e-3 of its norm where
    they add up, and twice that for sums that partly cancel. That is for
    normal values; the mean over 358400 outputs leaves gradients of 2 / 358400 =
    5.6e-6 of them, dO of some 3e-6 and, through weights of 1 / 700, dQ and dK of
    1e-7, where fp16's step is 2^-24 and half of it 3e-8: a hundredth of dO and
    a third of dQ and dK. The SDPA block in fp16 has the same roundings, so its
    own distance from fp32 says what these cost; twice that for two such blocks."""
    torch.manual_seed(0)
    x = torch.randn(2, 700, 4 * 64, device="cuda")
    rot = Rotary(64, device="cuda")
    runs = (("hip", torch.float16), ("sdpa_expanded_kv", torch.float32), ("sdpa_expanded_kv", torch.float16))
    blocks = [bdb.DecoderBlock(4, 2, 64, attention_dtype=t, rotary=rot).cuda() for _, t in runs]
    for block, (backend, _) in zip(blocks, runs):
        block.load_state_dict(blocks[0].state_dict())
        block(x, backend).square().mean().backward()
    for (name, a), b, c in zip(blocks[0].named_parameters(), blocks[1].parameters(), blocks[2].parameters()):
        err, plain = (float((t.grad - b.grad).norm() / b.grad.norm()) for t in (a, c))
        print(name, err, plain)
        assert err < 1e-2 + 2 * plain, (name, err, plain)
