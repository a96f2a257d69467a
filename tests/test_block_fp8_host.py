"""CPU-only checks of the block-scaled 8-bit floating point operators: what the C entry points and their Python wrappers
refuse, size queries, and the reference that the GPU tests compare with.  No kernel is launched here."""
import ctypes

import pytest
import torch

import fp8_reference as R

P = ctypes.c_void_p
NULL = P(0)
BIG = 1 << 40


def lib():
    from quantization_amd import _native
    return _native.lib()


def test_reference_rounds_as_torch_does():
    v = torch.cat([torch.linspace(-448, 448, 20001), torch.logspace(-12, 2, 5000), torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 0.0, 463.9])])
    assert torch.equal(R.nearest_e4m3(v.double()), v.to(torch.float8_e4m3fn).double())


def test_quantizer_refusals():
    L = lib()
    p = P(4096)
    for f in (L.miq_quantize_blocks_fp8, L.miq_quantize_weight_fp8):
        assert f(NULL, 0, -1, 4, NULL, NULL, NULL) == -1 and b"negative" in L.miq_last_error()
        assert f(p, 3, 2, 4, p, p, NULL) == -1 and b"dtype" in L.miq_last_error()
        assert f(p, 0, 2, 4, NULL, p, NULL) == -1 and b"null" in L.miq_last_error()
        assert f(p, 0, BIG, 4, p, p, NULL) == -5
        assert f(p, 0, 1 << 30, 1 << 30, p, p, NULL) == -5
        assert f(P(4098), 0, 2, 4, p, p, NULL) == -2
        assert f(P(4097), 1, 2, 4, p, p, NULL) == -2
        assert f(p, 0, 2, 4, p, P(4098), NULL) == -2
        assert f(NULL, 0, 0, 4, NULL, NULL, NULL) == 0 and f(NULL, 0, 4, 0, NULL, NULL, NULL) == 0


def test_norm_refusals():
    L = lib()
    p = P(4096)

    def norm(x=p, r=NULL, w=p, dt=2, wdt=2, M=2, K=8, eps=1e-6, total=NULL, q=p, s=p):
        return L.miq_rms_norm_fp8(x, r, w, dt, wdt, M, K, eps, total, q, s, NULL)
    assert norm(M=-1) == -1
    assert norm(dt=4) == -1
    assert norm(dt=2, wdt=1) == -1 and b"weight_dtype" in L.miq_last_error()
    assert norm(eps=-1.0) == -1 and norm(eps=float("nan")) == -1 and norm(eps=float("inf")) == -1
    assert norm(r=p) == -1 and norm(total=p) == -1 and b"together" in L.miq_last_error()
    assert norm(x=NULL) == -1
    assert norm(x=P(4097)) == -2
    assert norm(M=BIG) == -5 and norm(M=1 << 25) == -5
    assert norm(M=0) == 0


def test_product_refusals():
    L = lib()
    p = P(4096)

    def gemm(x=p, xs=p, w=p, ws=p, M=2, N=8, K=128, b=NULL, out=p, dt=2):
        return L.miq_gemm_fp8(x, xs, w, ws, M, N, K, b, out, dt, NULL, 0, NULL)

    def gated(x=p, xs=p, wg=p, sg=p, wu=p, su=p, M=2, N=8, K=128, act=0, q=p, s=p, work=p, size=1 << 40):
        return L.miq_gated_fp8(x, xs, wg, sg, wu, su, M, N, K, act, q, s, work, size, NULL)
    for f in (gemm, gated):
        assert f(M=-1) == -1 and f(N=-1) == -1 and f(K=-1) == -1
        assert f(M=BIG) == -5 and f(N=BIG) == -5 and f(K=1 << 22) == -5 and f(M=1 << 20, N=1 << 20) == -5
        assert f(M=16, N=(1 << 26) + 1) == -5 and f(M=1, N=1 << 28) == -5 and f(M=17, N=(1 << 28) + 1) == -5
        assert f(x=NULL) == -1 and f(xs=NULL) == -1
        assert f(xs=P(4098)) == -2
        assert f(M=0) == 0 and f(N=0) == 0
    assert gemm(out=NULL) == -1 and gemm(dt=3) == -1 and gemm(dt=4) == -1 and gemm(out=P(4104)) == -2
    assert gated(act=2) == -1 and gated(q=NULL) == -1 and gated(su=NULL) == -1
    assert L.miq_gemm_fp8_workspace(BIG, 4, 4, 0) == 0 and L.miq_gated_fp8_workspace(4, -1, 4) == 0
    for m in (1, 16, 100, 1000):
        if L.miq_gated_fp8_workspace(m, 512, 8192):
            assert gated(M=m, N=512, K=8192, size=16) == -3
            assert gated(M=m, N=512, K=8192, work=P(4100)) == -2


def test_wrappers_refuse_host_tensors():
    from quantization_amd import block_fp8 as F
    x = torch.zeros(2, 128)
    q, s, ws = x.to(torch.float8_e4m3fn), torch.zeros(1, 2), torch.zeros(1, 1)
    for call in (lambda: F.quantize_blocks_fp8(x), lambda: F.quantize_weight_fp8(x), lambda: F.rms_norm_fp8(x, x[0]),
                 lambda: F.linear_fp8(q, s, q, ws), lambda: F.gated_linear_fp8(q, s, q, ws, q, ws)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_layer_owns_its_bias(dtype):
    """A layer built from a float one shares no storage with it: loading a state into the one leaves the other as it is."""
    from quantization_amd import block_fp8 as F
    lin = torch.nn.Linear(6, 3).to(dtype)
    before = lin.bias.detach().clone()
    layer = F.BlockFP8Linear(torch.zeros(3, 6).to(torch.float8_e4m3fn), torch.ones(1, 1), lin.bias)
    assert layer.bias.dtype == torch.float32 and torch.equal(layer.bias, before.float()) and not layer.bias.requires_grad
    layer.load_state_dict({"weight": layer.weight, "weight_scale": layer.weight_scale, "bias": torch.full((3,), 7.0)})
    assert torch.equal(lin.bias.detach(), before)
    with torch.no_grad():
        lin.bias.fill_(5.0)
    assert torch.equal(layer.bias, torch.full((3,), 7.0))


def test_gated_layer_calls_its_down_projection(monkeypatch):
    """Hooks on `down` run, and a module put in its place is what is called, with the pair and the type to answer in."""
    from quantization_amd import block_fp8 as F
    f8, pair = torch.zeros(4, 6).to(torch.float8_e4m3fn), (torch.zeros(2, 4).to(torch.float8_e4m3fn), torch.ones(1, 2))
    monkeypatch.setattr(F, "quantize_blocks_fp8", lambda x: (x.to(torch.float8_e4m3fn), torch.ones(1, 2)))
    monkeypatch.setattr(F, "gated_linear_fp8", lambda *a: pair)
    monkeypatch.setattr(F, "linear_fp8", lambda q, s, w, ws, b, dtype: torch.zeros(2, w.shape[0], dtype=dtype))
    down = F.BlockFP8Linear(torch.zeros(6, 4).to(torch.float8_e4m3fn), torch.ones(1, 1))
    mlp = F.BlockFP8GatedMLP(f8, torch.ones(1, 1), f8, torch.ones(1, 1), down)
    seen = []
    down.register_forward_hook(lambda module, args, out: seen.append(args) or out + 1)
    y = mlp(torch.zeros(2, 6, dtype=torch.float16))
    assert len(seen) == 1 and seen[0][0] is pair and y.dtype == torch.float16 and bool((y == 1).all())
    assert mlp(pair).dtype == torch.bfloat16 and mlp(torch.zeros(2, 6)).dtype == torch.float32
    down.out_dtype = torch.float32
    assert mlp(pair).dtype == torch.float32 and mlp(torch.zeros(2, 6).half()).dtype == torch.float32

    class Other(torch.nn.Module):
        def forward(self, x, out_dtype):
            return x, out_dtype
    mlp.down = Other()
    assert mlp(torch.zeros(2, 6).half()) == (pair, torch.float16)


def test_gated_layer_casts_another_down_projection():
    """Codes and scales keep their types in a cast of the model; a float module in the place of `down` is cast as any other."""
    from quantization_amd import block_fp8 as F
    f8 = torch.zeros(4, 6).to(torch.float8_e4m3fn)
    mlp = F.BlockFP8GatedMLP(f8, torch.ones(1, 1), f8, torch.ones(1, 1), F.BlockFP8Linear(f8, torch.ones(1, 1), torch.zeros(4)))
    mlp.half()
    assert {n: b.dtype for n, b in mlp.named_buffers(remove_duplicate=False)} == {   # (one tensor of codes for all three)
        "gate": f8.dtype, "gate_scale": torch.float32, "up": f8.dtype, "up_scale": torch.float32, "down.weight": f8.dtype,
        "down.weight_scale": torch.float32, "down.bias": torch.float32}
    mlp.down = torch.nn.Linear(4, 6)
    mlp.to(torch.bfloat16)
    assert mlp.gate.dtype == f8.dtype and mlp.gate_scale.dtype == torch.float32
    assert mlp.down.weight.dtype == mlp.down.bias.dtype == torch.bfloat16


def test_norm_refuses_a_residual_of_another_shape():
    """As many elements are not enough: rows of another order, or of another division into dimensions, are not x's."""
    from quantization_amd import block_fp8 as F
    x = torch.zeros(2, 3, 128)
    for other in (x.view(3, 2, 128), x.view(6, 128), x[:, :1], x[0, 0]):
        with pytest.raises(RuntimeError, match="residual must be"):
            F.rms_norm_fp8(x, x[0, 0], 1e-6, residual=other)
    with pytest.raises(RuntimeError, match="residual must be"):
        F.rms_norm_fp8(x.view(6, 128), x[0, 0], 1e-6, residual=x)


@pytest.mark.gpu
def test_wrappers_refuse_wrong_tensors():
    from quantization_amd import block_fp8 as F
    x = torch.randn(4, 256, device="cuda")
    q, s = F.quantize_blocks_fp8(x)
    w, ws = F.quantize_weight_fp8(torch.randn(130, 256, device="cuda"))
    bad = [lambda: F.quantize_blocks_fp8(x.double()), lambda: F.quantize_weight_fp8(x.t()), lambda: F.quantize_weight_fp8(x[0]),
           lambda: F.rms_norm_fp8(x, torch.ones(255, device="cuda")), lambda: F.rms_norm_fp8(x, torch.ones(256, device="cuda").half()),
           lambda: F.rms_norm_fp8(x, torch.ones(256, device="cuda"), residual=x[:2]),
           lambda: F.rms_norm_fp8(x, torch.ones(256, device="cuda"), residual=x.half()),
           lambda: F.rms_norm_fp8(x, torch.ones(256)), lambda: F.rms_norm_fp8(x, torch.ones(256, device="cuda"), -1.0),
           lambda: F.linear_fp8(x, s, w, ws), lambda: F.linear_fp8(q, s.t().contiguous(), w, ws), lambda: F.linear_fp8(q, s.t().contiguous().t(), w, ws),
           lambda: F.linear_fp8(q, s, w, ws.half()), lambda: F.linear_fp8(q, s, w[:, :128].contiguous(), ws[:, :1].contiguous()),
           lambda: F.linear_fp8(q, s, w, ws, torch.zeros(5, device="cuda")), lambda: F.linear_fp8(q, s, w, ws, None, torch.int32),
           lambda: F.linear_fp8(q, s, w.cpu(), ws), lambda: F.gated_linear_fp8(q, s, w, ws, w[:128].contiguous(), ws[:1].contiguous()),
           lambda: F.gated_linear_fp8(q, s, w, ws, w, ws, "relu")]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError(f"call {i} was taken")
