"""Host side of the 8-bit activation checkpoints, the RMS norm and the scaled embedding: what the entry points refuse, before
any launch, and the workspace sizes they ask for."""
import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from bifold_amd.hip import lib
    return lib


PTR = 4096                                     # an aligned address nothing reads: every call below is refused


def refused(L, rc, code, text):
    assert rc == code, (rc, L.lib.bf_last_error())
    assert text.encode() in L.lib.bf_last_error(), L.lib.bf_last_error()


def test_act8_refusals(L):
    lib = L.lib
    refused(L, lib.bf_act8_pack(PTR, 64, 7, PTR, PTR, 4, 64, None), -1, "bad dtype")
    refused(L, lib.bf_act8_pack(PTR, 64, L.F32, PTR, PTR, 4, 0, None), -1, "bad shape")
    refused(L, lib.bf_act8_pack(PTR, 64, L.F32, PTR, PTR, -1, 64, None), -1, "bad shape")
    refused(L, lib.bf_act8_pack(PTR, 63, L.F32, PTR, PTR, 4, 64, None), -1, "leading dimension")
    refused(L, lib.bf_act8_pack(None, 64, L.F32, PTR, PTR, 4, 64, None), -1, "null")
    refused(L, lib.bf_act8_pack(PTR, 64, L.F32, PTR, None, 4, 64, None), -1, "null")
    refused(L, lib.bf_act8_pack(PTR + 2, 64, L.F32, PTR, PTR, 4, 64, None), -2, "aligned")
    refused(L, lib.bf_act8_pack(PTR, 32, L.F16, PTR, PTR, 1 << 30, 32, None), -1, "2^34")
    refused(L, lib.bf_act8_pack(PTR, 128, L.F16, PTR, PTR, 1 << 60, 128, None), -1, "2^34")    # 2^60 rows of 2^4 vectors: 2^64
    refused(L, lib.bf_act8_unpack(PTR, PTR, PTR, 63, L.F16, 4, 64, None), -1, "leading dimension")
    refused(L, lib.bf_act8_unpack(PTR, PTR, PTR + 1, 64, L.F16, 4, 64, None), -2, "aligned")
    for act in (L.ACT_NONE, 3, 5, 99):
        refused(L, lib.bf_act8_gelu_fwd(PTR, 64, PTR, PTR, PTR, L.F16, act, 4, 64, None), -1, "act must be")
        refused(L, lib.bf_act8_gelu_bwd(PTR, 64, PTR, PTR, PTR, 64, L.F16, act, 4, 64, None), -1, "act must be")
    assert lib.bf_act8_pack(None, 64, L.F32, None, None, 0, 64, None) == 0         # no rows: nothing to do


def test_rmsnorm_refusals(L):
    lib = L.lib

    def fwd(x=PTR, ldx=64, xd=L.F32, delta=None, ldd=0, dd=0, gamma=PTR, xo=None, ldo=0, y=PTR, yd=L.F32, rstd=None, q=None,
            code=None, rows=4, cols=64, eps=1e-6):
        return lib.bf_rmsnorm_fwd(x, ldx, xd, delta, ldd, dd, gamma, xo, ldo, y, yd, rstd, q, code, rows, cols, eps, None)

    refused(L, fwd(xd=5), -1, "x_dtype")
    refused(L, fwd(yd=3), -1, "y_dtype")
    refused(L, fwd(delta=PTR, ldd=64, dd=9), -1, "delta_dtype")
    refused(L, fwd(cols=0), -1, "bad shape")
    refused(L, fwd(ldx=60), -1, "leading dimension")
    refused(L, fwd(delta=PTR, ldd=63), -1, "leading dimension")
    refused(L, fwd(delta=PTR, ldd=64, xo=PTR, ldo=3), -1, "leading dimension")
    refused(L, fwd(q=PTR), -1, "checkpoint")
    refused(L, fwd(eps=-1.0), -1, "eps")
    refused(L, fwd(gamma=None), -1, "null")
    refused(L, fwd(y=PTR + 1), -2, "aligned")
    refused(L, lib.bf_rmsnorm_fwd_fp8(PTR, 64, L.F32, None, 0, 0, PTR, None, 0, PTR, None, None, None, None, 4, 64, 1e-6, None),
            -1, "null")
    assert fwd(rows=0, x=None, y=None) == 0

    def bwd(dy=PTR, ldy=64, dyd=L.F16, x=PTR, ldx=64, xd=L.F32, q=None, code=None, gamma=PTR, rstd=PTR, dres=None, ldr=0,
            dx=2 * PTR, dxd=L.F16, dg=PTR, ws=PTR, rows=4, cols=64):
        return lib.bf_rmsnorm_bwd(dy, ldy, dyd, x, ldx, xd, q, code, gamma, rstd, dres, ldr, dx, dxd, dg, ws, rows, cols, None)

    refused(L, bwd(dyd=4), -1, "dy_dtype")
    refused(L, bwd(xd=4), -1, "x_dtype")
    refused(L, bwd(x=None), -1, "exactly one")
    refused(L, bwd(q=PTR, code=PTR), -1, "exactly one")
    refused(L, bwd(code=PTR), -1, "checkpoint")
    refused(L, bwd(dg=None), -1, "dgamma")
    refused(L, bwd(ws=None), -1, "null")
    refused(L, bwd(ldy=63), -1, "leading dimension")
    refused(L, bwd(dx=PTR, ldy=72), -1, "rows coincide")
    refused(L, bwd(dx=PTR, dxd=L.F32), -1, "rows coincide")
    refused(L, bwd(dres=2 * PTR, ldr=72), -1, "rows coincide")
    refused(L, bwd(rstd=PTR + 1), -2, "aligned")
    for rows, cols in ((0, 64), (1, 64), (5, 64), (10 ** 6, 64), (2 ** 31 - 129, 64), (7, 4096), (9000, 1024), (9000, 2048),
                       (9000, 4096), (9000, 8192), (9000, 9000), (9000, 20000), (3, 20000)):
        parts = lib.bf_rmsnorm_bwd_parts(rows, cols)
        assert (parts == 0) if rows == 0 else (1 <= parts <= min(rows, 1280)), (rows, cols, parts)


def test_embedding_refusals(L):
    lib = L.lib
    refused(L, lib.bf_embed_scaled_fwd(PTR, PTR, 6, PTR, L.F32, 1.0, 4, 64, 100, None, None), -1, "dtype")
    refused(L, lib.bf_embed_scaled_fwd(PTR, PTR, L.F32, PTR, L.F32, 1.0, 4, 64, 0, None, None), -1, "bad shape")
    refused(L, lib.bf_embed_scaled_fwd(PTR, None, L.F32, PTR, L.F32, 1.0, 4, 64, 100, None, None), -1, "null")
    refused(L, lib.bf_embed_scaled_fwd(PTR + 2, PTR, L.F32, PTR, L.F32, 1.0, 4, 64, 100, None, None), -2, "aligned")
    refused(L, lib.bf_embed_scaled_fwd(PTR, PTR, L.F32, PTR, L.F32, 1.0, 1 << 30, 4096, 100, None, None), -1, "too large")

    def bwd(dy=PTR, ld=64, dt=L.F16, ids=PTR, grad=PTR, n=2000, cols=64, vocab=100, ws=PTR, size=None, acc=1):
        size = lib.bf_embed_scaled_bwd_workspace_bytes(n, cols, vocab) if size is None else size
        return lib.bf_embed_scaled_bwd(dy, ld, dt, ids, grad, 1.0, acc, -1, n, cols, vocab, None, ws, size, None)

    refused(L, bwd(dt=3), -1, "dy_dtype")
    refused(L, bwd(vocab=0), -1, "bad shape")
    refused(L, bwd(cols=0), -1, "bad shape")
    refused(L, bwd(grad=None), -2, "grad")
    refused(L, bwd(ld=63), -1, "ld_dy")
    refused(L, bwd(dy=None), -1, "null")
    refused(L, bwd(dy=PTR + 1), -2, "aligned")
    refused(L, bwd(ws=None), -4, "workspace")
    refused(L, bwd(size=100), -4, "workspace")
    refused(L, bwd(ws=PTR + 4), -2, "workspace")
    refused(L, bwd(n=(1 << 30) + 1, size=0), -1, "2^30")
    assert bwd(n=0, dy=None, ids=None) == 0
    size = lib.bf_embed_scaled_bwd_workspace_bytes
    assert size(512, 64, 100) == 0 and size(513, 64, 100) > 16 * 513
    assert size(1 << 20, 1024, 1 << 20) < 1 << 29


def test_wrappers_refuse_before_the_library(L):
    from bifold_amd.hip import ops
    x = torch.zeros(4, 64)
    q, code = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    gamma, ids = torch.ones(64), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.act8_pack(x), lambda: ops.act8_unpack((q, code), torch.float32),
                 lambda: ops.act8_gelu_fwd(x, L.ACT_ERF_GELU), lambda: ops.act8_gelu_bwd(x, (q, code), L.ACT_ERF_GELU),
                 lambda: ops.rmsnorm_fwd(x, gamma, torch.float32), lambda: ops.rmsnorm_fwd_fp8(x, gamma),
                 lambda: ops.rmsnorm_bwd(x, x, gamma, torch.ones(4), torch.empty(64)),
                 lambda: ops.embed_scaled_fwd(ids, x, 1.0), lambda: ops.embed_scaled_bwd(x, ids, 10, 1.0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(RuntimeError, match="checkpoint is"):
        ops.act8_unpack((q, code[:, :1]), torch.float32)
    with pytest.raises(RuntimeError, match="checkpoint is"):
        ops.act8_unpack((q.to(torch.uint8), code), torch.float32)
    with pytest.raises(RuntimeError, match="does not match"):
        ops.act8_gelu_bwd(x[:3], (q, code), L.ACT_ERF_GELU)
    buf = torch.zeros(5, 64)
    with pytest.raises(RuntimeError, match="memory of its own"):
        ops.act8_gelu_bwd(buf[:4], (q, code), L.ACT_ERF_GELU, out=buf[1:])
    with pytest.raises(RuntimeError, match="unit inner stride"):
        ops.act8_pack(torch.zeros(64, 4).t())
    with pytest.raises(RuntimeError, match="do not overlap"):
        ops.act8_pack(torch.zeros(1, 64).expand(4, 64))
    with pytest.raises(RuntimeError, match="at least one element"):
        ops.act8_pack(torch.zeros(4, 0))
    with pytest.raises(RuntimeError, match="gamma"):
        ops.rmsnorm_fwd(x, gamma[:32], torch.float32)
    with pytest.raises(RuntimeError, match="without a delta"):
        ops.rmsnorm_fwd(x, gamma, torch.float32, x_out=torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match="x_out is x"):
        ops.rmsnorm_fwd(buf[:4], gamma, torch.float32, delta=x, x_out=buf[1:])
    with pytest.raises(RuntimeError, match="x_out is delta"):
        ops.rmsnorm_fwd(x, gamma, torch.float32, delta=buf[:4], x_out=buf[1:])
    with pytest.raises(RuntimeError, match="one shape"):
        ops.rmsnorm_bwd(x, x[:3], gamma, torch.ones(4), torch.empty(64))
    with pytest.raises(RuntimeError, match="out is dy"):
        ops.rmsnorm_bwd(buf[:4], x, gamma, torch.ones(4), torch.empty(64), out=buf[1:])
    with pytest.raises(RuntimeError, match="must not overlap"):
        ops.rmsnorm_bwd(x, buf[:4], gamma, torch.ones(4), torch.empty(64), out=buf[1:])
    both = torch.zeros(4 * 64 + 64)
    with pytest.raises(RuntimeError, match="overlap gamma"):
        ops.rmsnorm_fwd(x, both[200:264], torch.float32, delta=x, x_out=both[:256].view(4, 64))
    for used in (0, 1):
        with pytest.raises(RuntimeError, match="dgamma_out is memory of its own"):
            g, r = torch.ones(64), torch.ones(64)
            ops.rmsnorm_bwd(torch.zeros(64, 64), torch.zeros(64, 64), g, r, (g, r)[used])
    with pytest.raises(TypeError, match="int32"):
        ops.embed_scaled_fwd(ids.long(), x, 1.0)
    with pytest.raises(TypeError, match="err_flag"):
        ops.embed_scaled_fwd(ids, x, 1.0, err_flag=torch.zeros(1))
    with pytest.raises(RuntimeError, match="rows of dy"):
        ops.embed_scaled_bwd(x[:3], ids, 10, 1.0)
    with pytest.raises(ValueError, match="padding_idx"):
        ops.embed_scaled_bwd(x, ids, 10, 1.0, padding_idx=10)
    with pytest.raises(RuntimeError, match="add into"):
        ops.embed_scaled_bwd(x, ids, 10, 1.0, accumulate=True)
    with pytest.raises(RuntimeError, match="apart from dy"):
        ops.embed_scaled_bwd(x, ids, 10, 1.0, out=torch.zeros(9, 64))
    with pytest.raises(RuntimeError, match="and the ids"):
        ops.embed_scaled_bwd(x, both[:4].view(torch.int32), 4, 1.0, out=both[:256].view(4, 64))


def test_lora_checkpoint_values():
    from bifold.models.siglip_encoder import SiglipTowers
    tower = dict(hidden_size=64, intermediate_size=128, num_hidden_layers=1, num_attention_heads=2)
    vision, text = dict(tower, image_size=32, patch_size=16), dict(tower, vocab_size=100, max_position_embeddings=64)
    lora = dict(r=8, alpha=32, targets=["q_proj", "v_proj"])
    assert SiglipTowers(vision, text, lora=lora).lora["checkpoint"] == "native"
    assert SiglipTowers(vision, text, lora=dict(lora, checkpoint="int8")).lora["checkpoint"] == "int8"
    with pytest.raises(ValueError, match="native or int8"):
        SiglipTowers(vision, text, lora=dict(lora, checkpoint="int4"))


def test_norm_gradient_over_an_operand_is_refused(L):
    """dgamma_out is written while other workgroups still read, so it overlaps no operand, in part or whole."""
    from bifold_amd.hip import ops
    rows, cols = 4, 64

    def bwd(dg, dy=None, x=None, gamma=None, rstd=None, dres=None):
        return ops.rmsnorm_bwd(torch.zeros(rows, cols) if dy is None else dy, torch.zeros(rows, cols) if x is None else x,
                               torch.ones(cols) if gamma is None else gamma, torch.ones(rows) if rstd is None else rstd, dg, dres=dres)

    flat = torch.zeros((rows + 1) * cols)
    rows_of = flat[:rows * cols].view(rows, cols)
    wide = torch.zeros(rows, 2 * cols)
    mine = "dgamma_out is memory of its own"
    for dg in (flat[:cols], flat[100:100 + cols], flat[rows * cols - 1:(rows + 1) * cols - 1]):
        for name in ("dy", "x", "dres"):
            with pytest.raises(RuntimeError, match=mine):
                bwd(dg, **{name: rows_of})
    for name in ("dy", "x", "dres"):                              # a view that starts in front of dgamma_out and ends behind it
        with pytest.raises(RuntimeError, match=mine):
            bwd(wide[2, 8:8 + cols], **{name: wide[:, :cols]})
    with pytest.raises(RuntimeError, match=mine):
        bwd(flat[1:1 + cols], gamma=flat[:cols])
    with pytest.raises(RuntimeError, match=mine):
        bwd(flat[:cols], rstd=flat[60:64])
    q, code = flat[:rows * cols // 4].view(torch.int8).view(rows, cols), torch.ones(rows, 2, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match=mine):
        bwd(flat[8:8 + cols], x=(q, code))
    big = torch.zeros(2 * cols)
    with pytest.raises(RuntimeError, match=mine):
        bwd(big[:cols], x=(torch.zeros(rows, cols, dtype=torch.int8), big.view(torch.uint8)[12:20].view(rows, 2)))
    with pytest.raises(RuntimeError, match="no CPU path"):        # next to its operands: nothing to refuse but the device
        bwd(flat[rows * cols:], dy=rows_of, gamma=big[:cols], dres=None)


def test_norm_in_place_over_gamma_is_refused(L):
    """x += delta in place, with gamma inside x: rows would be scaled by what others have already written."""
    from bifold_amd.hip import ops
    flat = torch.zeros(5 * 64)
    x, delta = flat[:256].view(4, 64), torch.zeros(4, 64)
    for gamma in (flat[:64], flat[100:164], flat[255:319]):
        for out in (None, x):
            with pytest.raises(RuntimeError, match="must not overlap gamma"):
                ops.rmsnorm_fwd(x, gamma, torch.float32, delta=delta, x_out=out)
            with pytest.raises(RuntimeError, match="must not overlap gamma"):
                ops.rmsnorm_fwd_fp8(x, gamma, delta=delta, x_out=out)
    for call in (lambda: ops.rmsnorm_fwd(x, flat[256:], torch.float32, delta=delta),
                 lambda: ops.rmsnorm_fwd(x, flat[:64], torch.float32, delta=delta, write_x=False)):      # read only
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_columns_of_one_buffer_are_memory_of_their_own(L):
    """Outputs beside their inputs in one packed buffer share no element with them, and are taken."""
    from bifold_amd.hip import ops
    wide = torch.zeros(4, 3 * 64)
    left, mid, right = wide[:, :64], wide[:, 64:128], wide[:, 128:]
    gamma, kept = torch.ones(64), (torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8))
    for out in (left, right):
        for call in (lambda: ops.act8_gelu_bwd(mid, kept, L.ACT_ERF_GELU, out=out),
                     lambda: ops.rmsnorm_fwd(mid, gamma, torch.float32, delta=torch.zeros(4, 64), x_out=out),
                     lambda: ops.rmsnorm_fwd(torch.zeros(4, 64), gamma, torch.float32, delta=mid, x_out=out)):
            with pytest.raises(RuntimeError, match="no CPU path"):
                call()
    for out in (wide[:, 63:127], wide[:, 65:129], wide[:, 127:191], wide[:, 1:65]):
        with pytest.raises(RuntimeError, match="memory of its own"):
            ops.act8_gelu_bwd(mid, kept, L.ACT_ERF_GELU, out=out)


@pytest.mark.parametrize("seed", range(4))
def test_overlap_against_the_addresses(L, seed):
    """Views of one buffer share memory exactly where a set of their bytes says so; other layouts are never missed."""
    import random
    from bifold_amd.hip import ops
    rng = random.Random(seed)
    buf = torch.zeros(400, dtype=torch.uint8)

    def view():
        dtype = rng.choice([torch.uint8, torch.float16, torch.float32])
        flat = buf.view(dtype)
        rows, cols = rng.randint(0, 5), rng.randint(1, 9)
        step = rng.choice([cols, rng.randint(cols, 20), 40 // flat.element_size()])
        step = max(step, cols)
        first = rng.randint(0, len(flat) - max(0, rows - 1) * step - cols)
        return flat.as_strided((rows, cols), (step, 1), first)

    def bytes_of(t):
        base, e = t.data_ptr() - buf.data_ptr(), t.element_size()
        return {base + (i * t.stride(0) + j) * e + k for i in range(t.shape[0]) for j in range(t.shape[1]) for k in range(e)}

    exact = 0
    for _ in range(3000):
        a, b = view(), view()
        meet, says = bool(bytes_of(a) & bytes_of(b)), ops._overlap(a, b)
        assert says == ops._overlap(b, a)
        if a.stride(0) * a.element_size() == b.stride(0) * b.element_size() and (a.shape[0] > 1 or b.shape[0] > 1):
            exact += not meet and not (a.is_contiguous() and b.is_contiguous())
            far = a.shape[0] <= 1 or b.shape[0] <= 1
            assert says == meet or (far and says)
        assert says or not meet, (a.shape, a.stride(), b.shape, b.stride())
    assert exact > 20


def test_size_limits_as_the_header_states_them(L):
    """One step over each limit is refused for its size; at the limit of the gradient the next check (a workspace of one byte)
    is what refuses."""
    lib = L.lib
    most = 2 ** 31 - 4096
    for dtype, v in ((L.F32, 4), (L.BF16, 8), (L.F16, 8)):
        for cols in (1, v, v + 1, 1000, 1 << 30):
            n = most // -(-cols // v) + 1
            if n < 2 ** 31:
                refused(L, lib.bf_embed_scaled_fwd(PTR, PTR, dtype, PTR, dtype, 1.0, n, cols, 100, None, None), -1, "too large")
    refused(L, lib.bf_embed_scaled_fwd(PTR, PTR, L.F32, PTR, L.F32, 1.0, 1, (1 << 30) + 1, 100, None, None), -1, "bad shape")
    refused(L, lib.bf_act8_pack(PTR, 33, L.F16, PTR, PTR, (2 ** 29 - 1024) // 2 + 1, 33, None), -1, "2^34")

    def bwd(dt, n, cols, vocab):
        return lib.bf_embed_scaled_bwd(PTR, cols, dt, PTR, PTR, 1.0, 0, -1, n, cols, vocab, None, PTR, 1, None)

    def fits(n, cols, vocab, width):
        return (n // 16 + 1) * -(-cols // width) // 4 + vocab // 32 < 2 ** 24 - 2

    for dt, width in ((L.F32, 256), (L.BF16, 512), (L.F16, 512)):
        for cols in (1, width, width + 1, 40 * width):
            for vocab in (1, 2 ** 28, 2 ** 29 - 10 ** 6):
                low, high = 513, 2 ** 30                            # the largest n that fits
                if not fits(low, cols, vocab, width):
                    continue
                while low < high:
                    mid = (low + high + 1) // 2
                    low, high = (mid, high) if fits(mid, cols, vocab, width) else (low, mid - 1)
                refused(L, bwd(dt, low, cols, vocab), -4, "workspace")
                if low < 2 ** 30:
                    refused(L, bwd(dt, low + 1, cols, vocab), -1, "too large")
                else:
                    refused(L, bwd(dt, low + 1, cols, vocab), -1, "2^30")


def test_polynomials_of_the_normal_tail():
    """The coefficients in the source against Phi(-a) e^(a^2/2), in 64 bits: as near as the comments beside them say."""
    import os
    import re

    import numpy as np
    from scipy.special import erfcx
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "bifold_amd", "csrc", "act8.hip")).read()

    def coefficients(name):
        body = text[text.index(f"float {name}(float x, float& e) {{"):]
        body = body[:body.index("return e * (r * q);")]
        number = r"(-?[0-9.]+e[+-][0-9]+)f"
        first = re.findall(r"float r = " + number, body)
        return [np.float64(np.float32(c)) for c in first + re.findall(r"r = fmaf\(r, [uq], " + number, body)]

    def horner(c, u):
        r = np.zeros_like(u)
        for v in c:
            r = r * u + v
        return r

    for name, top, terms, near in (("normal_tail", 15.0, 9, 4.6e-8), ("normal_tail_fast", 14.3, 7, 8.0e-7)):
        a = np.linspace(0, top, 300001)
        c, q = coefficients(name), 1 / (a + 3.75)
        assert len(c) == terms, name
        got = q * horner(c, q if name.endswith("fast") else (a - 3.75) * q)
        off = np.abs(got / (0.5 * erfcx(a / np.sqrt(2))) - 1).max()
        assert off <= near, (name, off)
