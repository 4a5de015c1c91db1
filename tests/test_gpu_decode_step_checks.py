"""What a bound step of the example decoder refuses (leanstream_amd.decode_step): its calls point into buffers of one
number of tokens, which other numbers would resize under them.
"""
import pytest

pytestmark = pytest.mark.gpu


def test_lengths_that_do_not_fit_the_step(torch_gpu):
    torch = torch_gpu
    from leanstream_amd.decode_step import Decoder

    decoder = Decoder(layers=1, sequences=2, max_context=64)
    step = decoder.bind(6, 4)
    u = torch.full((2,), 0.5, device="cuda")
    ids = torch.arange(8, device="cuda")
    where = step.hidden.data_ptr()
    for count, lengths in ((8, [(4, 4), (4, 4)]), (6, [(4, 4), (1, 1)]), (6, [(5, 5), (1, 1)]), (6, [(4, 4), (2, 65)]),
                           (6, [(4, 3), (2, 2)]), (6, [(6, 6)]), (6, [(7, 7), (-1, 1)])):
        with pytest.raises(ValueError, match="step"):
            step.run(ids[:count], lengths, u)
    assert step.hidden.data_ptr() == where and tuple(step.hidden.shape) == (6, decoder.width)
    step.run(ids[:6], [(4, 4), (2, 64)], u)
    torch.cuda.synchronize()
    assert int(step.status) == 0
