// Host only: the forms of the int8 product that i8_form_for takes, for sizes read as lines "n_strips m_strips steps behind": the threads of its launch, and the form.
#include "../../nihilus_amd/csrc/i8_product.h"

#include <cstdio>

int main() {
	long long n, m, steps, behind;
	while (std::scanf("%lld %lld %lld %lld", &n, &m, &steps, &behind) == 4) {
		const nh::i8_form form = nh::i8_form_for(n, m, steps, behind);
		long long fn = 2, fm = 2, threads = 512; // as in i8_launch_product
		switch (form) {
		case nh::I8_ROWS_16: fn = 1, fm = 1; break;
		case nh::I8_ROWS_32: break;
		case nh::I8_TILE_64: fn = fm = 4; break;
		case nh::I8_TILE_128_64: fn = 8, fm = 4; break;
		case nh::I8_TILE_128_HALVES: fn = fm = 8, threads = 1024; break;
		case nh::I8_TILE_128_96: fn = 8, fm = 6; break;
		case nh::I8_TILE_128: fn = fm = 8; break;
		case nh::I8_TILE_128_160: fn = 8, fm = 10; break;
		case nh::I8_TILE_128_192: fn = 8, fm = 12; break;
		case nh::I8_TILE_256: fn = fm = 16; break;
		}
		std::printf("%lld %d\n", nh::i8_grid((n + fn - 1) / fn, (m + fm - 1) / fm) * threads, static_cast<int>(form));
	}
}
