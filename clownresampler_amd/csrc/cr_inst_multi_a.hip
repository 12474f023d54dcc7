// cr_inst_multi_a.hip - instance unit: 8 channels 48 -> 44.1 kHz with every tuning variant  (see cr_instances.hpp)
#include "cr_instances.hpp"

namespace crk
{

int specials_multi_a(void *table, int capacity)
{
	static const special mine[] = {
	    // cfg 4: 8 channels 48 -> 44.1 kHz (5-6 taps; 6 slots on shifted windows).  Ticketed tiles: 252.2 us, round-robin tiles: 260.9 us on one
	    // box (with a vmcnt(0) behind the draw or the mailbox they were 1-8 % SLOWER here)
	    with_signed_chain<8, 6, CRHIP_ROWMODE_AFFINE, CRHIP_NORM_S31, 2, true>(make_special<8, 6, CRHIP_ROWMODE_AFFINE, CRHIP_NORM_S31, 2, false, true>()),
	};
	const int n = (int)(sizeof(mine) / sizeof(mine[0]));
	if (table == nullptr)
		return n;   // (asked for the count: specials() sizes its table from the providers)
	if (n > capacity)
		return -1;
	memcpy(table, mine, sizeof(mine));
	return n;
}

} // namespace crk
